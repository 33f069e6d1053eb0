"""Newton-Schulz into views whose axes step just past what the ones below them span."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_newton_schulz import iterate, near, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape, strides", [
    ((70, 4), (7, 2)),            # every second column of 7
    ((4, 70), (2, 7)),            # the same transposed
    ((3, 20, 11), (420, 21, 2)),  # and of a stack whose matrices begin where the last one ends
], ids=str)
def test_columns_of_wider_rows(shape, strides):
    print(f"newton_schulz {shape} {strides}", flush=True)
    rng = np.random.RandomState(1)
    g = rng.randn(*shape).astype(np.float32)
    size = 1 + sum((e - 1) * s for e, s in zip(shape, strides))
    got = run(g, "f32", place=(strides, 0, size), place_out=(strides, 0, size))
    want = np.stack([iterate(m) for m in g]) if g.ndim == 3 else iterate(g)
    near(got, want, 3.3e-4, "f32", f"{shape} {strides}")
