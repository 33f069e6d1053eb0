"""Newton-Schulz of 16-bit matrices: the iteration has the accuracy of the float32 one and its result is rounded
once, so that it equals the rounded 64-bit result but where an error moves a value over a rounding border.

For an error e_i of value v_i before its rounding, whose steps are at most eps |v_i| (eps: torch.finfo's, 2^-7 and
2^-10), that happens with probability |e_i| / step and costs a step: the squared difference to the rounded exact
result is on average the sum of step_i |e_i|, at most eps |v| |e|. With |e| = 2e-5 |v|, as for float32, the norm is
sqrt(2e-5 eps) |v|; half as much again is allowed for the spread of so many elements. Factors of 11 bits leave
2.4e-3 of it, six times that much, in bfloat16."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_newton_schulz import iterate, run
from token_cases import load, store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind, eps", [("bf16", 2.0 ** -7), ("f16", 2.0 ** -10)])
@pytest.mark.parametrize("shape", [(256, 640), (300, 800), (800, 300), (1100, 2900), (2605, 1001)], ids=str)
def test_rounded_once(shape, kind, eps):
    print(f"newton_schulz {kind} {shape}", flush=True)
    rng = np.random.RandomState(shape[0])
    g = load(store(rng.randn(*shape).astype(np.float32), kind))
    got = run(g, kind).astype(np.float64)
    want = iterate(g)
    once = load(store(want.astype(np.float32), kind)).astype(np.float64)
    off, bar = np.linalg.norm(got - once), 1.5 * np.sqrt(2e-5 * eps) * np.linalg.norm(want)
    assert off <= bar, f"{kind} {shape}: off by {off:.3g} from the rounded result, at most {bar:.3g}"
