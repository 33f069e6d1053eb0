"""Layer norm's gradients over rows of more columns than one grid joins the shares of."""
from __future__ import annotations

import numpy as np
import pytest

from block_cases import U
from plast_amd.abi import KernelParams

pytestmark = pytest.mark.gpu


def test_more_columns_than_one_grid_joins():
    """Eight lanes a column of either sum reach 2^32 lanes at 2^28 columns. x is 1 and -1 in turn: a mean of 0 and a variance of
    1, each off by the roundings of some sixteen sums of whole numbers."""
    from plast_amd.runtime import DeviceTensor, backward, forward
    width = 2 ** 28 + 40
    print(f"layer norm 1 x {width}", flush=True)
    x = np.resize(np.array([1, -1], np.float16), width)
    dy = np.resize(np.arange(-7, 8).astype(np.float16) / 8, width)
    X, Y = DeviceTensor.from_numpy(x[None]), DeviceTensor.from_numpy(np.zeros((1, width), np.float16))
    G = DeviceTensor.from_numpy(dy[None])
    Y.t.grad = G.p
    W, B = (DeviceTensor((width,), requires_grad=True) for _ in range(2))
    S, p = DeviceTensor((1, 2)), KernelParams(0, 0, 1e-5)
    forward("layer_norm", [X, W, B, S], Y, p)
    backward("layer_norm", [X, W, B, S], Y, p)
    db, dw = B.grad.numpy(), W.grad.numpy()
    assert np.array_equal(db, dy)
    want = dy.astype(np.float32) * x * np.float32((1 + 1e-5) ** -0.5)
    assert (np.abs(dw - want) <= 24 * U * np.abs(want)).all()
