"""The fp32 optimizers refuse 16-bit gradients and moments, and leave the parameter as it is."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from plast_amd import abi
from plast_amd.abi import BFLOAT16, FLOAT16

pytestmark = pytest.mark.gpu


def _step(L, kind, arr, m=None, v=None):
    if kind == "sgd":
        L.sgd_step_hip(C.byref(abi.SGD(0.1)), arr, 1)
        return None
    o = (abi.Adam if kind == "adam" else abi.AdamW)()
    o.lr, o.beta1, o.beta2, o.epsilon = 0.1, 0.9, 0.999, 1e-8
    if m is not None:
        o.m, o.v = m, v
    getattr(L, f"{kind}_step_hip")(C.byref(o), arr, 1)
    return o


@pytest.mark.parametrize("half", [FLOAT16, BFLOAT16])
@pytest.mark.parametrize("kind", ["sgd", "adam", "adamw"])
def test_half_gradients_and_moments(kind, half):
    from plast_amd import runtime as rt
    L = rt.lib()
    values = np.arange(12, dtype=np.float32)
    p, g = rt.DeviceTensor.from_numpy(values, requires_grad=True), rt.DeviceTensor((12,), half)
    full = p.t.grad
    p.t.grad = C.pointer(g.t)
    arr, keep = abi.tensor_array(p.t)
    o = _step(L, kind, arr)
    with pytest.raises(rt.PlastHipError, match="not a float32 tensor"):
        L.check()
    if o is not None:
        getattr(L, f"plast_hip_{kind}_release")(C.byref(o), 1)
        p.t.grad = full
        m, v = rt.DeviceTensor((12,), half), rt.DeviceTensor((12,))
        for a, b in ((m, v), (v, m)):
            (ma, ka), (va, kb) = abi.tensor_array(a.t), abi.tensor_array(b.t)
            _step(L, kind, arr, ma, va)
            with pytest.raises(rt.PlastHipError, match="moment tensors of parameter 0"):
                L.check()
    assert np.array_equal(p.numpy(), values)
