"""The fp32 ops refuse 16-bit tensors where they would write or accumulate 32-bit values into half the bytes. Checked
before the GPU is touched."""
from __future__ import annotations

import ctypes as C

import pytest

from plast_amd.abi import BFLOAT16, DIM_ALL, FLOAT16, INT32, KernelParams
from plast_amd.runtime import LIB_PATH, DeviceTensor, Library, PlastHipError
from test_operator_refusals import T

pytestmark = pytest.mark.skipif(not LIB_PATH.exists(), reason="the library is not built")
HALF = [FLOAT16, BFLOAT16]


@pytest.fixture(scope="module")
def L():
    lib = Library()
    yield lib
    lib.plast_hip_clear_error()


def call(L, kind, name, ins, out, p=KernelParams(0, 0, 0.0)):
    L.plast_hip_clear_error()
    arr = (C.c_void_p * len(ins))(*[C.addressof(t) for t in ins])
    L.by_address[kind, name](arr, C.addressof(out), p)
    with pytest.raises(PlastHipError, match="16-bit dtype"):
        L.check()


@pytest.mark.parametrize("half", HALF)
@pytest.mark.parametrize("name", ["sum", "mean", "max", "min"])
def test_reductions(L, name, half):
    for p in (KernelParams(DIM_ALL, 0, 0.0), KernelParams(1, 0, 0.0)):
        call(L, "forward", name, [T((4, 6))], T((4,), half), p)
        call(L, "backward", name, [T((4, 6), grad=T((4, 6), half))], T((4,), grad=T((4,))), p)
        call(L, "backward", name, [T((4, 6), grad=T((4, 6)))], T((4,), grad=T((4,), half)), p)


@pytest.mark.parametrize("half", HALF)
@pytest.mark.parametrize("name", ["add", "sub", "mul", "div"])
def test_binary_gradients(L, name, half):
    a, b, out = T((4, 6), grad=T((4, 6))), T((6,), grad=T((6,))), T((4, 6), grad=T((4, 6)))
    call(L, "backward", name, [T((4, 6), grad=T((4, 6), half)), b], out)
    call(L, "backward", name, [a, T((6,), grad=T((6,), half))], out)
    call(L, "backward", name, [a, b], T((4, 6), grad=T((4, 6), half)))


@pytest.mark.parametrize("half", HALF)
@pytest.mark.parametrize("name", ["exp", "log", "neg", "abs", "sin", "cos", "tan", "leaky_relu", "view", "flatten",
                                  "squeeze", "unsqueeze", "transpose", "softmax", "log_softmax"])
def test_unary_and_view_gradients(L, name, half):
    p = KernelParams(1, 0, 0.0)
    call(L, "backward", name, [T((4, 6), grad=T((4, 6), half))], T((4, 6), grad=T((4, 6))), p)
    call(L, "backward", name, [T((4, 6), grad=T((4, 6)))], T((4, 6), grad=T((4, 6), half)), p)


@pytest.mark.parametrize("half", HALF)
def test_cross_entropy_gradients(L, half):
    rest = [T((4,), INT32), T((4, 2))]
    call(L, "backward", "softmax_cross_entropy", [T((4, 6), grad=T((4, 6), half)), *rest], T((4,), grad=T((4,))))
    call(L, "backward", "softmax_cross_entropy", [T((4, 6), grad=T((4, 6))), *rest], T((4,), grad=T((4,), half)))


@pytest.mark.parametrize("half", HALF)
def test_ones_of_a_gradient(L, half):
    L.plast_hip_clear_error()
    t = T((4,), grad=T((4,), half))
    L.set_ones_grad_hip(C.byref(t))
    with pytest.raises(PlastHipError, match="16-bit dtype"):
        L.check()


def test_generated_values():
    t = DeviceTensor.__new__(DeviceTensor)
    t.itemsize, t.shape = 2, (4,)
    with pytest.raises(ValueError, match="32 bits"):
        t.fill_("normal", 0, 0.0, 1.0)
