"""What the token log-probability and the orthogonalisation entry points refuse, on the CPU: arguments
are checked before the GPU is touched, and every refusal is an error with a message."""
from __future__ import annotations

import ctypes as C

import pytest

from plast_amd import abi
from plast_amd.abi import BFLOAT16, CPU, FLOAT16, FLOAT32, GPU, INT32, INT64, KernelParams
from plast_amd.runtime import LIB_PATH, Library, PlastHipError

AT = 1 << 20  # an address that is never followed

pytestmark = pytest.mark.skipif(not LIB_PATH.exists(), reason="the library is not built")


@pytest.fixture(scope="module")
def L():
    lib = Library()
    yield lib
    lib.plast_hip_clear_error()


def T(shape, dtype=FLOAT32, strides=None, device=GPU, data=AT, grad=None):
    return abi.make_tensor(data, shape, strides, dtype, device, grad is not None, grad)


def token_call(L, kind="forward", x=None, tokens=None, stats=None, entropy=None, logp=None, top=0, temp=1.0,
               tops=None, drop=None):
    n, v = 6, 10
    ins = [x or T((n, v)), tokens or T((n,), INT32), stats or T((n, 2)), entropy or T((n,))]
    ins += list(tops or ())
    if drop is not None:
        ins[drop] = None
    arr = (C.c_void_p * 6)(*[C.addressof(t) if t is not None else None for t in ins])
    out = logp or T((n,))
    L.plast_hip_clear_error()
    L.by_address[kind, "token_logprob"](arr, C.addressof(out), KernelParams(top, 0, temp))


def refused(L, match):
    with pytest.raises(PlastHipError, match=match):
        L.check()


@pytest.mark.parametrize("kw, match", [
    (dict(x=T((6, 10), INT32)), "FLOAT32, FLOAT16 or BFLOAT16"),
    (dict(x=T((6, 10), INT64)), "FLOAT32, FLOAT16 or BFLOAT16"),
    (dict(x=T((6, 10), device=CPU)), "GPU tensor"),
    (dict(x=T(())), "last axis"),
    (dict(x=T((6, 10), strides=(1, 6))), "contiguous, not strided by 6"),
    (dict(x=T((6, 0))), "rows of 0 logits"),
    (dict(x=T((6, 1 << 31))), "logits are not supported"),
    (dict(x=T((6, 10), data=0)), "no data"),
    (dict(drop=0), "NULL"),
    (dict(drop=1), "NULL"),
    (dict(drop=2), "stats, entropy and logp"),
    (dict(drop=3), "stats, entropy and logp"),
    (dict(tokens=T((6,), INT64)), "tokens must be"),
    (dict(tokens=T((5,), INT32)), "tokens must be"),
    (dict(tokens=T((6,), INT32, strides=(2,))), "tokens must be"),
    (dict(stats=T((6,))), "stats, entropy and logp"),
    (dict(stats=T((6, 2), FLOAT16)), "stats, entropy and logp"),
    (dict(entropy=T((6,), strides=(0,))), "stats, entropy and logp"),
    (dict(logp=T((7,))), "stats, entropy and logp"),
    (dict(logp=T((6,), BFLOAT16)), "stats, entropy and logp"),
    (dict(temp=0.0), "temperature"),
    (dict(temp=-1.0), "temperature"),
    (dict(temp=float("nan")), "temperature"),
    (dict(temp=float("inf")), "temperature"),
    (dict(temp=1e-40), "too small"),
    (dict(top=33, tops=(T((6, 33)), T((6, 33), INT32))), "more than 32"),
    (dict(top=2, tops=(T((6, 3)), T((6, 2), INT32))), "top_logp and top_ids"),
    (dict(top=2, tops=(T((6, 2)), T((6, 2), INT64))), "top_logp and top_ids"),
    (dict(top=2), "top_logp and top_ids"),
])
def test_forward_refuses(L, kw, match):
    token_call(L, **kw)
    refused(L, match)


@pytest.mark.parametrize("grad, match", [
    (T((6, 10), FLOAT16), "x's type and shape"),
    (T((6, 11)), "x's type and shape"),
    (T((6, 10), strides=(20, 2)), "contiguous last axis"),
    (T((6, 10), strides=(0, 1)), "overlap"),
    (T((6, 10), strides=(9, 1)), "overlap"),
    (T((6, 10), data=0), "x's type and shape"),
])
def test_backward_refuses(L, grad, match):
    token_call(L, "backward", x=T((6, 10), grad=grad))
    refused(L, match)


def test_backward_without_a_gradient(L):
    x = T((6, 10))
    token_call(L, "backward", x=x)
    L.check()  # nothing asked for
    x.requires_grad = True
    token_call(L, "backward", x=x)
    refused(L, "has none")
    token_call(L, "backward", x=T((6, 10), grad=T((6, 10))), logp=T((6,), grad=T((5,))))
    refused(L, "upstream")


def test_step_refuses(L):
    def call(dx=None, dlogp=None, temp=1.0, entropy=None):
        a = [T((6, 10)), T((6,), INT32), dlogp, None, T((6,)), entropy or T((6,)), dx]
        L.plast_hip_clear_error()
        L.token_logprob_step_hip(*[C.addressof(t) if t is not None else None for t in a], temp)
    call()
    refused(L, "dx is NULL")
    call(T((6, 10), BFLOAT16))
    refused(L, "x's type and shape")
    call(T((6, 10)), dlogp=T((6,), FLOAT16))
    refused(L, "upstream")
    call(T((6, 10)), entropy=T((5,)))
    refused(L, "entropy and logp")
    call(T((6, 10)), temp=0.0)
    refused(L, "temperature")


def rule(**kw):
    return abi.NewtonSchulz(**{**dict(a=3.4445, b=-4.775, c=2.0315, eps=1e-7, steps=5), **kw})


@pytest.mark.parametrize("g, out, r, match", [
    (T((8,)), T((8,)), rule(), "matrix or stack"),
    (T((2, 2, 8, 8)), T((2, 2, 8, 8)), rule(), "matrix or stack"),
    (T((8, 8), INT32), T((8, 8), INT32), rule(), "matrix or stack"),
    (T((8, 8), device=CPU), T((8, 8)), rule(), "matrix or stack"),
    (T((8, 8)), T((8, 8), FLOAT16), rule(), "g's type and shape"),
    (T((8, 8)), T((8, 9)), rule(), "g's type and shape"),
    (T((8, 8)), T((1, 8, 8)), rule(), "g's type and shape"),
    (T((8, 8)), T((8, 8), strides=(0, 1)), rule(), "overlap"),
    (T((8, 8)), T((8, 8), strides=(7, 1)), rule(), "overlap"),
    (T((3, 8, 8)), T((3, 8, 8), strides=(32, 8, 1)), rule(), "overlap"),
    (T((8, 8), data=0), T((8, 8)), rule(), "no data"),
    (T((8, 1 << 20)), T((8, 1 << 20)), rule(), "not supported"),
    (T((8, 8)), T((8, 8)), rule(steps=-1), "0 to 1000 steps"),
    (T((8, 8)), T((8, 8)), rule(a=float("nan")), "finite coefficients"),
    (T((8, 8)), T((8, 8)), rule(eps=-1.0), "eps"),
    (T((8, 8)), T((8, 8)), rule(a=5.5, b=-12.0, c=7.5), "diverges"),
    (T((8, 8)), T((8, 8)), rule(a=1e30), "diverges"),
])
def test_newton_schulz_refuses(L, g, out, r, match):
    L.plast_hip_clear_error()
    L.newton_schulz_hip(C.addressof(g), C.addressof(out), C.addressof(r))
    refused(L, match)


@pytest.mark.parametrize("p, m, match", [
    (T((8,), grad=T((8,))), T((8,)), "parameter 0"),
    (T((8, 8), FLOAT16, grad=T((8, 8), FLOAT16)), T((8, 8)), "parameter 0"),
    (T((8, 8), strides=(1, 8), grad=T((8, 8))), T((8, 8)), "parameter 0"),
    (T((8, 8), grad=T((8, 4))), T((8, 8)), "parameter 0"),
])
def test_muon_refuses(L, p, m, match):
    arr, keep = abi.tensor_array(p)
    held, keep_m = abi.tensor_array(m)
    opt = abi.Muon(0.02, 0.95, 0.0, 1, rule(), held)
    L.plast_hip_clear_error()
    L.muon_step_hip(C.addressof(opt), C.cast(arr, C.c_void_p), 1)
    refused(L, match)
    L.muon_step_hip(None, C.cast(arr, C.c_void_p), 1)
    refused(L, "NULL")
    opt.rule.steps = -1
    L.muon_step_hip(C.addressof(opt), C.cast(arr, C.c_void_p), 1)
    refused(L, "steps")
