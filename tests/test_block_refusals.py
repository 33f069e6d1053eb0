"""What layer norm, the gated recurrence and gradient clipping refuse, on the CPU: arguments are checked before the GPU is
touched, and every refusal is an error with a message."""
from __future__ import annotations

import ctypes as C

import pytest

from plast_amd import abi
from plast_amd.abi import BFLOAT16, CPU, FLOAT16, FLOAT32, INT32, INT64, KernelParams
from plast_amd.runtime import LIB_PATH
from test_operator_refusals import AT, L, T, refused  # noqa: F401

pytestmark = pytest.mark.skipif(not LIB_PATH.exists(), reason="the library is not built")


def _call(L, kind, name, ins, out, p):  # noqa: F811
    arr = (C.c_void_p * 8)(*[C.addressof(t) if t is not None else None for t in ins])
    L.plast_hip_clear_error()
    L.by_address[kind, name](arr, C.addressof(out) if out is not None else None, p)


def norm_call(L, kind="forward", eps=1e-5, out=True, **kw):  # noqa: F811
    ins = [kw.get("x", T((6, 10))), kw.get("w", T((10,))), kw.get("b", T((10,))), kw.get("stats", T((6, 2)))]
    _call(L, kind, "layer_norm", ins, T((6, 10), grad=T((6, 10))) if out is True else out, KernelParams(0, 0, eps))


@pytest.mark.parametrize("kw, match", [
    (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(b=None), "NULL"), (dict(stats=None), "NULL"), (dict(out=None), "NULL"),
    (dict(x=T((6, 10), INT32)), "FLOAT32, FLOAT16 or BFLOAT16"),
    (dict(x=T((6, 10), device=CPU)), "GPU tensor"),
    (dict(x=T(())), "last axis"),
    (dict(x=T((6, 10), strides=(1, 6))), "contiguous, not strided by 6"),
    (dict(x=T((6, 0))), "rows of 0"),
    (dict(x=T((1, 1 << 31))), "not supported"),
    (dict(x=T((1 << 31, 1))), "not supported"),
    (dict(x=T((6, 10), data=0)), "no data"),
    (dict(w=T((9,))), "weight and bias"), (dict(b=T((10,), FLOAT16)), "weight and bias"), (dict(w=T((10,), strides=(2,))), "weight and bias"),
    (dict(stats=T((6,))), "stats"), (dict(stats=T((6, 2), BFLOAT16)), "stats"),
    (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(out=T((6, 10), FLOAT16)), "output must have"), (dict(out=T((6, 11))), "output must have"),
    (dict(out=T((6, 10), strides=(0, 1))), "do not overlap"), (dict(out=T((6, 10), strides=(20, 2))), "contiguous last axis"),
    (dict(out=T((6, 10), data=0)), "output must have"), (dict(out=T((6, 10), strides=(20, 1), data=AT)), "other strides"),
    (dict(x=T((6, 10), strides=(0, 1)), out=T((6, 10), data=AT)), "other strides"),
])
def test_layer_norm_refuses(L, kw, match):  # noqa: F811
    norm_call(L, **kw)
    refused(L, match)


@pytest.mark.parametrize("kw, match", [
    (dict(out=None), "no gradient"), (dict(out=T((6, 10))), "no gradient"),
    (dict(out=T((6, 10), grad=T((6, 10), FLOAT16))), "output's gradient"), (dict(out=T((6, 10), grad=T((6, 9)))), "output's gradient"),
    (dict(out=T((6, 10), grad=T((6, 10), strides=(20, 2)))), "output's gradient"),
    (dict(x=T((6, 10), grad=T((6, 10), BFLOAT16))), "gradient of x"), (dict(x=T((6, 10), grad=T((6, 10), strides=(9, 1)))), "overlap"),
    (dict(x=T((6, 10), grad=T((6, 10), data=0))), "gradient of x"),
    (dict(w=T((10,), grad=T((9,)))), "weight and bias"), (dict(b=T((10,), grad=T((10,), FLOAT16))), "weight and bias"),
    (dict(w=T((10,), grad=T((10,))), b=T((10,), grad=T((10,)))), "one gradient"),
    (dict(x=T((6, 10), grad=T((6, 10)))), "in the place of"), (dict(x=T((6, 10), data=AT + 4096, grad=T((6, 10)))), "in the place of"),
])
def test_layer_norm_backward_refuses(L, kw, match):  # noqa: F811
    norm_call(L, "backward", **kw)
    refused(L, match)


def test_layer_norm_backward_with_gradients_that_are_missing(L):  # noqa: F811
    norm_call(L, "backward")
    L.check()  # nothing asked for
    for name, match in (("x", "has none"), ("w", "weight and bias"), ("b", "weight and bias")):
        t = T((6, 10) if name == "x" else (10,))
        t.requires_grad = True
        norm_call(L, "backward", **{name: t})
        refused(L, match)


def scan_call(L, kind="forward", dim=1, out=True, **kw):  # noqa: F811
    B, N, D = 3, 200, 5
    ins = [kw.get("f", T((B, N, D))), kw.get("v", T((B, N, D))), kw.get("initial", T((B, D))), kw.get("lengths", T((B,), INT32)),
           kw.get("last", T((B, D))), kw.get("states", T((B, -(-N // abi.RECURRENCE_CHUNK), D)))]
    _call(L, kind, "gated_recurrence", ins, T((B, N, D), grad=T((B, N, D))) if out is True else out, KernelParams(dim, 0, 0.0))


@pytest.mark.parametrize("kind", ["forward", "backward"])
@pytest.mark.parametrize("kw, match", [
    (dict(f=None), "NULL"), (dict(v=None), "NULL"), (dict(initial=None), "NULL"), (dict(lengths=None), "NULL"), (dict(last=None), "NULL"),
    (dict(f=T((3, 200, 5), INT64)), "FLOAT32, FLOAT16 or BFLOAT16"), (dict(f=T((600, 5))), "batch, time, channels"),
    (dict(f=T((3, 200, 5), device=CPU)), "GPU tensor"), (dict(f=T((3, 200, 5), data=0)), "f and v"),
    (dict(f=T((1 << 31, 1, 1))), "not supported"), (dict(f=T((1 << 16, 1, 1 << 16))), "not supported"),
    (dict(v=T((3, 200, 5), FLOAT16)), "f and v"), (dict(v=T((3, 201, 5))), "f and v"), (dict(v=T((3, 200, 5), strides=(2000, 10, 2))), "f and v"),
    (dict(f=T((3, 200, 5), strides=(1, 15, 3))), "f and v"),
    (dict(initial=T((3, 6))), "initial and the last"), (dict(last=T((3, 5), BFLOAT16)), "initial and the last"),
    (dict(last=T((3, 5), strides=(10, 1))), "initial and the last"),
    (dict(lengths=T((3,), INT64)), "lengths"), (dict(lengths=T((4,), INT32)), "lengths"), (dict(lengths=T((3,), INT32, data=0)), "lengths"),
    (dict(states=T((3, 1, 5))), "states"), (dict(states=None), "states"), (dict(states=T((3, -(-200 // abi.RECURRENCE_CHUNK), 5), FLOAT16)), "states"),
    (dict(dim=2), "params.dim|params.dim 1"),
])
def test_recurrence_refuses(L, kind, kw, match):  # noqa: F811
    scan_call(L, kind, **kw)
    refused(L, match)


@pytest.mark.parametrize("out", [None, T((3, 200, 5), FLOAT16), T((3, 200, 4)), T((3, 200, 5), strides=(1000, 0, 1)), T((3, 200, 5), strides=(0, 5, 1)),
                                 T((3, 200, 5), strides=(2000, 10, 2)), T((3, 200, 5), data=0)])
def test_recurrence_refuses_outputs(L, out):  # noqa: F811
    scan_call(L, out=out)
    refused(L, "the output must have")


def test_recurrence_refuses_its_operands_places(L):  # noqa: F811
    scan_call(L, out=T((3, 200, 5)), f=T((3, 200, 5), data=AT + 65536))
    refused(L, "in the place of")
    scan_call(L, out=T((3, 200, 5)), v=T((3, 200, 5), data=AT + 65536))
    refused(L, "in the place of")
    for steps in ((1 << 22) + 1, 2 ** 64 - 5):
        scan_call(L, f=T((3, 200, 5), strides=(5, steps, 1)))
        refused(L, "f and v")


def G(grad, shape=(3, 200, 5)):
    return T(shape, grad=grad)


@pytest.mark.parametrize("kw, match", [
    (dict(dim=0), "states that a forward pass"),
    (dict(out=G(T((3, 200, 5), FLOAT16))), "output's gradient"), (dict(out=G(T((3, 200, 5), strides=(2000, 10, 2)))), "output's gradient"),
    (dict(last=G(T((3, 4)), (3, 5))), "last state's gradient"), (dict(last=G(T((3, 5), FLOAT16), (3, 5))), "last state's gradient"),
    (dict(f=G(T((3, 200, 5), BFLOAT16))), "gradients of f and v"), (dict(v=G(T((3, 200, 5), strides=(0, 5, 1)))), "gradients of f and v"),
    (dict(v=G(T((3, 200, 5), data=0))), "gradients of f and v"),
    (dict(f=G(T((3, 200, 5), data=AT + 4096)), v=G(T((3, 200, 5), data=AT + 4096))), "one gradient"),
    (dict(initial=G(T((3, 4)), (3, 5))), "initial state's gradient"),
    (dict(f=G(T((3, 200, 5), data=AT))), "in the place of"), (dict(out=G(T((3, 200, 5), data=AT + 4096)), v=G(T((3, 200, 5), data=AT + 4096))), "in the place of"),
    (dict(initial=G(T((3, 5), data=AT + 64), (3, 5)), last=G(T((3, 5), data=AT + 64), (3, 5))), "have one gradient"),
])
def test_recurrence_backward_refuses(L, kw, match):  # noqa: F811
    scan_call(L, "backward", **kw)
    refused(L, match)


def test_recurrence_backward_with_gradients_that_are_missing(L):  # noqa: F811
    scan_call(L, "backward")
    L.check()  # nothing asked for
    for name, match in (("f", "gradients of f and v"), ("v", "gradients of f and v"), ("initial", "initial state's")):
        t = T((3, 5) if name == "initial" else (3, 200, 5))
        t.requires_grad = True
        scan_call(L, "backward", **{name: t})
        refused(L, match)


def clip_call(L, grads, bound=1.0, norm=None):  # noqa: F811
    params = [T(g[0] if isinstance(g, tuple) else tuple(g.shape[:g.ndim]), grad=g[1] if isinstance(g, tuple) else g) for g in grads]
    arr, keep = abi.tensor_array(*params)
    L.plast_hip_clear_error()
    L.clip_grad_norm_hip(C.cast(arr, C.c_void_p), len(params), bound, C.addressof(norm) if norm is not None else None)


@pytest.mark.parametrize("grads, kw, match", [
    ([T((8,))], dict(bound=-1.0), "max_norm"), ([T((8,))], dict(bound=float("nan")), "max_norm"),
    ([T((8,))], dict(norm=T((2,))), "one element"), ([T((8,))], dict(norm=T((1,), INT32)), "one element"),
    ([T((8,))], dict(norm=T((1,), data=0)), "one element"),
    ([T((8,), INT32)], {}, "parameter 0"), ([T((8,)), T((8, 8), device=CPU, data=AT + 4096)], {}, "parameter 1"),
    ([T((8, 8), strides=(1, 8))], {}, "parameter 0"), ([T((8,), data=0)], {}, "parameter 0"), ([((9,), T((8,)))], {}, "parameter 0"),
    ([T((8,)), T((8,))], {}, "share memory"), ([T((8,)), T((8,), data=AT + 28)], {}, "share memory"),
    ([T((8,)), T((8,), data=AT + 32)], dict(norm=T((1,), data=AT + 60)), "share memory"), ([T((8,))], dict(norm=T((1,), data=AT)), "share memory"),
    ([T((4,), data=AT + 32), T((8,), data=AT + 64), T((4,), BFLOAT16, data=AT + 40)], {}, "share memory"),
])
def test_clip_refuses(L, grads, kw, match):  # noqa: F811
    clip_call(L, grads, **kw)
    refused(L, match)
