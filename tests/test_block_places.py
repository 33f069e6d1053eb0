"""Layer norm and the gated recurrence refuse results that share memory with what a call reads or else writes, on the CPU:
arguments are checked before the GPU is touched."""
from __future__ import annotations

import pytest

from plast_amd.abi import FLOAT32, INT32
from plast_amd.runtime import LIB_PATH
from test_block_refusals import norm_call, scan_call
from test_operator_refusals import AT, L, T, refused  # noqa: F401

pytestmark = pytest.mark.skipif(not LIB_PATH.exists(), reason="the library is not built")
FAR = 1 << 16


def norm(**at):
    """Tensors of a call of 6 rows of 10, each in a place of its own but those that are given."""
    places = {n: AT + FAR * k for k, n in enumerate(("x", "w", "b", "stats", "y", "dx", "dw", "db", "dy"))}
    places.update(at)
    shape = {"x": (6, 10), "stats": (6, 2), "y": (6, 10), "dx": (6, 10), "dy": (6, 10)}
    made = {n: T(shape.get(n, (10,)), data=p) if isinstance(p, int) else p for n, p in places.items()}
    ins = {n: T(shape.get(n, (10,)), data=made[n].data, strides=tuple(made[n].strides[:made[n].ndim]), grad=made["d" + n]) for n in "xwb"}
    return dict(ins, stats=made["stats"], out=T((6, 10), data=made["y"].data, strides=tuple(made["y"].strides[:2]), grad=made["dy"]))


@pytest.mark.parametrize("at, match", [
    (dict(y=AT + 40), "the output shares memory with x"), (dict(y=AT - 4), "the output shares memory with x"),
    (dict(y=AT + 236), "the output shares memory with x"),
    (dict(y=T((6, 10), strides=(20, 1), data=AT + 36), x=T((6, 10), strides=(20, 1))), "the output shares memory with x"),
    (dict(y=AT + FAR), "the output shares memory with weight"), (dict(y=AT + 2 * FAR + 36), "the output shares memory with bias"),
    (dict(y=AT + 3 * FAR - 4), "the output shares memory with stats"), (dict(stats=AT + 8), "stats shares memory with x"),
    (dict(stats=AT + FAR - 8), "stats shares memory with weight"), (dict(stats=AT + 2 * FAR), "stats shares memory with bias"),
])
def test_layer_norm(L, at, match):  # noqa: F811
    norm_call(L, **norm(**at))
    refused(L, match)


@pytest.mark.parametrize("at, match", [
    (dict(dx=AT + 40), "the gradient of x shares memory with x"), (dict(dx=AT + 8 * FAR + 40), "the gradient of x shares memory with the output's"),
    (dict(dx=T((6, 10), strides=(20, 1), data=AT + 36), x=T((6, 10), strides=(20, 1))), "the gradient of x shares memory with x"),
    (dict(dx=AT + FAR + 4), "the gradient of x shares memory with weight"), (dict(dx=AT + 3 * FAR), "the gradient of x shares memory with stats"),
    (dict(dx=AT + 6 * FAR), "the gradient of x shares memory with the gradient of weight"),
    (dict(db=AT + 5 * FAR + 100), "the gradient of x shares memory with the gradient of bias"),
    (dict(db=AT + 6 * FAR + 36), "the gradient of weight shares memory with the gradient of bias"),
])
def test_layer_norm_backward(L, at, match):  # noqa: F811
    norm_call(L, "backward", **norm(**at))
    refused(L, match)


NAMES = ("f", "v", "initial", "lengths", "last", "states", "h", "df", "dv", "dinitial", "dlast", "dh")
SEQ, STATE, CHUNKS = (3, 200, 5), (3, 5), (3, 4, 5)
SIZE, STATE_SIZE = 4 * 3 * 200 * 5, 4 * 3 * 5


def scan(**at):
    """Tensors of a call of 3 sequences of 200 steps of 5 channels, each in a place of its own but those that are given."""
    shape = {"f": SEQ, "v": SEQ, "h": SEQ, "df": SEQ, "dv": SEQ, "dh": SEQ, "states": CHUNKS, "lengths": (3,)}
    places = {n: place(n) for n in NAMES}
    places.update(at)
    made = {n: T(shape.get(n, STATE), INT32 if n == "lengths" else FLOAT32, data=p) if isinstance(p, int) else p for n, p in places.items()}

    def with_grad(n):
        t = made[n]
        return T(tuple(t.shape[:t.ndim]), strides=tuple(t.strides[:t.ndim]), data=t.data, grad=made["d" + n])
    return dict({n: with_grad(n) for n in ("f", "v", "initial", "last")}, lengths=made["lengths"], states=made["states"], out=with_grad("h"))


def place(name):
    return AT + FAR * NAMES.index(name)


def interleaved(k, width=10, by=0):
    """The k-th part of 5 channels of steps of `width`, `by` elements on."""
    return T(SEQ, strides=(200 * width, width, 1), data=AT + 4 * (5 * k + by))


@pytest.mark.parametrize("at, match", [
    (dict(h=place("v") + 20), "the output shares memory with v"), (dict(h=place("f") + SIZE - 4), "the output shares memory with f"),
    (dict(f=interleaved(0), h=interleaved(1, by=-1)), "the output shares memory with f"),
    (dict(v=interleaved(1), h=interleaved(0, by=1), f=AT + 12 * FAR), "the output shares memory with v"),
    (dict(h=place("initial") + STATE_SIZE - 4), "the output shares memory with the initial"), (dict(h=place("last")), "the output shares memory with the last"),
    (dict(h=place("states") + 16), "the output shares memory with states"), (dict(h=place("lengths") - 4), "the output shares memory with lengths"),
    (dict(last=place("initial") + 4), "the last state shares memory with the initial"), (dict(last=place("initial") - 4), "the last state shares memory with the initial"),
    (dict(last=place("f")), "the last state shares memory with f"), (dict(last=place("v") + SIZE - 4), "the last state shares memory with v"),
    (dict(last=place("states") + 60), "the last state shares memory with states"), (dict(last=place("lengths") + 8), "the last state shares memory with lengths"),
    (dict(states=place("f")), "states shares memory with f"), (dict(states=place("v") + 40), "states shares memory with v"),
    (dict(states=place("initial")), "states shares memory with the initial"), (dict(states=place("lengths") + 4), "states shares memory with lengths"),
])
def test_recurrence(L, at, match):  # noqa: F811
    scan_call(L, **scan(**at))
    refused(L, match)


@pytest.mark.parametrize("at, match", [
    (dict(df=place("dh") + 20), "the gradient of f shares memory with the output's gradient"),
    (dict(dv=place("f") + 20), "the gradient of v shares memory with f"), (dict(df=place("v") - 4), "the gradient of f shares memory with v"),
    (dict(df=interleaved(0), dv=interleaved(1, by=-1), f=place("dinitial") + FAR * 9), "the gradient of f shares memory with the gradient of v"),
    (dict(dh=interleaved(0), dv=interleaved(1, by=-1), f=place("dinitial") + FAR * 9), "the gradient of v shares memory with the output's gradient"),
    (dict(dinitial=place("dlast") + 4), "the initial state's gradient shares memory with the last state's gradient"),
    (dict(dinitial=place("states") + 4), "the initial state's gradient shares memory with states"),
    (dict(dinitial=place("df") + 4), "the gradient of f shares memory with the initial state's gradient"),
    (dict(dv=place("dinitial")), "the gradient of v shares memory with the initial state's gradient"),
    (dict(df=place("states")), "the gradient of f shares memory with states"), (dict(dv=place("dlast") - 8), "the gradient of v shares memory with the last"),
    (dict(df=place("lengths") - 8), "the gradient of f shares memory with lengths"),
])
def test_recurrence_backward(L, at, match):  # noqa: F811
    scan_call(L, "backward", **scan(**at))
    refused(L, match)
