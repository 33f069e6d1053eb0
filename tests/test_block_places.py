"""Layer norm and the gated recurrence refuse results that share memory with what a call reads or else writes, on the CPU:
arguments are checked before the GPU is touched."""
from __future__ import annotations

import pytest

from plast_amd.runtime import LIB_PATH
from test_block_refusals import norm_call
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
