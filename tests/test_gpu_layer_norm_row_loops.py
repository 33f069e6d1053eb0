"""Layer norm over more rows than its workgroups take at once: each goes from row to row with others on their way, the
last ones of some and not of others, and keeps its columns' sums over all of them. The upstream gradients are eighths, so that fp32 holds every
sum of them: the bias's gradient is exact, and a row that is missed or counted twice shows in it."""
from __future__ import annotations

import numpy as np
import pytest

from block_cases import U, around, close, device, norm_exact, rounded, stored, values
from plast_amd.abi import KernelParams

pytestmark = pytest.mark.gpu
EPS = 1e-5

# Rows that 256 compute units take in one turn, forward and backward alike: 16384 of 16 lanes a row, 4096 of 64, 1024 of 256, 512 of 512, 256 of
# 1024; the rows end shortly behind the first, second and third turn, or in the midst of one.
SHAPES = [(16384 + 5, 33), (2 * 16384 + 9, 100), (3 * 16384 + 17, 60), (2 * 16384 + 8200, 64), (4096 + 3, 256), (2 * 4096 + 5, 300),
          (3 * 4096 + 1, 200), (4 * 1024 + 7, 511), (1024 + 1, 2048), (2 * 1024 + 3, 1500), (3 * 1024 + 700, 700), (4 * 1024, 1024),
          (512 + 1, 4096), (2 * 512 + 1, 3001), (3 * 512 + 5, 2500), (256 + 3, 8192), (2 * 256 + 3, 8191), (3 * 256 + 130, 5000),
          (256 + 3, 16384), (2 * 256 + 5, 16001), (3 * 256 + 1, 9000)]


def _eighths(rng, shape):
    return rng.randint(-24, 25, shape).astype(np.float32) / 8


def _case(shape, kind, seed):
    rng = np.random.RandomState(seed)
    x = rounded(rng.randn(*shape) * 1.5 + 0.5 + 3.0 * (rng.rand(shape[-1]) < 0.02), kind)
    w, b = (1 + 0.2 * rng.randn(shape[-1])).astype(np.float32), (0.3 * rng.randn(shape[-1])).astype(np.float32)
    return x, w, b, _eighths(rng, shape), rng


def _dw_tol(x, dy):
    """As norm_exact's, but with the additions that there are: a lane adds the rows of its turns, up to 5 here, the workgroup up to 32
    groups in halves, the last launch 512 workgroups in 64 turns of 8; or pieces of some ten rows, 64 turns of up to 512 pieces."""
    x = np.asarray(x, np.float64)
    mu = x.mean(1, keepdims=True)
    size = np.abs(x - mu).mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + EPS)
    add = (x.shape[1] / 64 + 48) * U
    off = (2 * U * np.abs(mu) + add * size) * r
    return (np.abs(dy * (x - mu) * r) * (add + 100 * U) + np.abs(dy) * off).sum(0)


def _check(shape, kind, add, pitch=0):
    from plast_amd.runtime import DeviceTensor, backward, forward
    print(f"layer norm loops {kind} {shape} add={add} pitch={pitch}", flush=True)
    x, w, b, dy, rng = _case(shape, kind, shape[1])
    want = norm_exact(x, w, b, np.float32(EPS), dy)
    dx0, dw0, db0 = rounded(rng.randn(*shape), kind), rng.randn(shape[1]).astype(np.float32), _eighths(rng, shape[1:])
    X = device(x, kind, 0, pitch, device(dx0, kind, 0, pitch))
    W, B = device(w, "f32", grad=device(dw0, "f32")), device(b, "f32", grad=device(db0, "f32"))
    Y = device(np.full(shape, 55.0), kind, 0, pitch, device(dy, kind, 0, pitch))
    S, p = DeviceTensor((shape[0], 2)), KernelParams(0, 0 if add else 1, EPS)
    forward("layer_norm", [X, W, B, S], Y, p)
    close(values(Y), want["y"], want["y_tol"] + stored(want["y"], kind), "y")
    assert (around(Y, kind) == rounded(77.0, kind)).all()
    backward("layer_norm", [X, W, B, S], Y, p)
    dx = want["dx"] + dx0 * add
    close(values(X.kept_grad), dx, want["dx_tol"] + stored(np.abs(dx) + np.abs(dx0) * add, kind), "dx")
    assert (around(X.kept_grad, kind) == rounded(77.0, kind)).all()
    assert np.array_equal(values(B.kept_grad), dy.sum(0, dtype=np.float64) + db0 * add)
    dw = want["dw"] + dw0 * add
    close(values(W.kept_grad), dw, _dw_tol(x, dy) + stored(np.abs(dw) + np.abs(dw0) * add, "f32"), "dw")


@pytest.mark.parametrize("kind, add", [("f32", False), ("f32", True), ("bf16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_in_turns(shape, kind, add):
    _check(shape, kind, add)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shape, pitch", [((2 * 16384 + 9, 50), 53), ((3 * 1024 + 1, 600), 700), ((2 * 256 + 3, 5001), 5003)])
def test_rows_in_turns_apart_from_each_other(shape, pitch, kind):
    _check(shape, kind, True, pitch)


@pytest.mark.parametrize("kind, shape", [("f32", (1000, 16400)), ("bf16", (1900, 16500))])
@pytest.mark.parametrize("add", [False, True])
def test_long_rows_in_pieces_of_more_than_eight(shape, kind, add):
    _check(shape, kind, add)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(16384 + 5, 33), (2 * 16384 + 9, 100), (3 * 4096 + 1, 200), (3 * 1024 + 70, 700), (2 * 1024 + 3, 1500),
                                   (2 * 512 + 1, 3001), (3 * 512 + 5, 4096), (2 * 256 + 3, 8191)])
def test_in_place_with_rows_on_their_way(shape, kind):
    from plast_amd.runtime import DeviceTensor, forward
    x, w, b, _, _ = _case(shape, kind, 11)
    X, S = device(x, kind), DeviceTensor((shape[0], 2))
    forward("layer_norm", [X, device(w, "f32"), device(b, "f32"), S], X, KernelParams(0, 0, EPS))
    want = norm_exact(x, w, b, np.float32(EPS))
    close(values(X), want["y"], want["y_tol"] + stored(want["y"], kind), "in place")


def test_replayed_with_other_work_between():
    """Captured passes over more rows than a turn's, replayed over other rows with eager work between."""
    from plast_amd import runtime as rt
    L = rt.lib()
    for shape, kind in (((2 * 4096 + 5, 300), "f32"), ((3 * 512 + 1, 2500), "bf16")):
        x, w, b, dy, _ = _case(shape, kind, 5)
        X, Y = device(x, kind, grad=device(np.zeros(shape), kind)), device(np.zeros(shape), kind, grad=device(dy, kind))
        W, B = (device(t, "f32", grad=device(np.zeros(shape[1]), "f32")) for t in (w, b))
        S, p = rt.DeviceTensor((shape[0], 2)), KernelParams(0, 1, EPS)
        outs = (Y, X.kept_grad, W.kept_grad, B.kept_grad)

        def call():
            rt.forward("layer_norm", [X, W, B, S], Y, p)
            rt.backward("layer_norm", [X, W, B, S], Y, p)
        call()
        assert L.plast_hip_capture_begin() == 0
        call()
        graph = L.plast_hip_capture_end()
        L.check("capture")
        for rep in range(3):
            img = device(rounded(x * (1 + rep), kind), kind)
            L.arena_memcpy_d2d_hip(X.ptr, img.ptr, x.size * X.itemsize)
            call()
            eager = [values(t) for t in outs]
            a = rt.DeviceTensor((1000, 1000)).fill_("normal", rep, 0.0, 1.0)
            rt.forward("sum", [a], rt.DeviceTensor((1000,)), KernelParams(0, 0, 0.0))
            for t in outs:
                L.zeros_hip(t.p, int(np.prod(t.shape)))
            assert L.plast_hip_graph_launch(graph) == 0
            for e, t in zip(eager, outs):
                assert np.array_equal(e, values(t)), (shape, rep)
        L.plast_hip_graph_destroy(graph)
