"""Layer norm and its gradients against the formulas in 64 bits, with tolerances that count fp32's roundings and the
result's own (block_cases.py)."""
from __future__ import annotations

import numpy as np
import pytest

from block_cases import around, close, device, norm_exact, rounded, stored, values
from plast_amd.abi import FLOAT32, KernelParams

pytestmark = pytest.mark.gpu
EPS = 1e-5

# rows of a lane, of a wave, of a workgroup, of several passes; one column; odd ones; one row; none
SHAPES = [(1, 1), (3, 1), (5, 2), (7, 3), (33, 18), (70, 31), (64, 64), (9, 65), (40, 127), (300, 128), (3, 255),
          (11, 256), (2, 3, 257), (17, 500), (4, 5, 1000), (129, 333), (20, 1024), (6, 1031), (1500, 40), (5, 2048), (9, 2500),
          (600, 512), (3, 4096), (37, 4100), (2, 2, 8192), (5, 9001), (3, 16384), (2, 16390), (4, 20000), (2, 40001), (1, 70001)]


def _case(shape, kind, seed, offset=0.5):
    rng = np.random.RandomState(seed)
    x = rounded(rng.randn(*shape) * 1.5 + offset + 3.0 * (rng.rand(shape[-1]) < 0.02), kind)
    w, b = (1 + 0.2 * rng.randn(shape[-1])).astype(np.float32), (0.3 * rng.randn(shape[-1])).astype(np.float32)
    return x, w, b, rounded(rng.randn(*shape), kind)


def _check(shape, kind, add, lead=0, pitch=0, seed=None, offset=0.5, wanted=(1, 1, 1)):
    """The forward pass and the backward pass of one call, into gradients that hold something already."""
    from plast_amd.runtime import DeviceTensor, backward, forward
    print(f"layer norm {kind} {shape} add={add} lead={lead} pitch={pitch}", flush=True)
    x, w, b, dy = _case(shape, kind, len(shape) + shape[-1] if seed is None else seed, offset)
    width, rows = shape[-1], int(np.prod(shape[:-1]))
    want = norm_exact(x.reshape(rows, width), w, b, np.float32(EPS), dy.reshape(rows, width))
    rng = np.random.RandomState(1)
    dx0, dw0, db0 = rounded(rng.randn(*shape), kind), rng.randn(width).astype(np.float32), rng.randn(width).astype(np.float32)
    X = device(x, kind, lead, pitch, device(dx0, kind, lead, pitch))
    W, B = device(w, "f32", lead, 0, device(dw0, "f32")), device(b, "f32", lead, 0, device(db0, "f32"))
    for t, wants in zip((X, W, B), wanted):
        t.t.requires_grad = bool(wants)
    Y = device(np.full(shape, 55.0), kind, lead, pitch, device(dy, kind, lead, pitch))
    S = DeviceTensor(shape[:-1] + (2,), FLOAT32)
    p = KernelParams(0, 0 if add else 1, EPS)
    forward("layer_norm", [X, W, B, S], Y, p)
    y = want["y"].reshape(shape)
    close(values(Y), y, want["y_tol"].reshape(shape) + stored(y, kind), "y")
    assert (around(Y, kind) == rounded(77.0, kind)).all()
    backward("layer_norm", [X, W, B, S], Y, p)
    for got, name, old, k, wants in ((X, "dx", dx0, kind, wanted[0]), (W, "dw", dw0, "f32", wanted[1]),
                                     (B, "db", db0, "f32", wanted[2])):
        ref, tol = want[name].reshape(old.shape), want[name + "_tol"].reshape(old.shape)
        if add:
            ref = ref + old
        if not wants:
            ref, tol = old, 0.0
        close(values(got.kept_grad), ref, tol + stored(np.abs(ref) + np.abs(old) * add, k), name)
        assert (around(got.kept_grad, k) == rounded(77.0, k)).all(), name
    return X, W, B, S, Y


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, kind):
    _check(shape, kind, add=(sum(shape) % 2 == 0))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape, lead, pitch", [((50, 100), 1, 0), ((50, 100), 0, 101), ((3, 7, 64), 3, 200), ((20, 1000), 5, 1003),
                                                ((9, 4096), 1, 4099), ((3, 20000), 7, 20011), ((6, 1), 0, 3)])
@pytest.mark.parametrize("add", [False, True])
def test_strides(shape, lead, pitch, kind, add):
    _check(shape, kind, add, lead, pitch)


@pytest.mark.parametrize("shape", [(40, 300), (6, 4096), (3, 20000)])
@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 0), (0, 0, 0)])
def test_only_what_is_wanted(shape, wanted):
    for add in (False, True):
        _check(shape, "f32", add, wanted=wanted)


@pytest.mark.parametrize("kind, offset", [("f32", 1000.0), ("f32", -3.0e4), ("f16", 100.0), ("bf16", 64.0)])
@pytest.mark.parametrize("shape", [(20, 100), (5, 4096), (3, 20000)])
def test_rows_far_from_zero(shape, kind, offset):
    _check(shape, kind, False, offset=offset)


def test_values_that_are_no_numbers_stay_in_their_rows():
    from plast_amd.runtime import DeviceTensor, forward
    for width in (5, 300, 5000, 40000):
        x = np.random.RandomState(0).randn(7, width).astype(np.float32)
        x[1, width // 2], x[3, 0], x[5, width - 1] = np.nan, np.inf, -np.inf
        X, W, B = device(x, "f32"), device(np.ones(width), "f32"), device(np.zeros(width), "f32")
        Y, S = DeviceTensor((7, width)), DeviceTensor((7, 2))
        forward("layer_norm", [X, W, B, S], Y, KernelParams(0, 0, EPS))
        bad = np.isnan(Y.numpy())
        assert bad[[1, 3, 5]].all() and not bad[[0, 2, 4, 6]].any(), width


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(3000, 100), (40, 333), (700, 4096), (9, 20000), (3, 140000)])
def test_in_place(shape, kind):
    from plast_amd.runtime import DeviceTensor, forward
    x, w, b, _ = _case(shape, kind, 11)
    X, S = device(x, kind), DeviceTensor((shape[0], 2))
    forward("layer_norm", [X, device(w, "f32"), device(b, "f32"), S], X, KernelParams(0, 0, EPS))
    want = norm_exact(x, w, b, np.float32(EPS))
    close(values(X), want["y"], want["y_tol"] + stored(want["y"], kind), "in place")


def test_equal_values():
    """Rows of one value: the differences are exactly 0 where the mean of equal values is exact, the bias is left."""
    from plast_amd.runtime import DeviceTensor, backward, forward
    for width in (1, 64, 1024, 32768):
        b = np.arange(width, dtype=np.float32)
        X = device(np.full((4, width), 0.75), "f32", grad=device(np.zeros((4, width)), "f32"))
        W, B = device(np.ones(width), "f32"), device(b, "f32")
        Y, S = device(np.zeros((4, width)), "f32", grad=device(np.ones((4, width)), "f32")), DeviceTensor((4, 2))
        forward("layer_norm", [X, W, B, S], Y, KernelParams(0, 0, EPS))
        assert np.array_equal(values(Y), np.tile(b, (4, 1)))
        backward("layer_norm", [X, W, B, S], Y, KernelParams(0, 1, EPS))
        assert not values(X.kept_grad).any()


def test_no_rows():
    from plast_amd.runtime import DeviceTensor, backward, forward
    dw, db = device(np.ones(8), "f32"), device(np.ones(8), "f32")
    X, W, B = DeviceTensor((0, 8)), device(np.ones(8), "f32", grad=dw), device(np.ones(8), "f32", grad=db)
    Y, S = DeviceTensor((0, 8), requires_grad=True), DeviceTensor((0, 2))
    forward("layer_norm", [X, W, B, S], Y, KernelParams(0, 0, EPS))
    backward("layer_norm", [X, W, B, S], Y, KernelParams(0, 0, EPS))
    assert (values(dw) == 1).all() and (values(db) == 1).all()
    backward("layer_norm", [X, W, B, S], Y, KernelParams(0, 1, EPS))
    assert not values(dw).any() and not values(db).any()


def test_overlapping_rows_are_read():
    """Windows of one buffer, each a step of 3 behind the one before."""
    from plast_amd.runtime import DeviceTensor, forward
    buf = np.random.RandomState(2).randn(400).astype(np.float32)
    base = DeviceTensor.from_numpy(buf)
    X = DeviceTensor((50, 200), FLOAT32, base=base, strides=(3, 1))
    w, b = np.ones(200, np.float32), np.zeros(200, np.float32)
    Y, S = DeviceTensor((50, 200)), DeviceTensor((50, 2))
    forward("layer_norm", [X, device(w, "f32"), device(b, "f32"), S], Y, KernelParams(0, 0, EPS))
    want = norm_exact(np.lib.stride_tricks.sliding_window_view(buf, 200)[:150:3], w, b, np.float32(EPS))
    close(Y.numpy(), want["y"], want["y_tol"] + stored(want["y"], "f32"), "windows")


def test_the_gradient_against_differences():
    """sum(y c) moved by the weight, the bias and x: central differences of the forward pass itself in fp32. A step of 2^-6
    leaves a third-order rest of its square; the sums' rounding is divided by the step."""
    from plast_amd.runtime import DeviceTensor, backward, forward
    rng = np.random.RandomState(3)
    x, w, b, c = (rng.randn(*s).astype(np.float32) for s in ((4, 24), (24,), (24,), (4, 24)))

    def total(x, w, b):
        Y = DeviceTensor((4, 24))
        forward("layer_norm", [device(x, "f32"), device(w, "f32"), device(b, "f32"), DeviceTensor((4, 2))], Y,
                KernelParams(0, 0, EPS))
        return float((Y.numpy().astype(np.float64) * c).sum())
    grads = [device(np.zeros(t.shape), "f32") for t in (x, w, b)]
    ins = [device(t, "f32", grad=g) for t, g in zip((x, w, b), grads)] + [DeviceTensor((4, 2))]
    Y = device(np.zeros((4, 24)), "f32", grad=device(c, "f32"))
    forward("layer_norm", ins, Y, KernelParams(0, 0, EPS))
    backward("layer_norm", ins, Y, KernelParams(0, 0, EPS))
    step = 2.0 ** -6
    for k, t in enumerate((x, w, b)):
        for i in rng.choice(t.size, 12, replace=False):
            moved = []
            for sign in (1, -1):
                args = [x.copy(), w.copy(), b.copy()]
                args[k].reshape(-1)[i] += sign * step
                moved.append(total(*args))
            slope = (moved[0] - moved[1]) / (2 * step)
            assert abs(slope - values(grads[k]).reshape(-1)[i]) < 40 * step ** 2 + 96 * 8 * 2.0 ** -24 / step, (k, i)


def test_same_bits_every_time():
    for shape in ((3000, 100), (500, 4096), (40, 20000)):
        runs = [_check(shape, "bf16", False, seed=4) for _ in range(2)]
        for a, b in zip(*[[values(t.kept_grad) for t in r[:3]] for r in runs]):
            assert np.array_equal(a, b)


def test_replayed_with_other_work_between():
    """A captured forward and backward pass, replayed with eager work of the library and of its own between replays."""
    from plast_amd import runtime as rt
    L = rt.lib()
    for shape, kind in (((300, 1000), "f32"), ((64, 4096), "bf16"), ((5, 20000), "f16")):
        x, w, b, dy = _case(shape, kind, 5)
        width = shape[-1]
        X = device(x, kind, grad=device(np.zeros(shape), kind))
        W, B = (device(t, "f32", grad=device(np.zeros(width), "f32")) for t in (w, b))
        Y, S = device(np.zeros(shape), kind, grad=device(dy, kind)), rt.DeviceTensor(shape[:-1] + (2,))
        outs = (Y, X.kept_grad, W.kept_grad, B.kept_grad)

        def call():
            rt.forward("layer_norm", [X, W, B, S], Y, KernelParams(0, 1, EPS))
            rt.backward("layer_norm", [X, W, B, S], Y, KernelParams(0, 1, EPS))
        call()
        assert L.plast_hip_capture_begin() == 0
        call()
        graph = L.plast_hip_capture_end()
        L.check("capture")
        for rep in range(3):
            new = rounded(x * (1 + rep), kind)
            img = device(new, kind)
            L.arena_memcpy_d2d_hip(X.ptr, img.ptr, int(np.prod(shape)) * X.itemsize)
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


def test_functional_form():
    from plast_amd import ops
    x, w, b, dy = _case((6, 50), "f32", 8)
    X = device(x, "f32", grad=device(np.zeros((6, 50)), "f32"))
    W, B = (device(t, "f32", grad=device(np.zeros(50), "f32")) for t in (w, b))
    inputs, y, p = ops.layer_norm(X, W, B, EPS, requires_grad=True)
    want = norm_exact(x, w, b, np.float32(EPS), dy)
    close(y.numpy(), want["y"], want["y_tol"] + stored(want["y"], "f32"), "y")
    keep = device(dy, "f32")
    y.t.grad = keep.p
    ops.backward("layer_norm", inputs, y, p)
    for t, name in ((X, "dx"), (W, "dw"), (B, "db")):
        close(values(t.kept_grad), want[name], want[name + "_tol"] + stored(want[name], "f32"), name)
