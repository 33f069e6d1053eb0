"""The Newton-Schulz orthogonalisation and the Muon step on the GPU against the iteration in 64 bits:
shapes on each side of the tiles, tall and wide, stacks, strides, types, rank-deficient and extreme
inputs, graph capture.

An iteration's products are summed in 32 bits from factors of 22 bits, so each step is off by some 2^-22
of the iterate's largest singular value (below 1.3), and a step multiplies what small singular directions
hold, errors too, by at most a = 3.4445. Relative to the result, whose singular values lie around 1: 2e-5
for a Gaussian matrix, whose singular values lie together; where they are far apart, the sum of 2^-21
a^k over five steps, 3.3e-4. Results of 16 bits are rounded once more, by half a step of theirs."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from plast_amd import abi
from plast_amd.abi import BFLOAT16, FLOAT16, FLOAT32
from token_cases import HALF_STEP, load, store

pytestmark = pytest.mark.gpu
KINDS = {"f32": FLOAT32, "f16": FLOAT16, "bf16": BFLOAT16}
A, B, CC, EPS = 3.4445, -4.7750, 2.0315, 1e-7


def _rt():
    from plast_amd import runtime
    return runtime


def iterate(g, steps=5, a=A, b=B, c=CC, eps=EPS):
    a, b, c, eps = (float(np.float32(v)) for v in (a, b, c, eps))
    x = g.astype(np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.linalg.norm(x) + eps)
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T if tall else x


def near(got, want, rel, kind, what):
    """In the Frobenius norm, with each value's rounding."""
    half, tiny = HALF_STEP[kind]
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)), f"{what}: infinities or NaN differ"
    err = np.linalg.norm((got.astype(np.float64) - want)[fine])
    bar = (rel + half) * np.linalg.norm(want[fine]) + tiny * np.sqrt(want.size)
    assert err <= bar, f"{what}: off by {err:.3g}, at most {bar:.3g}"


def run(stack, kind, steps=5, place=None, place_out=None, in_place=False, eps=EPS):
    """newton_schulz_hip over [count, rows, cols] (or one matrix); place: (strides, offset, elements)."""
    rt = _rt()
    L = rt.lib()
    raw = store(stack, kind)

    def tensor(place, values):
        if place is None:
            return rt.DeviceTensor.from_numpy(values)
        strides, offset, size = place
        buf = np.full(size, 9, raw.dtype)
        np.lib.stride_tricks.as_strided(buf[offset:], raw.shape, [s * buf.itemsize for s in strides])[...] = values
        base = rt.DeviceTensor.from_numpy(buf)
        return rt.DeviceTensor(raw.shape, KINDS[kind], base=base, offset=offset, strides=strides, zero=False)

    g = tensor(place, raw)
    out = g if in_place else tensor(place_out, np.full_like(raw, 7))
    r = abi.NewtonSchulz(A, B, CC, eps, steps)
    L.newton_schulz_hip(C.byref(g.t), C.byref(out.t), C.byref(r))
    L.check("newton_schulz")
    if not in_place:
        assert np.array_equal(g.numpy(), raw, equal_nan=raw.dtype != np.uint16), "the input was written"
    return load(out.numpy())


SHAPES = [(1, 1, 1), (1, 1, 7), (1, 7, 1), (2, 2, 3), (1, 16, 16), (3, 33, 65), (1, 64, 64), (2, 100, 300),
          (1, 300, 100), (2, 128, 128), (1, 129, 257), (3, 127, 255), (1, 256, 256), (1, 257, 1000),
          (2, 1000, 257), (5, 40, 1030), (1, 512, 640), (1, 520, 1300)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
def test_shapes(shape, kind):
    print(f"newton_schulz {kind} {shape}", flush=True)
    rng = np.random.RandomState(sum(shape))
    g = load(store((rng.randn(*shape) * 1e-3).astype(np.float32), kind))
    got = run(g, kind)
    for b in range(shape[0]):
        want = iterate(g[b])
        sv = np.linalg.svd(g[b].astype(np.float64), compute_uv=False)
        near(got[b], want, 2e-5 if sv[-1] > 0.05 * sv[0] else 3.3e-4, kind, f"{kind} {shape}[{b}]")


@pytest.mark.parametrize("shape", [(300, 700), (700, 300), (130, 130)])
def test_strong_directions_and_low_rank(shape):
    rng = np.random.RandomState(1)
    noise = rng.randn(*shape)
    strong = rng.randn(shape[0], 8) @ rng.randn(8, shape[1])
    for name, g in (("strong", noise + 3 * strong), ("low rank", strong), ("one", np.outer(noise[:, 0], noise[0]))):
        print(f"newton_schulz {name} {shape}", flush=True)
        g = g.astype(np.float32)
        near(run(g, "f32"), iterate(g), 3.3e-4, "f32", f"{name} {shape}")


@pytest.mark.parametrize("shape", [(1, 700, 3000), (1, 3000, 700), (2, 530, 2700), (1, 1030, 2100)])
def test_large(shape):
    """Sizes from which the products run in the largest tiles and two steps go at once, the strong directions
    of a gradient among them."""
    print(f"newton_schulz large {shape}", flush=True)
    rng = np.random.RandomState(7)
    g = rng.randn(*shape).astype(np.float32)
    g[0] += (rng.randn(shape[1], 8) @ rng.randn(8, shape[2])).astype(np.float32)
    for kind, steps in (("f32", 5), ("f32", 4), ("bf16", 5)):
        h = load(store(g, kind))
        got = run(h, kind, steps)
        for b in range(shape[0]):
            near(got[b], iterate(h[b], steps), 2e-5, kind, f"{kind} {shape}[{b}] {steps} steps")


@pytest.mark.parametrize("rule", [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (5.5, -12.0, 7.5)])
def test_other_rules(rule):
    """The last one takes singular values to 1e5 and is refused."""
    rt = _rt()
    rng = np.random.RandomState(8)
    g = rng.randn(1030, 2100).astype(np.float32)
    x = rt.DeviceTensor.from_numpy(g)
    out = rt.DeviceTensor(g.shape, zero=False)
    r = abi.NewtonSchulz(*rule, EPS, 4)
    rt.lib().newton_schulz_hip(C.byref(x.t), C.byref(out.t), C.byref(r))
    if rule[0] > 5:
        with pytest.raises(rt.PlastHipError, match="diverges"):
            rt.lib().check("newton_schulz")
        return
    rt.lib().check("newton_schulz")
    near(out.numpy(), iterate(g, 4, *rule), 2e-5, "f32", f"{rule}")


def test_steps_and_extremes():
    rng = np.random.RandomState(2)
    g = rng.randn(70, 90).astype(np.float32)
    for steps in (0, 1, 2, 7):
        near(run(g, "f32", steps), iterate(g, steps), 2e-5 * 2 ** max(0, steps - 5), "f32", f"{steps} steps")
    for scale in (1e-30, 1e-20, 1e18, 3e37):  # squares that leave 32 bits
        h = (g / np.abs(g).max() * scale).astype(np.float32)
        near(run(h, "f32"), iterate(h), 2e-5, "f32", f"scale {scale}")
    near(run(g, "f32", eps=100.0), iterate(g, eps=100.0), 2e-5, "f32", "eps")
    assert not run(np.zeros((2, 40, 50), np.float32), "f32").any(), "the zero matrix"
    one = np.zeros((40, 50), np.float32)
    one[3, 4] = 2.0
    near(run(one, "f32"), iterate(one), 2e-5, "f32", "a single entry")
    bad = np.stack([g, g, g])
    bad[1, 5, 6] = np.nan
    got = run(bad, "f32")
    assert np.isnan(got[1]).all() and np.array_equal(got[0], got[2]) and np.isfinite(got[0]).all()


@pytest.mark.parametrize("kind", list(KINDS))
def test_strides_and_in_place(kind):
    rng = np.random.RandomState(3)
    g = load(store(rng.randn(3, 70, 45).astype(np.float32), kind))
    want = np.stack([iterate(m) for m in g])
    places = [None, ((70 * 64, 64, 1), 0, 3 * 70 * 64), ((70 * 45, 1, 70), 0, 3 * 70 * 45),
              ((45, 3 * 45, 1), 5, 3 * 70 * 45 + 5), ((2, 6 * 45, 6), 1, 70 * 6 * 45 + 1)]
    for k, place in enumerate(places):
        out = places[(k + 2) % len(places)]
        print(f"newton_schulz {kind} strides {place} {out}", flush=True)
        near(run(g, kind, place=place, place_out=out), want, 2e-5, kind, f"{kind} {place}")
    near(run(g, kind, in_place=True), want, 2e-5, kind, f"{kind} in place")
    broadcast = np.broadcast_to(g[:1], g.shape)  # one matrix as a stack (stride 0)
    got = run(np.ascontiguousarray(broadcast), kind, place=((0, 45, 1), 0, 70 * 45))
    near(got, np.stack([want[0]] * 3), 2e-5, kind, "broadcast stack")


def muon_exact(p, g, m, lr, mom, decay, nesterov, steps=5):
    lr, mom, decay = (float(np.float32(v)) for v in (lr, mom, decay))
    m = mom * m + (1 - mom) * g
    u = (1 - mom) * g + mom * m if nesterov else m
    o = iterate(u, steps)
    rows, cols = p.shape
    return p * (1 - lr * decay) - lr * max(1.0, rows / cols) ** 0.5 * o, m


@pytest.mark.parametrize("nesterov", [0, 1])
@pytest.mark.parametrize("own_moments", [False, True])
def test_muon_steps(nesterov, own_moments):
    rt = _rt()
    L = rt.lib()
    rng = np.random.RandomState(4)
    shapes = [(64, 64), (100, 30), (64, 64), (30, 100), (1, 5), (257, 130), (64, 64), (0, 4), (9, 9)]
    lr, mom, decay = 0.02, 0.9, 0.1
    p0 = [rng.randn(*s).astype(np.float32) for s in shapes]
    dev = [rt.DeviceTensor.from_numpy(p, requires_grad=True) for p in p0]
    dev[8].t.grad = None                                   # no gradient: left alone
    slots = dev[:3] + [None] + dev[3:]
    arr = (abi.TensorP * len(slots))(*[C.pointer(d.t) if d is not None else None for d in slots])
    moments = [rt.DeviceTensor(d.shape if d is not None else (1, 1)) for d in slots]
    held, keep = abi.tensor_array(*[m.t for m in moments])
    opt = abi.Muon(lr, mom, decay, nesterov, abi.NewtonSchulz(A, B, CC, EPS, 5),
                   held if own_moments else None)
    want_p, want_m = [p.astype(np.float64) for p in p0], [np.zeros(s) for s in shapes]
    for step in range(3):
        for k, d in enumerate(dev[:8]):
            g = rng.randn(*shapes[k]).astype(np.float32)
            if g.size:
                L.arena_memcpy_h2d_hip(d.grad.ptr, g.ctypes.data, g.nbytes)
                want_p[k], want_m[k] = muon_exact(want_p[k], g, want_m[k], lr, mom, decay, nesterov)
        L.muon_step_hip(C.byref(opt), arr, len(slots))
        L.check("muon_step")
        for k, d in enumerate(dev):
            # a step's update is lr times a matrix of singular values around 1, off by 2e-5 of it (by
            # 3.3e-4 where the momentum's singular values lie far apart, as a square one's do); the
            # parameter rounds twice a step
            got = d.numpy().astype(np.float64)
            r = min(shapes[k])
            bar = (step + 1) * (lr * 3.3e-4 * 1.3 * np.sqrt(r * max(1, shapes[k][0] / max(1, shapes[k][1])))
                                + 2.0 ** -23 * np.linalg.norm(want_p[k])) + 1e-30
            assert np.linalg.norm(got - want_p[k]) <= bar, f"parameter {k} {shapes[k]}"
        where = opt.m if not own_moments else held
        for k, i in ((0, 0), (5, 6)):
            t = where[i].contents
            m = np.empty(shapes[k], np.float32)
            L.arena_memcpy_d2h_hip(m.ctypes.data, t.data, m.nbytes)
            assert np.abs(m - want_m[k]).max() <= 4 * 2.0 ** -23 * np.abs(want_m[k]).max()
    assert np.array_equal(dev[8].numpy(), p0[8])
    L.plast_hip_muon_release(C.byref(opt), len(slots))
    assert bool(opt.m) == own_moments                       # the caller's stay the caller's


def test_muon_refuses_moments_of_another_shape():
    rt = _rt()
    p, m = rt.DeviceTensor((8, 4), requires_grad=True), rt.DeviceTensor((4, 8))
    arr, keep = abi.tensor_array(p.t)
    held, keep_m = abi.tensor_array(m.t)
    opt = abi.Muon(0.02, 0.9, 0.0, 1, abi.NewtonSchulz(A, B, CC, EPS, 5), held)
    rt.lib().muon_step_hip(C.byref(opt), arr, 1)
    with pytest.raises(rt.PlastHipError, match="moment tensor of parameter 0"):
        rt.lib().check()


def test_captured_calls_replay():
    rt = _rt()
    L = rt.lib()
    rng = np.random.RandomState(5)
    shapes = [(200, 130), (130, 260), (200, 130)]
    G = rt.DeviceTensor.from_numpy(rng.randn(2, 96, 160).astype(np.float32))
    O = rt.DeviceTensor(G.shape, zero=False)
    r = abi.NewtonSchulz(A, B, CC, EPS, 5)
    dev = [rt.DeviceTensor.from_numpy(rng.randn(*s).astype(np.float32), requires_grad=True) for s in shapes]
    moments = [rt.DeviceTensor(s) for s in shapes]
    ptrs, keep = abi.tensor_array(*[d.t for d in dev])
    held, keep_m = abi.tensor_array(*[m.t for m in moments])
    opt = abi.Muon(0.02, 0.9, 0.1, 1, r, held)

    def call():
        L.newton_schulz_hip(C.byref(G.t), C.byref(O.t), C.byref(r))
        L.muon_step_hip(C.byref(opt), ptrs, len(dev))

    def load_state(seed):
        q = np.random.RandomState(seed)
        for t in [G] + dev + moments + [d.grad for d in dev]:
            a = q.randn(*t.shape).astype(np.float32)
            L.arena_memcpy_h2d_hip(t.ptr, a.ctypes.data, a.nbytes)

    def results():
        return [t.numpy() for t in [O] + dev + moments]

    call()
    L.check("eager")
    assert L.plast_hip_capture_begin() == 0
    try:
        call()
    finally:
        graph = L.plast_hip_capture_end()
    L.check("capture")
    assert graph
    try:
        for k in range(4):
            load_state(k)
            assert L.plast_hip_graph_launch(graph) == 0
            got = results()
            load_state(k)
            call()
            for a, b in zip(got, results()):
                assert np.array_equal(a, b), f"replay {k} differs from the eager call"
            near(got[0][1], iterate(np.random.RandomState(k).randn(2, 96, 160).astype(np.float32)[1]), 2e-5,
                 "f32", f"replay {k}")
    finally:
        L.plast_hip_graph_destroy(graph)


def test_ops_wrapper():
    from plast_amd import ops
    rng = np.random.RandomState(6)
    g = rng.randn(31, 50).astype(np.float32)
    got = ops.newton_schulz(_rt().DeviceTensor.from_numpy(g)).numpy()
    near(got, iterate(g), 2e-5, "f32", "ops")
