"""The gated linear recurrence and its gradients against the formulas in 64 bits, step by step, with tolerances that count
fp32's roundings and the result's own (block_cases.py)."""
from __future__ import annotations

import numpy as np
import pytest

from block_cases import around, close, device, give, rounded, scan_exact, scan_inputs, stored, values
from plast_amd import abi
from plast_amd.abi import FLOAT32, KernelParams

pytestmark = pytest.mark.gpu
CHUNK = abi.RECURRENCE_CHUNK

# one step, a few, around a chunk, several chunks; one channel, around a workgroup's columns, odd ones
SHAPES = [(1, 1, 1), (3, 1, 5), (2, 1, 64), (300, 1, 7), (5, 2, 33), (2, 7, 65), (3, 16, 4), (2, 17, 130), (1, 40, 1003), (2, 100, 66),
          (1, 127, 3), (2, 128, 64), (3, 129, 5), (70, 130, 6), (1, 256, 128), (2, 257, 63), (1, 500, 515), (3, 1000, 20),
          (1, 3001, 2), (2, 2050, 70), (33, 300, 1), (1, 63, 127), (2, 64, 128),
          (2, 65, 129), (8, 192, 130), (130, 140, 5), (1, 6400, 3), (1, 8300, 130), (2, 9001, 33), (600, 70, 3)]


class Scan:
    """The tensors of one call: sequences `lead` elements into their buffers, steps `pitch` apart."""

    def __init__(self, f, v, initial, lengths, kind, dy=None, dlast=None, lead=0, pitch=0, old=None):
        from plast_amd.runtime import DeviceTensor
        B, T, D = f.shape
        self.kind, self.shape = kind, f.shape
        self.old = {k: np.zeros(s, np.float32) for k, s in (("df", f.shape), ("dv", f.shape), ("dinitial", (B, D)))}
        if old is not None:
            self.old = {k: rounded(old.randn(*t.shape), kind if t.ndim == 3 else "f32") for k, t in self.old.items()}
        self.f = device(f, kind, lead, pitch, device(self.old["df"], kind, lead, pitch))
        self.v = device(v, kind, lead, pitch, device(self.old["dv"], kind, lead, pitch))
        self.initial = device(initial, "f32", grad=device(self.old["dinitial"], "f32"))
        self.lengths = DeviceTensor.from_numpy(np.asarray(lengths, np.int32))
        self.last = device(np.full((B, D), 55.0), "f32")
        self.states = DeviceTensor((B, -(-T // CHUNK), D), FLOAT32)
        self.h = device(np.full(f.shape, 55.0), kind, lead, pitch)
        if dy is not None:
            give(self.h, device(dy, kind, lead, pitch))
        if dlast is not None:
            give(self.last, device(dlast, "f32"))
        self.ins = [self.f, self.v, self.initial, self.lengths, self.last, self.states]

    def forward(self, keep=True):
        from plast_amd.runtime import forward
        forward("gated_recurrence", self.ins if keep else self.ins[:5], self.h, KernelParams(int(keep), 0, 0.0))

    def backward(self, add=False):
        from plast_amd.runtime import backward
        backward("gated_recurrence", self.ins, self.h, KernelParams(1, 0 if add else 1, 0.0))

    def check_forward(self, want, what):
        close(values(self.h), want["h"], want["h_tol"] + stored(want["h"], self.kind), f"{what} h")
        close(values(self.last), want["last"], want["last_tol"] + stored(want["last"], "f32"), f"{what} last")
        assert (around(self.h, self.kind) == rounded(77.0, self.kind)).all()

    def check_backward(self, want, what, add=False):
        for t, name in ((self.f, "df"), (self.v, "dv"), (self.initial, "dinitial")):
            kind = self.kind if name != "dinitial" else "f32"
            old = self.old[name] if add else 0.0 * self.old[name]
            ref = want[name] + old
            if not t.t.requires_grad:
                ref, tol = self.old[name], 0.0
            else:
                tol = want[name + "_tol"] + stored(np.abs(ref) + np.abs(old), kind)
            close(values(t.kept_grad), ref, tol, f"{what} {name}")
            assert (around(t.kept_grad, kind) == rounded(77.0, kind)).all(), name


def _data(shape, kind, seed, keep=(-2.0, 5.0), ragged=False):
    rng = np.random.RandomState(seed)
    B, T, D = shape
    f, v = scan_inputs(rng, shape, kind, keep)
    lengths = rng.randint(0, T + 1, B) if ragged else np.full(B, T)
    return (f, v, rng.randn(B, D).astype(np.float32), lengths, rounded(rng.randn(*shape), kind),
            rng.randn(B, D).astype(np.float32))


def _check(shape, kind, add=False, lead=0, pitch=0, ragged=False, keep=(-2.0, 5.0), edit=None, upstream="both", seed=None):
    what = f"{kind} {shape} add={add} lead={lead} pitch={pitch} ragged={ragged}"
    print("recurrence", what, flush=True)
    f, v, initial, lengths, dy, dlast = _data(shape, kind, sum(shape) if seed is None else seed, keep, ragged)
    if edit is not None:
        edit(f, v, initial, lengths)
    dy, dlast = (dy if upstream in ("both", "h") else None), (dlast if upstream in ("both", "last") else None)
    want = scan_exact(f, v, initial, lengths, dy, np.zeros_like(initial) if dlast is None else dlast)
    s = Scan(f, v, initial, lengths, kind, dy, dlast, lead, pitch, np.random.RandomState(9))
    s.forward(keep=False)
    s.check_forward(want, "serving " + what)
    for t in (s.h, s.last):
        t.buffer.t.grad = None
    s.forward()
    s.check_forward(want, what)
    s.backward(add)
    s.check_backward(want, what, add)
    return s


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, kind):
    _check(shape, kind, add=sum(shape) % 2 == 0)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [3, 4, 5, 6, 7, 63, 65, 66, 67, 68, 69, 129, 131, 133, 191, 193])
def test_ends_of_rows(width, kind):
    """Whole tiles of steps whose channels end inside a tile, or a few channels into one."""
    _check((2, 520, width), kind, lead=1, pitch=width + 3)
    _check((2, 520, width), kind, add=True, seed=3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("width", [6, 69, 131])
@pytest.mark.parametrize("channel", [-1, -3, -5])
def test_what_is_not_finite_near_the_end_of_rows_stays_in_its_channel(channel, width, kind):
    f, v, initial, lengths, dy, dlast = _data((2, 520, width), kind, 4)
    results = []
    for bad in (False, True):
        if bad:
            f, v, dy = f.copy(), v.copy(), dy.copy()
            f[:, 7, channel], v[:, 9, channel], dy[:, 11, channel] = np.nan, np.inf, -np.inf
        s = Scan(f, v, initial, lengths, kind, dy, dlast)
        s.forward()
        s.backward()
        results.append([np.delete(values(t), width + channel, axis=-1) for t in (s.h, s.last, s.f.kept_grad, s.v.kept_grad,
                                                                                 s.initial.kept_grad)])
    for clean, beside in zip(*results):
        assert np.isfinite(clean).all() and (clean == beside).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(5, 1, 70), (6, 9, 40), (7, 200, 65), (20, 400, 12), (4, 1500, 130)])
def test_ragged(shape, kind):
    _check(shape, kind, ragged=True)
    _check(shape, kind, ragged=True, add=True, seed=1)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shape, lead, pitch", [((2, 1, 20), 1, 41), ((3, 150, 64), 3, 64), ((2, 300, 63), 1, 127), ((2, 140, 128), 0, 384),
                                                ((1, 20, 5), 7, 6)])
@pytest.mark.parametrize("add", [False, True])
def test_strides(shape, lead, pitch, kind, add):
    _check(shape, kind, add, lead, pitch)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("keep", [(-30.0, -10.0), (8.0, 20.0), (-90.0, 90.0)])
def test_gates_far_out(keep, kind):
    """Channels that forget at once, that remember for millions of steps, and gates next to and beyond fp32's range."""
    _check((2, 700, 66), kind, keep=keep)


def test_lengths_beyond_the_range():
    """Negative lengths count as 0, those beyond T as T."""
    def edit(f, v, initial, lengths):
        lengths[:] = [-5, 0, 10 ** 9, 200, 2 ** 31 - 1]
    _check((5, 200, 30), "f32", edit=edit)
    _check((5, 1, 30), "f32", edit=edit)


@pytest.mark.parametrize("upstream", ["h", "last", "none"])
def test_upstream_gradients_that_are_not_there(upstream):
    _check((3, 260, 40), "f32", ragged=True, upstream=upstream)
    _check((3, 260, 40), "f32", add=True, upstream=upstream)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_padding_is_not_looked_at(kind):
    def edit(f, v, initial, lengths):
        for b, n in enumerate(lengths):
            f[b, n:], v[b, n:] = np.nan, np.inf
    for shape in ((6, 300, 40), (9, 1, 5), (5, 128, 64), (4, 1000, 10)):
        _check(shape, kind, ragged=True, edit=edit)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_closed_and_open_gates_select(kind):
    """-inf starts a sequence anew whatever the state was, NaN too; +inf holds the state whatever the value is."""
    def edit(f, v, initial, lengths):
        T = f.shape[1]
        rng = np.random.RandomState(3)
        initial[0] = np.nan
        f[0, 0] = -np.inf
        for b in range(f.shape[0]):
            for t in rng.choice(T, max(1, T // 7), replace=False):
                f[b, t] = -np.inf
                if t:
                    v[b, t - 1] = np.nan      # the state just before is NaN
                    f[b, t - 1] = 0.0
            for t in rng.choice(T, max(1, T // 7), replace=False):
                if np.isfinite(v[b, t]).all() and np.isfinite(f[b, t]).all():
                    f[b, t], v[b, t] = np.inf, np.nan
    for shape in ((2, 1, 9), (2, 60, 33), (2, 300, 70), (1, 900, 10)):
        print("selecting gates", kind, shape, flush=True)
        f, v, initial, lengths, _, _ = _data(shape, kind, 5)
        edit(f, v, initial, lengths)
        want = scan_exact(f, v, initial, lengths)
        s = Scan(f, v, initial, lengths, kind)
        s.forward()
        got = values(s.h)
        bad = ~np.isfinite(want["h"])
        assert not np.isfinite(got[bad]).any()
        close(got[~bad], want["h"][~bad], (want["h_tol"] + stored(want["h"], kind))[~bad], "h")


def test_gradients_stop_at_selecting_gates():
    """No gradient passes a start, and none reaches what a held state does not look at, NaN there or not."""
    shape = (2, 300, 40)
    f, v, initial, lengths, dy, dlast = _data(shape, "f32", 6)
    f[:, 100], f[:, 200:210], v[:, 200:210] = -np.inf, np.inf, np.nan
    dy[:, :100] = 0.0
    want = scan_exact(f, v, initial, lengths, dy, dlast)
    s = Scan(f, v, initial, lengths, "f32", dy, dlast)
    s.forward()
    s.backward()
    s.check_backward(want, "selecting")
    assert not values(s.v.kept_grad)[:, :100].any() and not values(s.v.kept_grad)[:, 200:210].any()
    assert not values(s.f.kept_grad)[:, 100].any() and not values(s.initial.kept_grad).any()


def test_not_a_number_spreads_along_its_channel_only():
    f, v, initial, lengths, _, _ = _data((2, 400, 70), "f32", 7)
    v[1, 250, 33], f[0, 140, 2] = np.nan, np.nan
    s = Scan(f, v, initial, lengths, "f32")
    s.forward()
    bad = np.isnan(values(s.h))
    want = np.zeros(bad.shape, bool)
    want[1, 250:, 33] = want[0, 140:, 2] = True
    assert np.array_equal(bad, want)
    assert np.array_equal(np.argwhere(np.isnan(values(s.last))), [[0, 2], [1, 33]])


@pytest.mark.parametrize("length", [20, 400, 9000])
def test_a_gate_that_is_not_a_number_is_not_lost(length):
    """With a value of 0 nothing but the state itself is NaN, and without gradients behind it but the last state's: what passes on
    from there is NaN in every step, up to a gate that selects."""
    shape = (1, length, 70)
    f, v, initial, lengths, _, dlast = _data(shape, "f32", 19)
    at, shut = length // 2, length * 3 // 4
    f[0, at, ::3], v[0, at:, ::3], f[0, shut, 6] = np.nan, 0.0, -np.inf
    s = Scan(f, v, initial, lengths, "f32", np.zeros(shape, np.float32), dlast)
    s.forward()
    bad = np.zeros(shape, bool)
    bad[0, at:, ::3] = True
    bad[0, shut:, 6] = False
    assert np.array_equal(np.isnan(values(s.h)), bad)
    assert np.array_equal(np.isnan(values(s.last)), bad[:, -1])
    s.backward()
    lost = np.zeros(70, bool)
    lost[::3] = True
    lost[6] = False  # a gradient of 0 times a gate that is NaN: 0 or NaN
    got = np.isnan(values(s.initial.kept_grad)[0])
    assert got[lost].all() and not got[np.arange(70) % 3 != 0].any()


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 0, 0)])
def test_only_what_is_wanted(wanted):
    f, v, initial, lengths, dy, dlast = _data((3, 300, 50), "f32", 8, ragged=True)
    want = scan_exact(f, v, initial, lengths, dy, dlast)
    for add in (False, True):
        s = Scan(f, v, initial, lengths, "f32", dy, dlast, old=np.random.RandomState(2))
        for t, w in zip((s.f, s.v, s.initial), wanted):
            t.t.requires_grad = bool(w)
        s.forward()
        s.backward(add)
        s.check_backward(want, f"{wanted} {add}", add)


@pytest.mark.parametrize("looks", [0, 4096])
@pytest.mark.parametrize("length", [1, 5, 300, 1000])
def test_the_state_in_place(length, looks):
    """The initial state's buffer is the last state's: a decoder that goes on from where it is."""
    from plast_amd.runtime import lib
    f, v, initial, lengths, _, _ = _data((4, length, 70), "f32", 9)
    lengths[:] = [length, length // 2, 0, length]
    want = scan_exact(f, v, initial, lengths)
    s = Scan(f, v, initial, lengths, "f32")
    s.ins[4] = s.initial
    lib().plast_hip_set_recurrence_looks(looks)
    try:
        s.forward(keep=False)
    finally:
        lib().plast_hip_set_recurrence_looks(4096)
    close(values(s.initial), want["last"], want["last_tol"] + stored(want["last"], "f32"), "state")
    close(values(s.h), want["h"], want["h_tol"] + stored(want["h"], "f32"), "h")


def test_token_by_token_is_the_sequence():
    """A prompt in one call and the rest token by token, against the whole sequence."""
    from plast_amd import ops
    rng = np.random.RandomState(10)
    B, T, D = 3, 150, 40
    f, v = scan_inputs(rng, (B, T, D), "f32")
    initial = rng.randn(B, D).astype(np.float32)
    want = scan_exact(f, v, initial, [T] * B)
    got, state = [], device(initial, "f32")
    for a, b in [(0, 141)] + [(t, t + 1) for t in range(141, T)]:
        inputs, h, _ = ops.gated_recurrence(device(f[:, a:b], "f32"), device(v[:, a:b], "f32"), state)
        got.append(h.numpy())
        state = inputs[4]
    close(np.concatenate(got, 1), want["h"], want["h_tol"] + stored(want["h"], "f32"), "h")


def test_halves_of_one_projection():
    """f and v as halves of one buffer, their gradients as halves of another."""
    from plast_amd.runtime import DeviceTensor
    B, T, D = 2, 300, 36
    f, v, initial, lengths, dy, dlast = _data((B, T, D), "bf16", 11)
    want = scan_exact(f, v, initial, lengths, dy, dlast)
    s = Scan(f, v, initial, lengths, "bf16", dy, dlast)
    both = device(np.concatenate([f, v], 2), "bf16")
    grads = device(np.zeros((B, T, 2 * D)), "bf16")
    for k, name in ((0, "f"), (1, "v")):
        t, g = (DeviceTensor((B, T, D), abi.BFLOAT16, base=x.buffer, offset=k * D, strides=(2 * D * T, 2 * D, 1)) for x in (both, grads))
        s.ins[k] = give(t, g)
    s.forward()
    s.check_forward(want, "halves")
    s.backward()
    got = values(grads)
    for k, name in ((0, "df"), (1, "dv")):
        close(got[..., k * D:(k + 1) * D], want[name], want[name + "_tol"] + stored(want[name], "bf16"), name)


def test_one_sequence_read_as_gate_and_value():
    """f and v may be one tensor where no gradient is asked for."""
    f, _, initial, lengths, _, _ = _data((2, 200, 20), "f32", 12)
    want = scan_exact(f, f, initial, lengths)
    s = Scan(f, f, initial, lengths, "f32")
    s.ins[1] = s.f
    s.forward()
    s.check_forward(want, "one tensor")


def test_no_steps():
    from plast_amd import ops
    initial = np.random.RandomState(1).randn(3, 5).astype(np.float32)
    from plast_amd.runtime import DeviceTensor, backward
    empty = DeviceTensor((3, 0, 5))
    inputs, h, p = ops.gated_recurrence(empty, DeviceTensor((3, 0, 5)), device(initial, "f32"))
    assert np.array_equal(inputs[4].numpy(), initial)
    for old in (0.0, 3.0):  # what comes for the last state goes to the initial one
        g, ini = device(np.full((3, 5), old), "f32"), np.ones((3, 5), np.float32)
        states, lengths = DeviceTensor((3, 0, 5)), DeviceTensor((3,), abi.INT32)
        ins = [empty, empty, device(ini, "f32", grad=g), lengths, device(ini, "f32", grad=device(initial, "f32")), states]
        h = DeviceTensor((3, 0, 5), requires_grad=True)
        backward("gated_recurrence", ins, h, KernelParams(1, 0 if old else 1, 0.0))
        assert np.array_equal(values(g), initial + np.float32(old))
    for shape in ((0, 4, 5), (3, 4, 0)):
        ops.gated_recurrence(DeviceTensor(shape), DeviceTensor(shape))


def test_the_gradient_against_differences():
    """sum(h c) + sum(last k) moved by gates, values and the initial state: central differences of the forward pass itself. A
    step of 2^-6 leaves a third-order rest, and the sums' rounding is divided by it."""
    shape = (1, 140, 3)
    f, v, initial, lengths, dy, dlast = _data(shape, "f32", 13, keep=(-1.0, 2.0))

    def total(f, v, initial):
        s = Scan(f, v, initial, lengths, "f32")
        s.forward(keep=False)
        return float((values(s.h).astype(np.float64) * dy).sum() + (values(s.last).astype(np.float64) * dlast).sum())
    s = Scan(f, v, initial, lengths, "f32", dy, dlast)
    s.forward()
    s.backward()
    step = 2.0 ** -6
    rng = np.random.RandomState(0)
    for k, (t, g) in enumerate(((f, s.f), (v, s.v), (initial, s.initial))):
        for i in rng.choice(t.size, min(t.size, 12), replace=False):
            moved = []
            for sign in (1, -1):
                args = [f.copy(), v.copy(), initial.copy()]
                args[k].reshape(-1)[i] += sign * step
                moved.append(total(*args))
            slope = (moved[0] - moved[1]) / (2 * step)
            assert abs(slope - values(g.kept_grad).reshape(-1)[i]) < 40 * step ** 2 + 420 * 4 * 2.0 ** -24 * 8 / step, (k, i)


def test_same_bits_every_time():
    for shape in ((1, 5000, 40), (2, 1000, 200)):
        runs = []
        for _ in range(3):
            s = _check(shape, "f32", seed=14)
            runs.append([values(t) for t in (s.h, s.last, s.f.kept_grad, s.v.kept_grad, s.initial.kept_grad)])
        for other in runs[1:]:
            for a, b in zip(runs[0], other):
                assert np.array_equal(a, b)


@pytest.mark.parametrize("looks", [0, 1])
def test_chunks_that_do_not_come_in_time(looks):
    """A workgroup that does not wait for the chunk before its own works it out itself: the same bits."""
    from plast_amd.runtime import lib
    for shape, kind in (((2, 1000, 200), "f32"), ((1, 3000, 40), "bf16"), ((8, 500, 128), "f16")):
        runs = []
        for most in (4096, looks):
            lib().plast_hip_set_recurrence_looks(most)
            try:
                s = _check(shape, kind, ragged=shape[0] > 1, seed=16)
            finally:
                lib().plast_hip_set_recurrence_looks(4096)
            runs.append([values(t) for t in (s.h, s.last, s.f.kept_grad, s.v.kept_grad, s.initial.kept_grad)])
        for a, b in zip(*runs):
            assert np.array_equal(a, b)


def test_replayed_with_other_work_between():
    """Captured forward and backward passes of two sizes, replayed in turn with eager work between."""
    from plast_amd import runtime as rt
    L = rt.lib()
    graphs = []
    for shape, kind in (((2, 700, 70), "f32"), ((1, 2000, 40), "bf16"), ((64, 1, 100), "f16"), ((2, 128, 64), "f32")):
        f, v, initial, lengths, dy, dlast = _data(shape, kind, 15, ragged=shape[0] > 1)
        s = Scan(f, v, initial, lengths, kind, dy, dlast)
        s.forward()
        s.backward()
        assert L.plast_hip_capture_begin() == 0
        s.forward()
        s.backward()
        graphs.append((s, f, L.plast_hip_capture_end()))
        L.check("capture")
    for rep in range(3):
        for s, f, graph in graphs:
            new = device(rounded(f + rep, s.kind), s.kind)
            L.arena_memcpy_d2d_hip(s.f.ptr, new.ptr, f.size * s.f.itemsize)
            outs = (s.h, s.last, s.f.kept_grad, s.v.kept_grad, s.initial.kept_grad)
            s.forward()
            s.backward()
            eager = [values(t) for t in outs]
            a = rt.DeviceTensor((1000, 1000)).fill_("normal", rep, 0.0, 1.0)
            rt.forward("sum", [a], rt.DeviceTensor((1000,)), KernelParams(0, 0, 0.0))
            for t in outs:
                L.zeros_hip(t.p, int(np.prod(t.shape)))
            assert L.plast_hip_graph_launch(graph) == 0
            for e, t in zip(eager, outs):
                assert np.array_equal(e, values(t)), (s.shape, rep)
    for _, _, graph in graphs:
        L.plast_hip_graph_destroy(graph)
