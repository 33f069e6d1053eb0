"""Token log-probabilities, entropies, alternatives and gradients on the GPU against 64 bits: types, row
lengths on each side of the dispatch lines, leading strides, odd alignments, masks that leave a row
little or nothing, padding, accumulation, the one-pass step, graph capture, and the gradient against
differences."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from plast_amd import abi
from plast_amd.abi import BFLOAT16, FLOAT16, FLOAT32, INT32, KernelParams
from token_cases import check_gradient, check_values, close, exact, load, logits, special, store

pytestmark = pytest.mark.gpu
KINDS = {"f32": FLOAT32, "f16": FLOAT16, "bf16": BFLOAT16}


def _rt():
    from plast_amd import runtime
    return runtime


def _vec(shape, dtype=FLOAT32, grad=None):
    """A vector holding something else than a result, with a gradient where one is given."""
    rt = _rt()
    t = rt.DeviceTensor(shape, dtype, zero=False)
    a = np.full(shape, 77, np.int32 if dtype == INT32 else np.float32)
    if a.nbytes:
        rt.lib().arena_memcpy_h2d_hip(t.ptr, a.ctypes.data, a.nbytes)
    if grad is not None:
        g = rt.DeviceTensor.from_numpy(np.ascontiguousarray(grad, np.float32))
        t.grad, t.t.grad, t.t.requires_grad = g, C.pointer(g.t), True
    return t


class Case:
    """x in a buffer of its own with `lead` axes of given strides, starting `offset` elements in."""

    def __init__(self, x, kind, tokens, temp=1.0, top=0, u=None, h=None, lead=None, strides=None, offset=0,
                 before=None, grad_strides=None, grad_offset=0):
        rt = _rt()
        n, vocab = x.shape
        lead = (n,) if lead is None else lead
        self.kind, self.temp, self.top, self.n, self.vocab, self.lead = kind, temp, top, n, vocab, lead
        self.x, self.u, self.h = x, u, h
        strides = tuple(abi.row_major(lead + (vocab,))) if strides is None else strides
        self.dx_base, self.x_t = None, self._place(store(x, kind), lead, strides, offset)
        if u is not None:
            gs = tuple(abi.row_major(lead + (vocab,))) if grad_strides is None else grad_strides
            fill = store(np.full(x.shape, 5.0, np.float32) if before is None else before, kind)
            self.dx_t = self._place(fill, lead, gs, grad_offset)
            self.x_t.t.grad, self.x_t.t.requires_grad = C.pointer(self.dx_t.t), True
        self.tokens = rt.DeviceTensor.from_numpy(np.ascontiguousarray(tokens, np.int32))
        self.stats = _vec((n, 2))
        self.logp, self.entropy = _vec((n,), grad=u), _vec((n,), grad=h)
        self.ins = [self.x_t, self.tokens, self.stats, self.entropy]
        if top:
            self.tl, self.ti = _vec((n, top)), _vec((n, top), INT32)
            self.ins += [self.tl, self.ti]

    def _place(self, values, lead, strides, offset):
        rt = _rt()
        shape = lead + (values.shape[-1],)
        size = offset + 1 + sum((e - 1) * s for e, s in zip(shape, strides)) if values.size else 1
        buf = np.full(size, 9, values.dtype)
        view = np.lib.stride_tricks.as_strided(buf[offset:], shape, [s * buf.itemsize for s in strides])
        view[...] = values.reshape(shape)
        base = rt.DeviceTensor.from_numpy(buf)
        return rt.DeviceTensor(shape, KINDS[self.kind], base=base, offset=offset, strides=strides, zero=False)

    def forward(self):
        _rt().forward("token_logprob", self.ins, self.logp, KernelParams(self.top, 0, self.temp))
        return self

    def backward(self, overwrite=True):
        _rt().backward("token_logprob", self.ins, self.logp, KernelParams(self.top, int(overwrite), self.temp))
        return self

    def step(self):
        L = _rt().lib()
        ref = [C.byref(t.t) if t is not None else None for t in
               (self.x_t, self.tokens, self.logp.grad, self.entropy.grad, self.logp, self.entropy, self.dx_t)]
        L.token_logprob_step_hip(*ref, self.temp)
        L.check("token_logprob_step")
        return self

    def values(self):
        got = {"logp": self.logp.numpy(), "entropy": self.entropy.numpy()}
        if self.top:
            got["top_logp"], got["top_ids"] = self.tl.numpy(), self.ti.numpy()
        return got

    def dx(self):
        return load(self.dx_t.numpy().reshape(self.n, self.vocab))


def _tokens(rng, n, vocab, pad=0.2):
    t = rng.randint(0, vocab, n)
    t[rng.rand(n) < pad] = -1
    return t


VOCABS = [1, 2, 3, 7, 10, 18, 31, 64, 65, 127, 200, 257, 511, 1000, 1023, 1025, 2047, 2051, 4096, 5003, 8191,
          16391, 32000, 33001, 50001]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("vocab", VOCABS)
def test_forward_and_alternatives(kind, vocab):
    rng = np.random.RandomState(vocab)
    n = 17 if vocab > 300 else 70
    for top, temp, masked in ((0, 1.0, 0.0), (1, 0.7, 0.3), (5, 1.5, 0.9), (32, 1.0, 0.0)):
        print(f"forward {kind} {n}x{vocab} top {top}", flush=True)
        x = special(logits(rng, n, vocab, kind, masked), kind)
        tok = _tokens(rng, n, vocab)
        c = Case(load(store(x, kind)), kind, tok, temp, top).forward()
        check_values(c.values(), exact(c.x, tok, temp, top), f"{kind} {n}x{vocab} top {top}")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows, vocab", [(1, 131072), (3, 131071), (2, 262147), (1, 20), (5000, 20), (3000, 700)])
def test_few_long_rows_and_many_short(kind, rows, vocab):
    rng = np.random.RandomState(rows)
    for top in (0, 20):
        print(f"forward {kind} {rows}x{vocab} top {top}", flush=True)
        x = logits(rng, rows, vocab, kind, 0.1)
        tok = _tokens(rng, rows, vocab, 0.1)
        c = Case(x, kind, tok, 0.7, top).forward()
        check_values(c.values(), exact(x, tok, 0.7, top), f"{kind} {rows}x{vocab}")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows, vocab", [(300, 20011), (600, 9001), (2100, 2603), (8200, 4100), (20, 70001)])
def test_alternatives_of_special_rows(kind, rows, vocab):
    """Masked, tied, sorted and NaN rows among enough rows for each way of sharing a row."""
    rng = np.random.RandomState(vocab)
    for top, masked in ((20, 0.0), (32, 0.95)) if rows < 8000 else ((7, 0.3),):
        print(f"special rows {kind} {rows}x{vocab} top {top}", flush=True)
        x = special(logits(rng, rows, vocab, kind, masked), kind)
        x[10:14] = x[0:4]
        x[14, 5:] = -np.inf                    # fewer legal tokens than alternatives
        x[15, : vocab - 4] = x[1, 0]           # the type's lowest value before a few others
        tok = _tokens(rng, rows, vocab, 0.1)
        tok[:16] = rng.randint(0, vocab, 16)
        c = Case(x, kind, tok, 1.0, top).forward()
        check_values(c.values(), exact(x, tok, 1.0, top), f"{kind} {rows}x{vocab} top {top}")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("vocab", VOCABS + [131073])
def test_gradient_and_step(kind, vocab):
    rng = np.random.RandomState(vocab + 1)
    n = 15 if vocab > 300 else 70
    x = special(logits(rng, n, vocab, kind, 0.2), kind)
    tok = _tokens(rng, n, vocab)
    u, h = rng.randn(n).astype(np.float32), rng.randn(n).astype(np.float32)
    want = exact(x, tok, 0.8, 0, u, h)
    before = load(store(rng.randn(n, vocab).astype(np.float32), kind))
    print(f"gradient {kind} {n}x{vocab}", flush=True)
    c = Case(x, kind, tok, 0.8, 0, u, h, before=before).forward().backward(overwrite=False)
    check_gradient(c.dx(), want, kind, f"{kind} {n}x{vocab} accumulated", before)
    c.backward()
    check_gradient(c.dx(), want, kind, f"{kind} {n}x{vocab}")
    s = Case(x, kind, tok, 0.8, 0, u, h)
    for k in range(2):
        s.step()
        check_values(s.values(), want, f"step {kind} {n}x{vocab}")
        check_gradient(s.dx(), want, kind, f"step {kind} {n}x{vocab}")


@pytest.mark.parametrize("rows, vocab", [(1500, 18), (700, 2052), (600, 8192), (520, 32000), (1300, 17000),
                                         (1100, 16392)])
@pytest.mark.parametrize("kind", list(KINDS))
def test_step_over_more_rows_than_are_resident(kind, rows, vocab):
    rng = np.random.RandomState(rows)
    x = special(logits(rng, rows, vocab, kind), kind)
    tok = _tokens(rng, rows, vocab)
    u, h = rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)
    print(f"step {kind} {rows}x{vocab}", flush=True)
    want = exact(x, tok, 1.0, 0, u, h)
    c = Case(x, kind, tok, 1.0, 0, u, h).step()
    check_values(c.values(), want, f"step {kind} {rows}x{vocab}")
    check_gradient(c.dx(), want, kind, f"step {kind} {rows}x{vocab}")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("vocab", [19, 257, 1001, 4099])
def test_strides_and_alignments(kind, vocab):
    rng = np.random.RandomState(7)
    lead = (3, 5)
    n = 15
    x = logits(rng, n, vocab, kind)
    tok = _tokens(rng, n, vocab)
    u, h = rng.randn(n).astype(np.float32), rng.randn(n).astype(np.float32)
    want = exact(x, tok, 1.0, 4, u, h)
    up = (vocab + 63) // 64 * 64
    layouts = [((6 * up, up, 1), 0, None, 0), ((vocab, 3 * vocab, 1), 1, None, 1),
               ((5 * up, up, 1), 3, (vocab, 3 * vocab, 1), 0), (None, 1, (7 * up, up, 1), 5)]
    for xs, off, gs, goff in layouts:
        print(f"strides {kind} {vocab} {xs} {gs}", flush=True)
        c = Case(x, kind, tok, 1.0, 4, u, h, lead, xs, off, None, gs, goff).forward().backward()
        check_values(c.values(), want, f"{kind} {xs}")
        check_gradient(c.dx(), want, kind, f"{kind} {xs}")
        around = c.dx_t.base.numpy().copy()
        view = np.lib.stride_tricks.as_strided(around[goff:], lead + (vocab,), [s * around.itemsize for s in
                                               abi.strides_of(c.dx_t.t)])
        view[...] = 9
        assert (around == 9).all(), "written outside the gradient's rows"
        c.top, c.ins = 0, c.ins[:4]
        s = Case(x, kind, tok, 1.0, 0, u, h, lead, xs, off, None, gs, goff).step()
        check_values(s.values(), {k: want[k] for k in ("logp", "entropy")}, f"step {kind} {xs}")
        check_gradient(s.dx(), want, kind, f"step {kind} {xs}")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows", [1, 2, 40, 300])
def test_step_over_rows_too_long_to_hold(kind, rows):
    """The step's two passes: its statistics and the pieces of cut rows share one workspace."""
    vocab = 70000 if kind == "f32" else 140003
    rng = np.random.RandomState(rows)
    x = special(logits(rng, rows, vocab, kind), kind)
    tok = _tokens(rng, rows, vocab)
    u, h = rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)
    want = exact(x, tok, 1.0, 0, u, h)
    c = Case(x, kind, tok, 1.0, 0, u, h)
    for k in range(3):
        print(f"long step {kind} {rows}x{vocab} {k}", flush=True)
        c.step()
        check_values(c.values(), want, f"long step {kind} {rows}")
        check_gradient(c.dx(), want, kind, f"long step {kind} {rows}")


def test_broadcast_rows():
    """One row of logits for many tokens (stride 0): its gradient has rows of its own."""
    rng = np.random.RandomState(3)
    x1 = logits(rng, 1, 300, "f32")
    x = np.repeat(x1, 6, 0)
    tok = np.arange(6) * 40
    u, h = rng.randn(6).astype(np.float32), rng.randn(6).astype(np.float32)
    c = Case(x, "f32", tok, 1.0, 0, u, h, strides=(0, 1)).forward().backward()
    want = exact(x, tok, 1.0, 0, u, h)
    check_values(c.values(), want, "broadcast")
    check_gradient(c.dx(), want, "f32", "broadcast")


def test_missing_upstreams_tokens_out_of_range_and_no_rows():
    rng = np.random.RandomState(4)
    x = logits(rng, 4, 50, "f32")
    tok = np.array([3, 50, 2 ** 31 - 1, 0])
    one, zero = np.ones(4, np.float32), np.zeros(4, np.float32)
    c = Case(x, "f32", tok, 1.0, 0, one, zero)
    c.entropy.t.grad = None
    want = exact(x, tok, 1.0, 0, one, zero)
    c.forward().backward()
    check_values(c.values(), want, "out of range")
    check_gradient(c.dx(), want, "f32", "no entropy gradient")
    c.logp.t.grad = None
    c.backward()
    got = c.dx()
    assert (got[[0, 3]] == 0).all() and np.isnan(got[[1, 2]]).all()
    Case(np.empty((0, 50), np.float32), "f32", np.empty(0), 1.0, 3).forward()


def test_large_offsets_and_temperatures():
    """Logits far from zero, and temperatures that make exponents large: log p is still right."""
    rng = np.random.RandomState(5)
    for shift, temp in ((1e4, 1.0), (-3e5, 1.0), (0.0, 0.01), (0.0, 50.0), (2e38, 0.5)):
        x = (rng.randn(6, 1003) * 2 + shift).astype(np.float32)
        tok = rng.randint(0, 1003, 6)
        c = Case(x, "f32", tok, temp, 3).forward()
        want = exact(x, tok, float(np.float32(temp)), 3)
        for name in ("logp", "entropy", "top_logp"):
            close(c.values()[name], want[name], 1e-5 + 1e-6 * np.abs(want[name]), f"{shift} {temp} {name}")


def test_gradient_against_differences():
    """u logp + h H moves by the gradient along a direction: central differences of the 64-bit values."""
    rng = np.random.RandomState(6)
    n, vocab, temp = 5, 37, 0.9
    x = logits(rng, n, vocab, "f32")
    tok = rng.randint(0, vocab, n)
    u, h = rng.randn(n).astype(np.float32), rng.randn(n).astype(np.float32)
    c = Case(x, "f32", tok, temp, 0, u, h).forward().backward()
    d = rng.randn(n, vocab)
    eps = 1e-5

    def value(xx):
        w = exact(xx, tok, temp)
        return u.astype(np.float64) * w["logp"] + h * w["entropy"]

    x64 = x.astype(np.float64)
    slope = (value(x64 + eps * d) - value(x64 - eps * d)) / (2 * eps)
    close((c.dx().astype(np.float64) * d).sum(1), slope, 1e-4 * np.abs(d).max(), "slope")


def test_captured_calls_replay():
    rt = _rt()
    L = rt.lib()
    rng = np.random.RandomState(8)
    for rows, vocab, kind, top in ((2, 131072, "bf16", 20), (300, 1001, "f32", 5), (600, 4096, "f16", 0)):
        tok = _tokens(rng, rows, vocab)
        u, h = rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)
        c = Case(logits(rng, rows, vocab, kind), kind, tok, 1.0, top, u, h).forward().backward()
        s = Case(c.x, kind, tok, 1.0, 0, u, h).step()
        print(f"capture {rows}x{vocab}", flush=True)
        assert L.plast_hip_capture_begin() == 0
        try:
            c.forward().backward()
            s.step()
        finally:
            graph = L.plast_hip_capture_end()
        L.check("capture")
        assert graph
        try:
            for k in range(4):
                x = logits(rng, rows, vocab, kind)
                raw = store(x, kind)
                for t in (c, s):
                    L.arena_memcpy_h2d_hip(t.x_t.ptr, raw.ctypes.data, raw.nbytes)
                assert L.plast_hip_graph_launch(graph) == 0
                got = [c.values(), c.dx(), s.values(), s.dx()]
                want = exact(x, tok, 1.0, top, u, h)
                check_values(got[0], want, f"replay {k}")
                check_gradient(got[1], want, kind, f"replay {k}")
                check_values(got[2], want, f"replay {k} step")
                check_gradient(got[3], want, kind, f"replay {k} step")
                c.forward().backward()
                s.step()
                for a, b in zip(got, (c.values(), c.dx(), s.values(), s.dx())):
                    for p, q in zip(a.values() if isinstance(a, dict) else [a],
                                    b.values() if isinstance(b, dict) else [b]):
                        assert np.array_equal(p, q, equal_nan=True), f"replay {k} differs from the eager call"
        finally:
            L.plast_hip_graph_destroy(graph)


def test_through_the_graph_and_ops():
    """The DAG harness runs the op's slots, and ops.token_logprob the same calls."""
    from plast_amd import ops
    from plast_amd.graph import Graph
    rt = _rt()
    rng = np.random.RandomState(9)
    x, tok = logits(rng, 6, 40, "f32"), rng.randint(0, 40, 6).astype(np.int32)
    X, T = rt.DeviceTensor.from_numpy(x, requires_grad=True), rt.DeviceTensor.from_numpy(tok)
    ins, logp, p = ops.token_logprob(X, T, 1.0, 3, requires_grad=True)
    want = exact(x, tok, 1.0, 3, np.ones(6, np.float32), np.ones(6, np.float32))
    check_values({"logp": logp.numpy(), "entropy": ins[3].numpy(), "top_logp": ins[4].numpy(),
                  "top_ids": ins[5].numpy()}, want, "ops")
    g = Graph()
    g.node("token_logprob", ins, logp, p)
    g.build(logp, fuse=True)
    g.forward()
    ones = np.ones(6, np.float32)
    for t in (logp, ins[3]):
        rt.lib().arena_memcpy_h2d_hip(t.grad.ptr, ones.ctypes.data, ones.nbytes)
    g.backward()
    check_gradient(X.grad.numpy(), want, "f32", "graph")
