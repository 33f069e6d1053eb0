"""Inputs of the tests of layer norm, the gated recurrence and gradient clipping, the operators in 64 bits, and the
tolerances, which count roundings: U is half a step of fp32 relative to the value."""
from __future__ import annotations

import ctypes as C

import numpy as np

from plast_amd import abi
from plast_amd.abi import BFLOAT16, FLOAT16, FLOAT32
from token_cases import HALF_STEP, load, store

U = 2.0 ** -24
# a product below 2^-126 is off by up to half of 2^-149, whatever its size; a step takes up to four, of the step itself and of
# the states that a run of steps is joined from, and the next steps pass it on times a
TINY = 4 * 2.0 ** -150
DTYPE = {"f32": FLOAT32, "f16": FLOAT16, "bf16": BFLOAT16}


def rounded(values, kind):
    """What a tensor of `kind` holds of float32 values."""
    return load(store(np.asarray(values, np.float32), kind))


def stored(want, kind):
    """How far a result rounded to `kind` may be from `want`, beside what fp32 is off. Subnormal numbers are as far apart as the
    smallest one, 2^-149 in fp32, 2^-24 in fp16 and 2^-133 in bf16: half of that, and of eight products in fp32."""
    low = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[kind] + 8 * 2.0 ** -150
    return HALF_STEP[kind][0] * np.abs(want) * (1 + 2.0 ** -6) + low


def close(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off, first at {i}: {got[i]} for {want[i]}, "
                             f"tolerance {np.broadcast_to(tol, want.shape)[i]}")


def device(values, kind, lead=0, pitch=0, grad=None):
    """A device tensor of `values` inside a larger buffer: `lead` elements in front of it, the last axis `pitch` apart
    (0: contiguous); what lies around is 77. Returns the tensor; `grad` becomes its gradient."""
    from plast_amd.runtime import DeviceTensor
    values = np.asarray(values, np.float32)
    width = values.shape[-1]
    pitch = pitch or width
    rows = int(np.prod(values.shape[:-1]))
    buf = np.full(lead + rows * pitch + 8, 77.0, np.float32)
    for r, row in enumerate(values.reshape(rows, width)):
        buf[lead + r * pitch:lead + r * pitch + width] = row
    base = DeviceTensor.from_numpy(store(buf, kind))
    strides, step = [1], pitch
    for n in reversed(values.shape[1:-1] if values.ndim > 1 else ()):
        strides.append(step)
        step *= n
    if values.ndim > 1:
        strides.append(step)
    t = DeviceTensor(values.shape, DTYPE[kind], base=base, offset=lead, strides=list(reversed(strides))[-values.ndim:])
    t.buffer = base
    if grad is not None:
        give(t, grad)
    return t


def give(t, grad):
    t.kept_grad = grad  # the struct points at it
    t.t.grad, t.t.requires_grad = C.pointer(grad.t), True
    return t


def values(t):
    return load(t.numpy()) if t.dtype != FLOAT32 else t.numpy()


def around(t, kind):
    """What lies in a device() tensor's buffer beside the tensor itself."""
    mark = np.zeros(t.buffer.shape, bool)
    item = np.lib.stride_tricks.as_strided(mark[(t.ptr - t.buffer.ptr) // t.itemsize:], t.shape, abi.strides_of(t.t))
    item[...] = True
    return load(t.buffer.numpy())[~mark] if kind != "f32" else t.buffer.numpy()[~mark]


# ----------------------------------------------------------------------------- layer norm

def norm_exact(x, w, b, eps, dy=None):
    """y, its tolerance in fp32, and for dy the gradients with theirs. x: [N, C] of float values."""
    x, w, b = (np.asarray(v, np.float64) for v in (x, w, b))
    N, width = x.shape
    mu = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + eps)
    n = (x - mu) * r
    # a lane adds at most width / 64 + 32 terms one after the other, then up to sixteen sums of lanes and waves
    add = (width / 64 + 48) * U
    # of n where n itself is small: the mean is a float32, and the sum of the differences that corrects it is off by up to
    # `add` times the sum of their sizes, as any sum of that many terms is: its C-th part is add mean|x - mu|
    off = (2 * U * np.abs(mu) + add * np.abs(x - mu).mean(1, keepdims=True)) * r
    out = {"y": n * w + b}
    out["y_tol"] = np.abs(n * w) * (add + 8 * U) + np.abs(w) * off + 2 * U * np.abs(out["y"])
    if dy is None:
        return out
    dy = np.asarray(dy, np.float64)
    g = dy * w
    mg, mgn = g.mean(1, keepdims=True), (g * n).mean(1, keepdims=True)
    ag, agn = np.abs(g).mean(1, keepdims=True), np.abs(g * n).mean(1, keepdims=True)
    out["dx"] = r * (g - mg - n * mgn)
    out["dx_tol"] = (r * (np.abs(g) + ag + np.abs(n) * agn) * 2 * (add + 8 * U)
                     + r * off * (np.abs(n) * ag + np.abs(mgn)))
    out["dw"], out["db"] = (dy * n).sum(0), dy.sum(0)
    # any order of N additions
    out["dw_tol"] = (np.abs(dy * n) * (add + (N + 8) * U) + np.abs(dy) * off).sum(0)
    out["db_tol"] = np.abs(dy).sum(0) * (N + 2) * U
    return out


# ----------------------------------------------------------------------------- gated recurrence

def scan_inputs(rng, shape, kind, keep=(-2.0, 5.0)):
    """Gates of channels that remember for a step to some hundreds, and values."""
    f = rng.randn(*shape) + rng.uniform(*keep, shape[-1])
    return rounded(f, kind), rounded(rng.randn(*shape) + 0.5, kind)


def scan_exact(f, v, initial, lengths, dy=None, dlast=None):
    """h, last, the gradients, and what fp32 may be off for each. A gate's smaller side is off by its exponent's rounding
    (|f| steps) and five more; a step adds to that eight roundings of what the state is made of, as the states of a run of steps
    are joined in other orders."""
    f, v, initial = (np.asarray(t, np.float64) for t in (f, v, initial))
    B, T, D = f.shape
    ends = np.clip(lengths, 0, T)
    with np.errstate(over="ignore", invalid="ignore"):
        e = np.exp(-np.abs(f))
        s = e / (1 + e)
        s = np.where(s < 2.0 ** -126, 0.0, s)
        a, z = np.where(f > 0, 1 - s, s), np.where(f > 0, s, 1 - s)
        rel = np.where(np.isfinite(f), (2 * np.abs(f) + 8) * U, 0.0)

    def mix(x, y, p, q):
        """p x + q y where a factor of 0 takes nothing, NaN neither."""
        with np.errstate(invalid="ignore"):
            return np.where(p == 0, 0.0, p * x) + np.where(q == 0, 0.0, q * y)
    h = np.zeros((B, T, D))
    E, M = np.zeros((B, T, D)), np.zeros((B, T, D))
    before, E_before = np.zeros((B, T, D)), np.zeros((B, T, D))
    state, err, size = initial.copy(), np.zeros((B, D)), np.abs(initial)
    for t in range(T):
        live = (t < ends)[:, None]
        before[:, t], E_before[:, t] = state, err
        new = mix(state, v[:, t], a[:, t], z[:, t])
        new_size = mix(size, np.abs(v[:, t]), a[:, t], z[:, t])
        with np.errstate(invalid="ignore"):
            new_err = mix(err, 0.0, a[:, t], 0.0 * z[:, t]) + np.where(
                s[:, t] == 0, 0.0, rel[:, t] * s[:, t] * np.abs(v[:, t] - state) + 8 * U * (new_size + s[:, t] * np.abs(state)) + TINY)
        state, err, size = (np.where(live, p, q) for p, q in ((new, state), (new_err, err), (new_size, size)))
        h[:, t], E[:, t], M[:, t] = np.where(live, state, 0.0), np.where(live, err, 0.0), size
    out = {"h": h, "h_tol": E, "last": state, "last_tol": err}
    if dy is None and dlast is None:
        return out
    dy = np.zeros((B, T, D)) if dy is None else np.asarray(dy, np.float64)
    df, dv, df_tol, dv_tol = (np.zeros((B, T, D)) for _ in range(4))
    g = np.zeros((B, D)) if dlast is None else np.asarray(dlast, np.float64).copy()
    err, size = np.zeros((B, D)), np.abs(g)
    for t in range(T - 1, -1, -1):
        live = (t < ends)[:, None]
        with np.errstate(invalid="ignore"):
            dh = dy[:, t] + g
            dh_size = np.abs(dy[:, t]) + size
            dh_err = err + U * dh_size
            zt, at, st, rt = z[:, t], a[:, t], s[:, t], rel[:, t]
            shut = st == 0
            dvt = np.where(zt == 0, 0.0, zt * dh)
            slope = np.where(shut, 0.0, at * zt * (before[:, t] - v[:, t]))
            dft = np.where(shut, 0.0, dh * slope)
            dvt_tol = np.where(zt == 0, 0.0, zt * (dh_err + (rt + 4 * U) * dh_size))
            dft_tol = np.where(shut, 0.0, np.abs(slope) * (dh_err + (2 * rt + 8 * U) * dh_size)
                               + at * zt * dh_size * (E_before[:, t] + 2 * U * (np.abs(before[:, t]) + np.abs(v[:, t]))))
            ng = np.where(at == 0, 0.0, at * dh)
            nsize = np.where(at == 0, 0.0, at * dh_size)
            nerr = np.where(at == 0, 0.0, at * dh_err + np.where(shut, 0.0, rt * st * dh_size + 8 * U * dh_size + TINY))
        for to, x in ((df, dft), (dv, dvt), (df_tol, dft_tol), (dv_tol, dvt_tol)):
            to[:, t] = np.where(live, x, 0.0)
        g, err, size = (np.where(live, p, q) for p, q in ((ng, g), (nerr, err), (nsize, size)))
    out.update(df=df, dv=dv, df_tol=df_tol, dv_tol=dv_tol, dinitial=g, dinitial_tol=err + U * size)
    return out
