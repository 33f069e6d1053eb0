"""Inputs of the token log-probability tests, the operator in 64 bits, and the tolerances."""
from __future__ import annotations

import numpy as np

from plast_amd import ops

# half a step of each type relative to the value, and of its subnormals
HALF_STEP = {"f32": (2.0 ** -24, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}


def store(values, kind):
    """float32 values as the array a tensor of `kind` is made from."""
    if kind == "bf16":
        return ops.bfloat16_bits(values)
    with np.errstate(over="ignore"):
        return np.ascontiguousarray(values, np.float16 if kind == "f16" else np.float32)


def load(array):
    return ops.bfloat16_values(array) if array.dtype == np.uint16 else array.astype(np.float32)


def logits(rng, rows, vocab, kind, masked=0.0, scale=2.0):
    x = (rng.randn(rows, vocab) * scale).astype(np.float32)
    if masked:
        x[rng.rand(rows, vocab) < masked] = -np.inf
    return load(store(x, kind))


def special(x, kind):
    """Rows that masks, infinities and ties leave, written into the first rows of x."""
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[kind]
    rows = [("masked", -np.inf), ("low", low), ("zero", 0.0)]
    for k, (_, v) in enumerate(rows):
        if k < len(x):
            x[k] = v
    vocab = x.shape[1]
    if len(x) > 9 and vocab > 4:
        x[2, 1::2] = -0.0                      # both zeros tie
        x[3] = low                             # a few legal tokens above the type's lowest value
        x[3, [1, vocab - 1]] = [1.0, 2.0]
        x[4] = -np.inf                         # the same above -inf
        x[4, [0, vocab // 2]] = [0.5, 0.25]
        x[5, vocab // 3] = np.nan
        x[6, vocab // 2] = np.inf
        x[7] = np.sort(x[7])                   # ascending: every logit a new maximum
        x[8] = np.sort(x[8])[::-1]
        x[9, vocab - 1] = -low                 # the type's largest value
    return x


def exact(x, tokens, temp, top=0, u=None, h=None):
    """logp, entropy, top_logp, top_ids and dx in 64 bits."""
    n, vocab = x.shape
    z = x.astype(np.float64) / temp
    out = {}
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = z.max(1, keepdims=True)
        e = np.exp(z - m)
        lp = np.where(m == -np.inf, -np.inf, z - m - np.log(e.sum(1, keepdims=True)))
        bad = np.isnan(z).any(1) | (z == np.inf).any(1)
        lp[bad] = np.nan
        p = np.exp(lp)
        plogp = np.where(p > 0, p * lp, 0.0)
        plogp[bad] = np.nan
        ent = -plogp.sum(1)
        live, empty = tokens >= 0, (m[:, 0] == -np.inf) & ~bad
        given = lp[np.arange(n), np.clip(tokens, 0, vocab - 1)]
        given = np.where(tokens >= vocab, np.nan, given)
        out["logp"] = np.where(live, given, 0.0)
        out["entropy"] = np.where(live, ent, 0.0)
        if top:
            key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
            nan_first = np.where(np.isnan(x), 0, 1)
            ids = np.empty((n, min(top, vocab)), np.int64)
            for r in range(n):
                ids[r] = np.lexsort((np.arange(vocab), -key[r], nan_first[r]))[:top]
            tl = np.take_along_axis(lp, ids, 1)
            tl[~live], ids[~live] = -np.inf, -1
            short = top - ids.shape[1]
            out["top_logp"] = np.pad(tl, ((0, 0), (0, short)), constant_values=-np.inf)
            out["top_ids"] = np.pad(ids, ((0, 0), (0, short)), constant_values=-1)
        if u is not None:
            u64, h64 = u.astype(np.float64)[:, None], h.astype(np.float64)[:, None]
            d = -u64 * p - np.where(p > 0, h64 * p * (lp + ent[:, None]), 0.0)
            scale = np.abs(u64) * p + np.abs(h64) * np.where(p > 0, p * (np.abs(lp) + ent[:, None]), 0.0)
            hit = np.zeros_like(d)
            ok = live & (tokens < vocab)
            hit[np.flatnonzero(ok), tokens[ok]] = 1.0
            d, scale = d + u64 * hit, scale + np.abs(u64) * hit
            d[bad] = np.nan
            d[tokens >= vocab] = np.nan
            gone = ~live | empty
            out["dx"] = np.where(gone[:, None], 0.0, d / temp)
            out["scale"] = np.where(gone[:, None], 0.0, scale / temp)
    return out


def close(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    with np.errstate(invalid="ignore"):
        ok = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= tol)
    if not ok.all():
        i = tuple(np.argwhere(~ok)[0])
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.size} off; first at {i}: {got[i]!r}, want "
                             f"{want[i]!r} within {np.broadcast_to(tol, got.shape)[i]!r}")


# The kernels' 32-bit errors. An exponential's argument z is off by half a step of |z| twice (its factor
# and itself), the exponential by one step, a sum of n terms by a step for each level it is added at;
# what a row sum passes on is below 1e-5 of it, this library's bar for sums. log p and H move by that
# and by their own rounding.
def check_values(got, want, what):
    for name in ("logp", "entropy", "top_logp"):
        if name in got:
            # a float32 result: beyond its range it is infinite
            with np.errstate(invalid="ignore", over="ignore"):
                value = want[name].astype(np.float32)
                tol = 1e-5 + 1e-6 * np.abs(value)
            close(got[name].reshape(value.shape), value, tol, f"{what} {name}")
    if "top_ids" in got:
        ids = got["top_ids"].reshape(want["top_ids"].shape)
        assert np.array_equal(ids, want["top_ids"]), \
            f"{what}: ids differ in rows {np.flatnonzero((ids != want['top_ids']).any(1))[:8]}"


def check_gradient(got, want, kind, what, before=None):
    """1e-5 of the magnitudes of an element's terms, and the rounding to the gradient's type."""
    rel, tiny = HALF_STEP[kind]
    total = want["dx"] if before is None else want["dx"] + before.astype(np.float64)
    with np.errstate(invalid="ignore"):
        tol = 1e-5 * want["scale"] * (1 + 2 * rel) + 1.001 * rel * np.abs(total) + tiny + 1e-37
    close(got, total, tol, f"{what} dx")
