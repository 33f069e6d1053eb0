"""Token log-probabilities under masks of large finite values, whatever part of a row they cover: c m, c = log2(e) /
temperature, is then far beyond what its rounding leaves of an exponent."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_token_logprob import KINDS, Case
from token_cases import check_gradient, check_values, exact, load, logits, store

pytestmark = pytest.mark.gpu
MASKS = [-1e4, -1e9, -1e10, -1e12, -1e15, -1e20, -1e30, -1e32, -1e36, -1.7014118e38, -3.3895314e38]


def _masked(rng, rows, vocab, kind):
    """Each row with one of MASKS over its start, all of it, all but its last logit, every second, or most of it."""
    x = logits(rng, rows, vocab, kind)
    for r in range(rows):
        mask = MASKS[r // 5 % len(MASKS)]
        if r % 5 == 0:
            x[r, : vocab // 2] = mask
        elif r % 5 == 1:
            x[r] = mask
        elif r % 5 == 2:
            x[r, : vocab - 1] = mask
        elif r % 5 == 3:
            x[r, 1::2] = mask
        else:
            x[r, rng.rand(vocab) < 0.9] = mask
    return load(store(x, kind))


def _tokens(rng, rows, vocab):
    t = rng.randint(0, vocab, rows)
    t[::7] = vocab - 1
    return t


@pytest.mark.parametrize("kind", [k for k in KINDS if k != "f16"])
@pytest.mark.parametrize("rows, vocab", [(60, 18), (60, 300), (60, 2051), (60, 20011), (600, 9001), (8200, 1100),
                                         (300, 50000), (2, 131072)])
def test_forward_under_finite_masks(kind, rows, vocab):
    rng = np.random.RandomState(rows + vocab)
    x, tok = _masked(rng, rows, vocab, kind), _tokens(rng, rows, vocab)
    for top, temp in ((0, 1.0), (5, 0.7), (20, 5.0), (3, 1e-6))[:4 if rows < 1000 else 2]:
        print(f"masks {kind} {rows}x{vocab} top {top} temperature {temp}", flush=True)
        c = Case(x, kind, tok, temp, top).forward()
        check_values(c.values(), exact(x, tok, float(np.float32(temp)), top), f"{kind} {rows}x{vocab} top {top} {temp}")


@pytest.mark.parametrize("kind", [k for k in KINDS if k != "f16"])
@pytest.mark.parametrize("rows, vocab", [(60, 18), (60, 300), (60, 8192), (60, 33001), (1100, 20000), (60, 140003)])
def test_gradient_and_step_under_finite_masks(kind, rows, vocab):
    rng = np.random.RandomState(rows + vocab)
    x, tok = _masked(rng, rows, vocab, kind), _tokens(rng, rows, vocab)
    u, h = rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)
    for temp in (1.0, 5.0)[:2 if rows < 1000 else 1]:
        print(f"masks step {kind} {rows}x{vocab} temperature {temp}", flush=True)
        want = exact(x, tok, temp, 0, u, h)
        c = Case(x, kind, tok, temp, 0, u, h).forward().backward()
        check_values(c.values(), want, f"{kind} {rows}x{vocab} {temp}")
        check_gradient(c.dx(), want, kind, f"{kind} {rows}x{vocab} {temp}")
        s = Case(x, kind, tok, temp, 0, u, h).step()
        check_values(s.values(), want, f"step {kind} {rows}x{vocab} {temp}")
        check_gradient(s.dx(), want, kind, f"step {kind} {rows}x{vocab} {temp}")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows, vocab", [(60, 18), (60, 300), (60, 20011), (1100, 20000), (600, 9001), (2, 131072),
                                         (60, 140003)])
def test_padding_whatever_its_rows_hold(kind, rows, vocab):
    rng = np.random.RandomState(rows + vocab)
    x, tok = logits(rng, rows, vocab, kind), rng.randint(0, vocab, rows)
    tok[::2] = [-1, -2 ** 31][rows % 4 // 2]
    x[::2] = np.resize(np.array([np.nan, np.inf, -np.inf, 1e4], np.float32), (len(x[::2]), vocab))
    u, h = rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)
    print(f"padding {kind} {rows}x{vocab}", flush=True)
    want = exact(x, tok, 1.0, 4, u, h)
    assert not want["dx"][::2].any() and not want["logp"][::2].any() and not want["entropy"][::2].any()
    c = Case(x, kind, tok, 1.0, 4, u, h).forward().backward()
    check_values(c.values(), want, f"padding {kind}")
    check_gradient(c.dx(), want, kind, f"padding {kind}")
    s = Case(x, kind, tok, 1.0, 0, u, h).step()
    check_values(s.values(), want, f"padding step {kind}")
    check_gradient(s.dx(), want, kind, f"padding step {kind}")
