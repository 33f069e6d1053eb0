"""Alternatives of rows whose largest logits stand together: rising rows, a masked start, a window, ties at the end. They
are found whatever the order, at the cost of a few passes over the row and not of one per alternative."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_token_logprob import KINDS, Case, _rt
from token_cases import check_values, exact, load, logits, store

pytestmark = pytest.mark.gpu


def _ordered(rng, x, form):
    """A row put in order, in place."""
    vocab = x.size
    if form == "sorted":
        x.sort()
    elif form == "prefix":
        x[: rng.randint(vocab // 4, vocab - 40)] = -np.inf
    elif form == "window":
        at, n = rng.randint(vocab // 4, vocab // 2), max(vocab // 8, 300)
        x[:at], x[at + n:] = -np.inf, -np.inf
    elif form == "ramp":
        x += np.linspace(0, 60, vocab, dtype=np.float32)
    elif form == "ties":                   # the largest value many times, towards the end
        x.sort()
        x[-(vocab // 5):] = x[-1]
    elif form == "far ties":               # and only in the last units' last places
        x[: vocab // 2] = -np.inf
        x[vocab // 2:] = -5.0
        x[-vocab // 4:: 8] = 4.0
    elif form == "columns":                # rising, and every 512th logit larger than the others
        x += np.linspace(0, 8, vocab, dtype=np.float32)
        x[3::512] += 40.0
    elif form == "one nan":
        x.sort()
        x[vocab - 5] = np.nan
    elif form == "one inf":
        x.sort()
        x[-1] = np.inf


FORMS = ("sorted", "prefix", "window", "ramp", "ties", "far ties", "columns", "one nan", "one inf")


# a wave, four and sixteen waves to a row, and rows in pieces
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows, vocab", [(4000, 2517), (4000, 5117), (1100, 20011), (300, 70001), (9, 300013), (40, 151936)])
def test_values(kind, rows, vocab):
    rng = np.random.RandomState(vocab)
    x = logits(rng, rows, vocab, kind)
    at = np.arange(0, rows, max(1, rows // 40))
    for k, r in enumerate(at):
        _ordered(rng, x[r], FORMS[k % len(FORMS)])
    x = load(store(x, kind))
    tok = rng.randint(0, vocab, rows)
    for top in (1, 5, 20, 32):
        print(f"ordered {kind} {rows}x{vocab} top {top}", flush=True)
        got = Case(x, kind, tok, 1.0, top).forward().values()
        check_values({k: v[at] for k, v in got.items()}, exact(x[at], tok[at], 1.0, top),
                     f"{kind} {rows}x{vocab} top {top}")


@pytest.mark.parametrize("kind, rows, vocab, top", [("bf16", 300, 131072, 20), ("f32", 1200, 32000, 10),
                                                    ("f16", 64, 131072, 20)])
def test_cost(kind, rows, vocab, top):
    """Three reads of the row, where one per alternative took ten to a hundred times as long as a single read."""
    L = _rt().lib()
    took = {}
    for form in ("any order", "sorted", "prefix", "window"):
        rng = np.random.RandomState(3)
        x = logits(rng, rows, vocab, kind)
        for r in range(rows):
            _ordered(rng, x[r], form)
        c = Case(x, kind, np.full(rows, 5), 1.0, top).forward()
        times = []
        for _ in range(20):
            L.plast_hip_timer_begin()
            c.forward()
            times.append(L.plast_hip_timer_end())
        took[form] = sorted(times)[10]
    print(f"ordered {kind} {rows}x{vocab} top {top}: {took} ms", flush=True)
    assert max(took.values()) < 5 * took["any order"], took
