"""Alternatives of few rows, which are cut into pieces over workgroups: the pieces' candidates are joined at once,
however the largest logits are spread over them, and at the cost of a pass and not of one per alternative."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_token_logprob import KINDS, Case, _rt
from token_cases import check_values, exact, load, logits, store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows, vocab", [(8, 131072), (20, 50001), (3, 270011), (200, 33000)])
def test_spread_over_pieces(kind, rows, vocab):
    rng = np.random.RandomState(vocab)
    x = logits(rng, rows, vocab, kind)
    part = vocab // 32
    for r in range(rows):
        form = r % 8
        if form == 1:                      # all in one piece's range
            x[r, 5 * part: 6 * part] += 20
        elif form == 2:                    # in every second
            x[r].reshape(-1)[: 32 * part].reshape(32, part)[::2] += 20
        elif form == 3:                    # more towards the end
            x[r] += np.linspace(0, 30, vocab, dtype=np.float32)
        elif form == 4:                    # nothing in the first half
            x[r, : vocab // 2] = -np.inf
        elif form == 5:                    # NaN in half of them
            x[r].reshape(-1)[: 32 * part].reshape(32, part)[::2] = np.nan
        elif form == 6:                    # all equal
            x[r] = 1.0
        elif form == 7:                    # a few legal tokens, far apart
            keep = x[r, ::part].copy()
            x[r] = -np.inf
            x[r, ::part] = keep
    x = load(store(x, kind))
    tok = rng.randint(0, vocab, rows)
    for top in (1, 3, 20, 32):
        print(f"pieces {kind} {rows}x{vocab} top {top}", flush=True)
        c = Case(x, kind, tok, 1.0, top).forward()
        check_values(c.values(), exact(x, tok, 1.0, top), f"{kind} {rows}x{vocab} top {top}")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("vocab", [131072, 50001])
def test_as_one_pass(kind, vocab):
    """A pass per alternative takes some 70 us each beside the call's 10 to 20."""
    L = _rt().lib()
    took = {}
    for top in (1, 32):
        c = Case(logits(np.random.RandomState(1), 1, vocab, kind), kind, np.array([5]), 1.0, top).forward()
        times = []
        for _ in range(20):
            L.plast_hip_timer_begin()
            c.forward()
            times.append(L.plast_hip_timer_end())
        took[top] = sorted(times)[10]
    print(f"pieces {kind} {vocab}: {took} ms", flush=True)
    assert took[32] < 10 * took[1], took
