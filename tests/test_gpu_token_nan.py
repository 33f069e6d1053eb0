"""Alternatives of rows with NaN: those come first, by their index, wherever they lie, and the rest follow in order."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_token_logprob import KINDS, Case
from token_cases import check_values, exact, load, logits, store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows, vocab", [(40, 1), (40, 18), (40, 64), (40, 300), (40, 2051), (16, 131072), (600, 9001),
                                         (300, 50001), (8200, 1100)])
def test_nan_rows(kind, rows, vocab):
    rng = np.random.RandomState(rows + vocab)
    x = logits(rng, rows, vocab, kind)
    for r in range(min(rows, 40)):
        at = [[0], [vocab - 1], [0, vocab - 1], [vocab // 2], range(0, vocab, 3), range(vocab // 2), range(vocab),
              rng.randint(0, vocab, 4)][r % 8]
        x[r, list(at)] = np.nan
        if r % 16 > 8:
            x[r, vocab // 3] = np.inf
    x = load(store(x, kind))
    tok = rng.randint(0, vocab, rows)
    for top in (1, 5, 32) if rows < 1000 else (5,):
        print(f"nan {kind} {rows}x{vocab} top {top}", flush=True)
        c = Case(x, kind, tok, 1.0, top).forward()
        check_values(c.values(), exact(x, tok, 1.0, top), f"{kind} {rows}x{vocab} top {top}")
