"""Rows of 257 to 640 16-byte units on each side of the number of rows from which a wave takes one by itself."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_token_logprob import Case
from token_cases import check_values, exact, logits, special

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind, vocab", [("f32", 1027), ("f32", 2561), ("f32", 2564), ("bf16", 2061), ("f16", 5121)])
@pytest.mark.parametrize("rows", [3999, 4000])
def test_row_counts(kind, rows, vocab):
    rng = np.random.RandomState(vocab)
    x, tok = special(logits(rng, rows, vocab, kind, 0.2), kind), rng.randint(0, vocab, rows)
    for top in (0, 7):
        print(f"row counts {kind} {rows}x{vocab} top {top}", flush=True)
        c = Case(x, kind, tok, 1.0, top).forward()
        check_values(c.values(), exact(x, tok, 1.0, top), f"{kind} {rows}x{vocab} top {top}")
