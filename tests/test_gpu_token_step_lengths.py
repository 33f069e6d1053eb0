"""The one-pass step over rows on each side of what a workgroup's registers hold, aligned and not: 65536 logits or one
unit less, by alignment (float32 rows of more than 32768 where they fill the chip), and the powers of two below."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_token_logprob import Case
from token_cases import check_gradient, check_values, exact, logits, special

pytestmark = pytest.mark.gpu
LENGTHS = {"f32": [8192, 16384, 32764, 32767, 32768, 32769, 65530, 65535, 65536, 65537],
           "f16": [8192, 65528, 65535, 65536, 65537, 100001, 131058, 131071, 131072, 131073],
           "bf16": [16384, 65536, 65537, 131058, 131072]}


def _step(kind, rows, vocab, up=0, offset=0):
    rng = np.random.RandomState(vocab)
    x, tok = special(logits(rng, rows, vocab, kind, 0.1), kind), rng.randint(0, vocab, rows)
    tok[1::5] = -1
    tok[2::5] = vocab - 1
    u, h = rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)
    print(f"step {kind} {rows}x{vocab} pitch +{up} offset {offset}", flush=True)
    want = exact(x, tok, 0.9, 0, u, h)
    strides = (vocab + up, 1)
    c = Case(x, kind, tok, 0.9, 0, u, h, strides=strides, offset=offset, grad_strides=strides, grad_offset=offset).step()
    check_values(c.values(), want, f"step {kind} {rows}x{vocab}")
    check_gradient(c.dx(), want, kind, f"step {kind} {rows}x{vocab}")


@pytest.mark.parametrize("kind, vocab", [(k, v) for k, vs in LENGTHS.items() for v in vs])
def test_lengths(kind, vocab):
    for up, offset in ((0, 0), (1, 3)):
        _step(kind, 12, vocab, up, offset)


@pytest.mark.parametrize("vocab", [32772, 65536, 65535])
def test_long_rows_that_fill_the_chip(vocab):
    _step("f32", 260, vocab)
    _step("f32", 260, vocab, 1, 3)


@pytest.mark.parametrize("vocab", [16388, 32764, 32768])
def test_streaming_rows(vocab):
    """Rows of whole 16-byte units, more than four for each compute unit."""
    _step("f32", 1100, vocab)
    _step("f32", 1100, vocab, 4)
