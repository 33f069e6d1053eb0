"""Token log-probabilities recorded into a graph by a library that has run nothing yet: rows cut over workgroups, the
step in two passes, the streaming step. Newton-Schulz asks for a run beforehand."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from plast_amd import abi
from test_gpu_capture_cold import _replayed, cold  # noqa: F401
from test_gpu_token_logprob import Case
from token_cases import check_gradient, check_values, exact, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, vocab, kind, top", [(1, 131072, "bf16", 20), (40, 50001, "f16", 5), (3, 200003, "f32", 0)])
def test_rows_cut_over_workgroups(cold, rows, vocab, kind, top):  # noqa: F811
    print(f"cold capture {kind} {rows}x{vocab} top {top}", flush=True)
    rng = np.random.RandomState(rows)
    x, tok = logits(rng, rows, vocab, kind), rng.randint(0, vocab, rows)
    c = Case(x, kind, tok, 1.0, top)
    _replayed(cold, c.forward, [c.logp, c.entropy, c.stats] + ([c.tl, c.ti] if top else []))
    check_values(c.values(), exact(x, tok, 1.0, top), f"{kind} {rows}x{vocab}")


@pytest.mark.parametrize("rows, vocab", [(20, 70000), (1100, 20000)])
def test_step(cold, rows, vocab):  # noqa: F811
    print(f"cold capture step {rows}x{vocab}", flush=True)
    rng = np.random.RandomState(rows)
    x, tok = logits(rng, rows, vocab, "f32"), rng.randint(0, vocab, rows)
    u, h = rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)
    c = Case(x, "f32", tok, 1.0, 0, u, h)
    _replayed(cold, c.step, [c.logp, c.entropy, c.dx_t])
    want = exact(x, tok, 1.0, 0, u, h)
    check_values(c.values(), want, f"step {rows}x{vocab}")
    check_gradient(c.dx(), want, "f32", f"step {rows}x{vocab}")


def test_newton_schulz_needs_its_workspace(cold):  # noqa: F811
    from plast_amd import runtime as rt
    g, out = rt.DeviceTensor.from_numpy(np.ones((8, 8), np.float32)), rt.DeviceTensor((8, 8))
    rule = abi.NewtonSchulz(3.4445, -4.775, 2.0315, 1e-7, 5)
    assert cold.plast_hip_capture_begin() == 0
    cold.newton_schulz_hip(C.byref(g.t), C.byref(out.t), C.byref(rule))
    graph = cold.plast_hip_capture_end()
    with pytest.raises(rt.PlastHipError, match="run the work once before"):
        cold.check()
    cold.plast_hip_graph_destroy(graph)
    assert not out.numpy().any()
