"""Nodes that read what token_logprob writes beside its output (entropy, alternatives) come after it, in
whatever order a loss names them. Building a graph touches structs only, so no GPU is needed."""
from __future__ import annotations

import ctypes as C

import pytest

from plast_amd import abi
from plast_amd import graph as graph_module
from plast_amd.graph import Graph


class _Lib:
    def plast_hip_get_op_impl(self, op):
        return abi.Op()


class _Tensor:
    def __init__(self):
        self.t = abi.Tensor()


@pytest.fixture()
def parts(monkeypatch):
    monkeypatch.setattr(graph_module, "lib", lambda: _Lib())
    g = Graph()
    x, tokens, stats, entropy, top_logp, top_ids, logp = (_Tensor() for _ in range(7))
    g.node("exp", [_Tensor()], x)
    g.node("token_logprob", [x, tokens, stats, entropy, top_logp, top_ids], logp)
    return g, logp, entropy, stats, top_logp


def _order(g, root):
    assert g.build(root) == 0
    return g.op_types()


def test_loss_over_the_entropy_alone(parts):
    g, _, entropy, _, _ = parts
    loss = g.node("mean", [entropy], _Tensor())
    assert _order(g, loss) == ["EXP", "TOKEN_LOGPROB", "MEAN"]
    assert _order(g, entropy) == ["EXP", "TOKEN_LOGPROB"]


@pytest.mark.parametrize("entropy_first", [False, True])
def test_loss_over_both(parts, entropy_first):
    g, logp, entropy, _, _ = parts
    a, b = g.node("sum", [logp], _Tensor()), g.node("mean", [entropy], _Tensor())
    loss = g.node("add", [b, a] if entropy_first else [a, b], _Tensor())
    assert _order(g, loss) == ["EXP", "TOKEN_LOGPROB"] + (["MEAN", "SUM"] if entropy_first else ["SUM", "MEAN"]) + ["ADD"]


def test_statistics_and_alternatives(parts):
    g, _, _, stats, top_logp = parts
    loss = g.node("add", [g.node("sum", [top_logp], _Tensor()), g.node("mean", [stats], _Tensor())], _Tensor())
    assert _order(g, loss) == ["EXP", "TOKEN_LOGPROB", "SUM", "MEAN", "ADD"]


def test_what_a_node_only_reads_keeps_its_creator(parts):
    g, _, _, _, _ = parts
    node = g.nodes[1]
    assert node.inputs[0].contents.creator == C.addressof(g.nodes[0])
    assert not node.inputs[1].contents.creator
    assert all(node.inputs[i].contents.creator == C.addressof(node) for i in range(2, 6))
