"""A recurrent block trained to name a symbol that it sees through noise: layer norm, a gate and a value for each channel, the gated
recurrence over the sequence, the log-probability of the true symbols, clipping by the gradients' norm, AdamW. Afterwards the
block goes on symbol by symbol from the state that a prompt has left.

    python -m plast_amd.examples.recurrent_block [steps]

A sequence's symbol changes now and then; a channel is a symbol, and a step shows all channels noise and the true one a signal. A
gate decides how long its channel remembers what it has seen.
"""
from __future__ import annotations

import ctypes as C
import sys

import numpy as np

from plast_amd import abi, ops
from plast_amd.graph import Graph
from plast_amd.runtime import DeviceTensor, lib

BATCH, LENGTH, SYMBOLS, EPS, BOUND = 16, 96, 24, 1e-5, 0.5


def draw(rng, batch=BATCH, length=LENGTH, symbols=SYMBOLS):
    """Sequences of symbols, what is seen of them, and how long each is."""
    tokens = rng.randint(0, symbols, (batch, length)).astype(np.int32)
    for t in range(1, length):
        tokens[:, t] = np.where(rng.rand(batch) < 0.95, tokens[:, t - 1], tokens[:, t])
    seen = rng.randn(batch, length, symbols).astype(np.float32)
    seen += 1.5 * (tokens[..., None] == np.arange(symbols))
    lengths = rng.randint(length // 2, length + 1, batch).astype(np.int32)
    return np.where(np.arange(length) < lengths[:, None], tokens, -1).astype(np.int32), seen, lengths


class Block:
    """The block over one batch as a graph: forward() gives the loss, backward() the gradients of the parameters."""

    NAMES = ("weight", "bias", "gate_scale", "gate_bias", "value_scale")

    def __init__(self, rng, tokens, seen, lengths):
        B, T, V = seen.shape
        start = [np.ones(V), np.zeros(V), 0.1 * rng.randn(V), np.ones(V), 1.0 + 0.1 * rng.randn(V)]
        self.params = {n: DeviceTensor.from_numpy(v.astype(np.float32), requires_grad=True) for n, v in zip(self.NAMES, start)}
        self.seen, self.tokens, self.lengths = (DeviceTensor.from_numpy(a) for a in (seen, tokens, lengths))
        p, made = self.params, []

        def t(shape, grad=True):
            made.append(DeviceTensor(shape, requires_grad=grad))
            return made[-1]
        g = self.graph = Graph()
        y = g.node("layer_norm", [self.seen, p["weight"], p["bias"], t((B, T, 2), False)], t((B, T, V)), abi.params(fval=EPS))
        gate = g.node("add", [g.node("mul", [y, p["gate_scale"]], t((B, T, V))), p["gate_bias"]], t((B, T, V)))
        value = g.node("mul", [y, p["value_scale"]], t((B, T, V)))
        chunks = -(-T // abi.RECURRENCE_CHUNK)
        self.last = t((B, V), False)
        self.h = g.node("gated_recurrence", [gate, value, t((B, V), False), self.lengths, self.last, t((B, chunks, V), False)],
                        t((B, T, V)), abi.params(dim=1))
        self.logp = g.node("token_logprob", [self.h, self.tokens, t((B, T, 2), False), t((B, T))], t((B, T)), abi.params(fval=1.0))
        mean = g.node("mean", [self.logp], t((1,)), abi.params(dim=abi.DIM_ALL))
        self.loss = g.node("neg", [mean], t((1,)))
        g.build(self.loss)
        self.made = [x for x in made if x.grad is not None]

    def forward(self) -> float:
        self.graph.forward()
        return float(self.loss.numpy()[0])

    def backward(self) -> None:
        L = lib()
        for x in self.made + list(self.params.values()):
            L.zero_grad_hip(x.p)
        L.set_ones_grad_hip(self.loss.p)
        self.graph.backward()

    def go_on(self, seen, state):
        """One or more steps of every sequence from `state`: what the block says of them, and the state that they leave."""
        p = self.params
        _, y, _ = ops.layer_norm(seen, p["weight"], p["bias"], EPS)
        gate = ops.binary("add", ops.binary("mul", y, p["gate_scale"]), p["gate_bias"])
        inputs, h, _ = ops.gated_recurrence(gate, ops.binary("mul", y, p["value_scale"]), state)
        return h, inputs[4]


def train(steps: int = 60, seed: int = 0):
    """The loss before and after, the gradients' norm in the last step before it was clipped, and the share of the symbols that
    are named right."""
    L, rng = lib(), np.random.RandomState(seed)
    tokens, seen, lengths = draw(rng)
    block = Block(rng, tokens, seen, lengths)
    params = list(block.params.values())
    arr, keep = abi.tensor_array(*[p.t for p in params])
    adamw = abi.AdamW(lr=0.05, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.0)
    before, norm = block.forward(), None
    for _ in range(steps):
        block.forward()
        block.backward()
        norm = ops.clip_grad_norm(params, BOUND)
        L.adamw_step_hip(C.byref(adamw), arr, len(params))
        L.check("adamw_step")
    after = block.forward()
    named = block.h.numpy().argmax(-1)
    live = tokens >= 0
    L.plast_hip_adamw_release(C.byref(adamw), len(params))
    return before, after, float(norm.numpy()[0]) if norm is not None else 0.0, float((named == tokens)[live].mean())


if __name__ == "__main__":
    a, b, norm, share = train(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
    print(f"-log p of the true symbols: {a:.3f} -> {b:.3f}; gradient norm {norm:.3f}; named right: {share:.0%}")
