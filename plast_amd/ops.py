"""Functional layer over the HIP entry points, shaped like the reference's Python `Tensor` methods
(plast/tensor.py): it computes output shapes the same way, allocates the output and calls the op.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import abi
from .abi import BFLOAT16, DIM_ALL, FLOAT32, INT32, INT64, KernelParams
from .runtime import DeviceTensor, backward, forward, lib


def broadcast_shape(s1, s2) -> tuple[int, ...]:
    """numpy broadcasting, raising on incompatible shapes (plast/tensor.py:74-93)."""
    n = max(len(s1), len(s2))
    out = []
    for i in range(n):
        a = s1[len(s1) - 1 - i] if i < len(s1) else 1
        b = s2[len(s2) - 1 - i] if i < len(s2) else 1
        if a != b and a != 1 and b != 1:
            raise ValueError(f"shapes {tuple(s1)} and {tuple(s2)} are not broadcastable")
        out.append(max(a, b))
    return tuple(reversed(out))


def binary(name: str, a: DeviceTensor, b: DeviceTensor, requires_grad: bool = False) -> DeviceTensor:
    out = DeviceTensor(broadcast_shape(abi.shape_of(a.t), abi.shape_of(b.t)), FLOAT32,
                       requires_grad, zero=False)
    forward(name, [a, b], out)
    return out


def unary(name: str, a: DeviceTensor, alpha: float = 0.0, requires_grad: bool = False) -> DeviceTensor:
    out = DeviceTensor(abi.shape_of(a.t), FLOAT32, requires_grad, zero=False)
    forward(name, [a], out, KernelParams(0, 0, alpha))
    return out


def reduced_shape(shape, dim, keepdim) -> tuple[int, ...]:
    """Output shape of a reduction (plast/tensor.py:597-659)."""
    if dim is None:
        return (1,)
    out = list(shape)
    if keepdim:
        out[dim] = 1
    else:
        out.pop(dim)
        if not out:
            out = [1]
    return tuple(out)


def reduce(name: str, a: DeviceTensor, dim=None, keepdim: bool = False,
           requires_grad: bool = False) -> DeviceTensor:
    shape = abi.shape_of(a.t)
    if dim is not None and dim < 0:
        dim += len(shape)
    dt = INT64 if name == "argmax" else FLOAT32
    out = DeviceTensor(reduced_shape(shape, dim, keepdim), dt, requires_grad, zero=False)
    forward(name, [a], out, KernelParams(DIM_ALL if dim is None else dim, int(keepdim), 0.0))
    return out


def transpose(a: DeviceTensor, d0: int, d1: int) -> DeviceTensor:
    """A view with two axes swapped (shape_ops.c:59-80), sharing a's buffer."""
    v = DeviceTensor(abi.shape_of(a.t), a.dtype, base=a.base or a, zero=False)
    v.t.data = a.t.data
    forward("transpose", [a], v, KernelParams(d0, d1, 0.0))
    v.shape = abi.shape_of(v.t)
    return v


def permute(a: DeviceTensor, dims) -> DeviceTensor:
    """As a sequence of transposes, the way plast/tensor.py:730-756 builds it."""
    cur = list(range(len(dims)))
    res = a
    for target, orig in enumerate(dims):
        pos = cur.index(orig)
        if pos != target:
            res = transpose(res, pos, target)
            cur[pos], cur[target] = cur[target], cur[pos]
    return res


def expand(a: DeviceTensor, shape) -> DeviceTensor:
    v = DeviceTensor(tuple(shape), a.dtype, base=a.base or a, zero=False)
    forward("expand", [a], v)
    return v


def softmax_cross_entropy(logits: DeviceTensor, labels: DeviceTensor, requires_grad: bool = False):
    """Per-row loss [N] and stats [N, 2] (row max, log exp-sum)."""
    n = abi.shape_of(logits.t)[0]
    stats = DeviceTensor((n, 2), FLOAT32, zero=False)
    loss = DeviceTensor((n,), FLOAT32, requires_grad, zero=False)
    forward("softmax_cross_entropy", [logits, labels, stats], loss)
    return loss, stats


def bfloat16_bits(values) -> np.ndarray:
    """The bit patterns (uint16, what a BFLOAT16 tensor's host image holds) of float32 values rounded
    to the nearest bfloat16, ties to even."""
    v = np.ascontiguousarray(values, np.float32)
    b = v.view(np.uint32).astype(np.uint64)
    b = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(v), np.uint16(0x7FC0), b)


def bfloat16_values(bits) -> np.ndarray:
    """The float32 values of bfloat16 bit patterns."""
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def token_logprob(x: DeviceTensor, tokens: DeviceTensor, temperature: float = 1.0, top: int = 0,
                  requires_grad: bool = False):
    """Log-probability of each row's token under softmax(x / temperature) and the row's entropy, with
    the `top` most likely alternatives. Returns (inputs, logp, params): `inputs` are
    [x, tokens, stats, entropy] and, with top > 0, top_logp and top_ids; backward("token_logprob",
    inputs, logp, params) accumulates into x's gradient from those of logp and entropy."""
    lead = abi.shape_of(x.t)[:-1]
    stats = DeviceTensor(lead + (2,), FLOAT32, zero=False)
    entropy = DeviceTensor(lead, FLOAT32, requires_grad, zero=False)
    logp = DeviceTensor(lead, FLOAT32, requires_grad, zero=False)
    inputs = [x, tokens, stats, entropy]
    if top:
        inputs += [DeviceTensor(lead + (top,), FLOAT32, zero=False),
                   DeviceTensor(lead + (top,), INT32, zero=False)]
    p = KernelParams(top, 0, temperature)
    forward("token_logprob", inputs, logp, p)
    return inputs, logp, p


def newton_schulz(g: DeviceTensor, steps: int = 5, a: float = 3.4445, b: float = -4.7750,
                  c: float = 2.0315, eps: float = 1e-7) -> DeviceTensor:
    """The orthogonalised g, a matrix or a stack of matrices (newton_schulz_hip)."""
    out = DeviceTensor(abi.shape_of(g.t), g.dtype, zero=False)
    rule = abi.NewtonSchulz(a, b, c, eps, steps)
    lib().newton_schulz_hip(C.byref(g.t), C.byref(out.t), C.byref(rule))
    lib().check("newton_schulz")
    return out


def make_tape(instructions, num_inputs: int) -> abi.FusedTape:
    """instructions: list of (op_name, src, idx, acc_rhs, imm)."""
    tape = abi.FusedTape()
    tape.num_inputs = num_inputs
    tape.num_ins = len(instructions)
    for i, (op, src, idx, rhs, imm) in enumerate(instructions):
        tape.ins[i] = abi.TapeIns(abi.TAPE[op], src, idx, rhs, imm)
    return tape


def fused(tape: abi.FusedTape, inputs, shape) -> DeviceTensor:
    out = DeviceTensor(tuple(shape), FLOAT32, zero=False)
    forward("fused_elementwise", inputs, out,
            KernelParams(C.addressof(tape), 0, 0.0))
    return out


__all__ = ["binary", "unary", "reduce", "transpose", "permute", "expand", "softmax_cross_entropy",
           "token_logprob", "newton_schulz", "bfloat16_bits", "bfloat16_values", "BFLOAT16", "make_tape", "fused", "broadcast_shape", "reduced_shape", "backward", "forward", "lib",
           "DeviceTensor", "np", "INT32"]
