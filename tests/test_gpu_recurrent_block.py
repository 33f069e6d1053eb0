"""The new operators as they are used together: a block trained as a graph (layer norm, gate and value, gated recurrence, token
log-probabilities), its gradients clipped and stepped by AdamW, and a decoder that goes on from a prompt's state in a captured
graph. Gradients against torch's in 64 bits on the CPU."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from block_cases import U, close, device, norm_exact, rounded, scan_exact, stored, values
from plast_amd import abi
from plast_amd.abi import KernelParams
from plast_amd.examples import recurrent_block as rb

pytestmark = pytest.mark.gpu


def _torch_loss(params, tokens, seen, lengths):
    p = {n: torch.tensor(v, dtype=torch.float64, requires_grad=True) for n, v in params.items()}
    x = torch.tensor(seen, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(x, x.shape[-1:], p["weight"], p["bias"], float(np.float32(rb.EPS)))
    a = torch.sigmoid(y * p["gate_scale"] + p["gate_bias"])
    v = y * p["value_scale"]
    h, out = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * v[:, t]
        out.append(h)
    lp = torch.log_softmax(torch.stack(out, 1), -1)
    tok = torch.tensor(tokens.astype(np.int64))
    logp = torch.where(tok >= 0, lp.gather(-1, tok.clamp(min=0)[..., None])[..., 0], 0.0)
    loss = -logp.mean()
    loss.backward()
    return float(loss.detach()), {n: t.grad.numpy() for n, t in p.items()}


def test_training_step():
    from plast_amd import ops
    from plast_amd.runtime import lib
    rng = np.random.RandomState(3)
    tokens, seen, lengths = rb.draw(rng)
    block = rb.Block(rng, tokens, seen, lengths)
    for _ in range(2):  # twice, and nothing left over from the first pass
        before = {n: p.numpy() for n, p in block.params.items()}
        want, grads = _torch_loss(before, tokens, seen, lengths)
        got = block.forward()
        # a loss of some hundred roundings of values around it
        assert abs(got - want) < 512 * U * abs(want)
        block.backward()
        # sums over 1536 rows of products of some hundred roundings each; most of a sum cancels, a tenth of it is left here
        for n, p in block.params.items():
            scale = np.abs(grads[n]).max()
            assert np.abs(p.grad.numpy() - grads[n]).max() < 10 * 1536 * U * scale, n
    exact = np.sqrt(sum((p.grad.numpy().astype(np.float64) ** 2).sum() for p in block.params.values()))
    raw = {n: p.grad.numpy() for n, p in block.params.items()}
    params = list(block.params.values())
    bound = float(np.float32(exact / 4))
    norm = ops.clip_grad_norm(params, bound).numpy()[0]
    assert abs(norm - exact) <= 1.01 * U * exact
    for n, p in block.params.items():
        close(p.grad.numpy(), raw[n].astype(np.float64) * (bound / exact), np.abs(raw[n]) * U + 2.0 ** -149, n)
    L = lib()
    adamw = abi.AdamW(lr=0.05, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.0)
    arr, keep = abi.tensor_array(*[p.t for p in params])
    L.adamw_step_hip(C.byref(adamw), arr, len(params))
    L.check()
    for n, p in block.params.items():
        # Adam's first step is lr times the sign, less what eps takes: sqrt((1 - beta2) g^2) beside 1e-8
        g = np.abs(raw[n]).astype(np.float64) * (bound / exact)
        big = g > 1e-4
        moved = before[n] - p.numpy()
        assert big.any() and np.abs(np.abs(moved[big]) - 0.05).max() < 0.05 * 0.002
        assert (np.sign(moved[big]) == np.sign(raw[n][big])).all()
    L.plast_hip_adamw_release(C.byref(adamw), len(params))


def test_the_example_runs():
    before, after, norm, share = rb.train(3)
    assert all(np.isfinite(v) for v in (before, after, norm)) and 0.0 <= share <= 1.0 and norm > 0.0


def test_going_on_from_a_prompt():
    """The prompt's last state and the rest step by step, against the whole sequence."""
    rng = np.random.RandomState(5)
    tokens, seen, _ = rb.draw(rng)
    block = rb.Block(rng, tokens, seen, np.full(rb.BATCH, rb.LENGTH, np.int32))
    block.forward()
    whole = block.h.numpy()
    from plast_amd.runtime import DeviceTensor
    zero = DeviceTensor((rb.BATCH, rb.SYMBOLS))
    _, state = block.go_on(DeviceTensor.from_numpy(seen[:, :70]), zero)
    for t in range(70, rb.LENGTH):
        h, state = block.go_on(DeviceTensor.from_numpy(np.ascontiguousarray(seen[:, t:t + 1])), state)
        # convex steps of values up to some four: 96 of them, eight roundings each
        assert np.abs(h.numpy()[:, 0] - whole[:, t]).max() < 96 * 8 * U * 4


def test_a_captured_decoder():
    """Layer norm and one step of the recurrence with the state in place, captured once and replayed token by token with new inputs,
    two decoders of other sizes in turn."""
    from plast_amd import runtime as rt
    L = rt.lib()
    rng = np.random.RandomState(6)
    made = []
    for B, D, kind in ((5, 70, "f32"), (64, 512, "bf16")):
        T = 9
        x = rounded(rng.randn(B, T, D), kind)
        w, b, init = (1 + 0.1 * rng.randn(D)).astype(np.float32), (0.1 * rng.randn(D)).astype(np.float32), rng.randn(B, D).astype(np.float32)
        f = rounded(rng.randn(B, T, D) + 1.0, kind)
        X, F = device(x[:, :1], kind), device(f[:, :1], kind)
        W, Bi, S = device(w, "f32"), device(b, "f32"), rt.DeviceTensor((B, 1, 2))
        V, H = device(np.zeros((B, 1, D)), kind), device(np.zeros((B, 1, D)), kind)
        state, lengths = device(init, "f32"), rt.DeviceTensor.from_numpy(np.ones(B, np.int32))

        def call():
            rt.forward("layer_norm", [X, W, Bi, S], V, KernelParams(0, 0, rb.EPS))
            rt.forward("gated_recurrence", [F, V, state, lengths, state], H, KernelParams(0, 0, 0.0))
        call()
        assert L.plast_hip_capture_begin() == 0
        call()
        graph = L.plast_hip_capture_end()
        L.check("capture")
        back = device(init, "f32")
        L.arena_memcpy_d2d_hip(state.ptr, back.ptr, B * D * 4)
        norm = norm_exact(x.reshape(-1, D), w, b, np.float32(rb.EPS))
        made.append((B, T, D, kind, x, f, norm, X, F, V, H, state, graph, init, [], (W, Bi, S, lengths)))  # a graph's buffers live as long as it does
    for t in range(9):
        for B, T, D, kind, x, f, norm, X, F, V, H, state, graph, init, got, _ in made:
            for to, values_ in ((X, x), (F, f)):
                new = device(values_[:, t:t + 1], kind)
                L.arena_memcpy_d2d_hip(to.ptr, new.ptr, B * D * to.itemsize)
            assert L.plast_hip_graph_launch(graph) == 0
            got.append((values(V)[:, 0], values(H)[:, 0]))
    for B, T, D, kind, x, f, norm, X, F, V, H, state, graph, init, got, _ in made:
        v = np.stack([g[0] for g in got], 1)
        y = norm["y"].reshape(B, T, D)
        close(v, y, norm["y_tol"].reshape(B, T, D) + stored(y, kind), "norm")
        want = scan_exact(f, v, init, [T] * B)
        close(np.stack([g[1] for g in got], 1), want["h"], want["h_tol"] + stored(want["h"], kind), "h")
        close(values(state), want["last"], want["last_tol"] + stored(want["last"], "f32"), "state")
        L.plast_hip_graph_destroy(graph)
