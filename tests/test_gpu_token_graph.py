"""Losses over token_logprob's results as graphs: the entropy alone, and both results in either order."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from plast_amd.abi import DIM_ALL, KernelParams
from token_cases import check_gradient, close, exact, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("loss", ["entropy", "logp then entropy", "entropy then logp"])
def test_losses(loss):
    from plast_amd.graph import Graph
    from plast_amd.runtime import DeviceTensor, lib
    rng = np.random.RandomState(len(loss))
    n, vocab = 12, 75
    x, tok = logits(rng, n, vocab, "f32"), rng.randint(0, vocab, n).astype(np.int32)
    X, T = DeviceTensor.from_numpy(x, requires_grad=True), DeviceTensor.from_numpy(tok)
    stats, entropy, logp = DeviceTensor((n, 2)), DeviceTensor((n,), requires_grad=True), DeviceTensor((n,), requires_grad=True)
    g = Graph()
    g.node("token_logprob", [X, T, stats, entropy], logp, KernelParams(0, 0, 1.0))
    means = {k: g.node("mean", [t], DeviceTensor((1,), requires_grad=True), KernelParams(DIM_ALL, 0, 0.0))
             for k, t in (("logp", logp), ("entropy", entropy))}
    names = loss.split(" then ")
    root = means[names[0]]
    if len(names) > 1:
        root = g.node("add", [means[k] for k in names], DeviceTensor((1,), requires_grad=True))
    g.build(root, fuse=True)
    w = {k: np.full(n, 1.0 / n if k in names else 0.0, np.float32) for k in means}
    for step in range(2):  # with other logits, and nothing left over from the first pass
        want = exact(x, tok, 1.0, 0, w["logp"], w["entropy"])
        g.forward()
        value = sum(want[k].mean() for k in names)
        close(root.numpy()[0], value, 1e-5 + 1e-6 * sum(np.abs(want[k]).mean() for k in names), f"{loss} {step}")
        for t in [X, logp, entropy, *means.values(), root]:
            lib().zero_grad_hip(C.byref(t.t))
        lib().set_ones_grad_hip(C.byref(root.t))
        g.backward()
        check_gradient(X.grad.numpy(), want, "f32", f"{loss} {step}")
        x = logits(rng, n, vocab, "f32")
        lib().arena_memcpy_h2d_hip(X.ptr, x.ctypes.data, x.nbytes)
