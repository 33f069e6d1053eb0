"""Both sides of the gated recurrence's gates to some roundings of fp32 of themselves, however far out the gate is."""
from __future__ import annotations

import numpy as np
import pytest

from block_cases import U, device, give, values
from plast_amd.abi import RECURRENCE_CHUNK, KernelParams

pytestmark = pytest.mark.gpu

# Half steps of fp32 relative to the value. The exponential and the reciprocal are off by a whole step each, 2; what the
# exponential's argument has lost is brought back in one rounding. So e: 3; 1 / (1 + e): at most 3 and its share of e's, below 5; e / (1 + e):
# 3 + 1 + 2 and the product's 1.
LARGE, SMALL = 5, 7


@pytest.mark.parametrize("length", [1, 40, 300])
def test_sides_of_gates_far_out(length):
    """Sequences of one step, padded to none, within a tile and over several: from a state of 0 h is z v, and with a value of 0 it is
    a times the state; dv is z dy, df is dy (h[-1] - v) a z and the initial state's gradient a dy. Every product's rounding is one
    more, and df's difference of the state and the value another."""
    from plast_amd.runtime import DeviceTensor, backward, forward
    B, D = 16, 1001
    rng = np.random.RandomState(length)
    f1 = rng.uniform(-80, 80, (B, D)).astype(np.float32)
    v1, h1, dy1 = (rng.uniform(0.5, 1, (B, D)).astype(np.float32) for _ in range(3))
    zero = np.zeros((B, D), np.float32)
    e = np.exp(-np.abs(f1.astype(np.float64)))
    large, small = 1 / (1 + e), e / (1 + e)
    a, z = np.where(f1 > 0, large, small), np.where(f1 > 0, small, large)
    a_tol, z_tol = np.where(f1 > 0, LARGE, SMALL), np.where(f1 > 0, SMALL, LARGE)

    def sequence(step):
        out = np.full((B, length, D), 3.0, np.float32)
        out[:, 0] = step
        return out

    def near(got, want, steps, what):
        bad = np.abs(got - want) > np.abs(want) * steps * U * (1 + 2.0 ** -10)
        assert not bad.any(), (what, f1[bad][0], got[bad][0], want[bad][0])

    for v, h0 in ((v1, zero), (zero, h1), (v1, -h1)):
        print(f"gates far out, length {length}", flush=True)
        F = device(sequence(f1), "f32", grad=device(sequence(0), "f32"))
        V = device(sequence(v), "f32", grad=device(sequence(0), "f32"))
        initial, last = device(h0, "f32", grad=device(zero, "f32")), device(zero, "f32")
        H = give(device(sequence(0), "f32"), device(sequence(dy1), "f32"))
        states = DeviceTensor((B, -(-length // RECURRENCE_CHUNK), D))
        ins = [F, V, initial, DeviceTensor.from_numpy(np.ones(B, np.int32)), last, states]
        forward("gated_recurrence", ins, H, KernelParams(1, 0, 0.0))
        if not (v.any() and h0.any()):
            want, steps = (z * v, z_tol + 1) if v.any() else (a * h0, a_tol + 1)
            near(values(H)[:, 0], want, steps, "h")
            near(values(last), want, steps, "last")
        backward("gated_recurrence", ins, H, KernelParams(1, 1, 0.0))
        near(values(V.kept_grad)[:, 0], z * dy1, z_tol + 1, "dv")
        near(values(initial.kept_grad), a * dy1, a_tol + 1, "dinitial")
        near(values(F.kept_grad)[:, 0], dy1 * (h0.astype(np.float64) - v) * a * z, LARGE + SMALL + 4, "df")
        for t in (V, F):
            assert not values(t.kept_grad)[:, 1:].any()
