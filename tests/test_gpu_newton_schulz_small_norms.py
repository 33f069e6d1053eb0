"""Newton-Schulz where eps leaves X small, by rules that take singular values between 1 and 4: what X is scaled by has
to leave them room."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from plast_amd import abi
from test_gpu_newton_schulz import _rt, iterate, near

pytestmark = pytest.mark.gpu
# rules, steps and singular values whose iterates reach more than 2 from below 1/8, and the usual rule's
RULES = [(3.402219960322026, -1.1335748539535262, 0.12480052473758271, 4, 0.10452026818075455),
         (4.2015670464322925, -1.272017426208024, 0.07842315678096642, 4, 0.06538769181422799),
         (2.690574991448999, -0.20633512950177474, 0.004332192231654639, 4, 0.12435024050760021),
         (3.4445, -4.775, 2.0315, 5, 0.1), (3.4445, -4.775, 2.0315, 5, 1e-6), (1.0, 0.5, 0.0, 2, 0.45)]


@pytest.mark.parametrize("rule", RULES, ids=[f"{r[0]:.3f}-{r[4]:.2g}" for r in RULES])
def test_small_norms(rule):
    a, b, c, steps, x = rule
    rt = _rt()
    rng = np.random.RandomState(3)
    for shape in ((1, 1), (40, 90), (200, 150)):
        print(f"newton_schulz small norms {rule} {shape}", flush=True)
        g = np.outer(rng.randn(shape[0]), rng.randn(shape[1]))
        g = (g / np.linalg.norm(g) * x / (1 - x)).astype(np.float32)   # with eps = 1: a singular value of x
        t, out = rt.DeviceTensor.from_numpy(g), rt.DeviceTensor(g.shape, zero=False)
        r = abi.NewtonSchulz(a, b, c, 1.0, steps)
        rt.lib().newton_schulz_hip(C.byref(t.t), C.byref(out.t), C.byref(r))
        rt.lib().check("newton_schulz")
        near(out.numpy(), iterate(g, steps, a, b, c, 1.0), 3.3e-4, "f32", f"{rule} {shape}")
