"""Muon's moments and graphs: the step that makes them is refused in a capture, later ones replay as they run."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from plast_amd import abi

pytestmark = pytest.mark.gpu


def test_moments_are_made_outside_captures():
    from plast_amd import runtime as rt
    L = rt.lib()
    rng = np.random.RandomState(1)
    p = rt.DeviceTensor.from_numpy(rng.randn(40, 30).astype(np.float32), requires_grad=True)
    g = rng.randn(40, 30).astype(np.float32)
    L.arena_memcpy_h2d_hip(p.grad.ptr, g.ctypes.data, g.nbytes)
    arr, keep = abi.tensor_array(p.t)
    assert L.plast_hip_workspace_reserve(0, 1 << 24) == 0

    def optimizer():
        return abi.Muon(0.02, 0.9, 0.0, 1, abi.NewtonSchulz(3.4445, -4.775, 2.0315, 1e-7, 5), None)

    def capture(o):
        assert L.plast_hip_capture_begin() == 0
        L.muon_step_hip(C.byref(o), arr, 1)
        return L.plast_hip_capture_end()

    before = p.numpy()
    fresh = optimizer()
    graph = capture(fresh)
    with pytest.raises(rt.PlastHipError, match="run one before capturing"):
        L.check()
    L.plast_hip_graph_destroy(graph)
    assert not fresh.m and np.array_equal(p.numpy(), before)

    eager, replayed = optimizer(), optimizer()
    for _ in range(4):
        L.muon_step_hip(C.byref(eager), arr, 1)
    L.check()
    want = p.numpy()
    L.arena_memcpy_h2d_hip(p.ptr, before.ctypes.data, before.nbytes)
    L.muon_step_hip(C.byref(replayed), arr, 1)
    graph = capture(replayed)
    L.check()
    for _ in range(3):
        assert L.plast_hip_graph_launch(graph) == 0
    assert np.array_equal(p.numpy(), want)
    L.plast_hip_graph_destroy(graph)
    for o in (eager, replayed):
        L.plast_hip_muon_release(C.byref(o), 1)
