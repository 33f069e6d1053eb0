"""Layer norm's gradients, the gated recurrence and clipping recorded into a graph by a library that has run nothing yet: what they
leave in the workspace fits the library's fixed array there, with the bits of the eager call."""
from __future__ import annotations

import numpy as np
import pytest

from block_cases import close, device, norm_exact, rounded, stored, values
from plast_amd import abi
from plast_amd.abi import KernelParams
from test_gpu_capture_cold import _replayed, cold  # noqa: F401
from test_gpu_gated_recurrence import Scan, _data
from block_cases import scan_exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape, kind", [((300, 1000), "f32"), ((40, 20000), "f32")])
def test_layer_norm(cold, shape, kind):  # noqa: F811
    from plast_amd import runtime as rt
    print(f"cold capture layer norm {shape}", flush=True)
    rng = np.random.RandomState(1)
    x, dy = rounded(rng.randn(*shape), kind), rounded(rng.randn(*shape), kind)
    w, b = rng.randn(shape[1]).astype(np.float32), rng.randn(shape[1]).astype(np.float32)
    X, Y = rt.DeviceTensor.from_numpy(x, True), rt.DeviceTensor(shape, requires_grad=True)
    W, B = rt.DeviceTensor.from_numpy(w, True), rt.DeviceTensor.from_numpy(b, True)
    cold.arena_memcpy_h2d_hip(Y.grad.ptr, dy.ctypes.data, dy.nbytes)
    S = rt.DeviceTensor((shape[0], 2))

    def call():
        rt.forward("layer_norm", [X, W, B, S], Y, KernelParams(0, 1, 1e-5))
        rt.backward("layer_norm", [X, W, B, S], Y, KernelParams(0, 1, 1e-5))
    got = _replayed(cold, call, [Y, X.grad, W.grad, B.grad])
    want = norm_exact(x, w, b, np.float32(1e-5), dy)
    for g, name in zip(got, ("y", "dx", "dw", "db")):
        close(g, want[name], want[name + "_tol"] + stored(want[name], kind), name)


@pytest.mark.parametrize("shape", [(2, 700, 70), (1, 5000, 40), (3, 60, 20)])
def test_gated_recurrence(cold, shape):  # noqa: F811
    print(f"cold capture recurrence {shape}", flush=True)
    f, v, initial, lengths, dy, dlast = _data(shape, "f32", 17)
    s = Scan(f, v, initial, lengths, "f32", dy, dlast)

    def call():
        s.forward()
        s.backward()
    outs = [s.last, s.f.kept_grad, s.v.kept_grad, s.initial.kept_grad]
    for t in outs + [s.h]:
        t.shape = tuple(t.shape)
    _replayed(cold, call, outs)
    want = scan_exact(f, v, initial, lengths, dy, dlast)
    s.check_forward(want, "cold")
    s.check_backward(want, "cold")


@pytest.mark.parametrize("shape", [(4, 300, 70), (1, 9000, 40)])
def test_a_state_in_place(cold, shape):  # noqa: F811
    """The last state takes the place of the initial one, of which several tiles need a copy beside what they leave each other."""
    print(f"cold capture of a state in place {shape}", flush=True)
    f, v, initial, lengths, _, _ = _data(shape, "f32", 18)
    s = Scan(f, v, initial, lengths, "f32")
    fresh, s.ins[4] = device(initial, "f32"), s.initial

    def call():
        cold.arena_memcpy_d2d_hip(s.initial.ptr, fresh.ptr, initial.nbytes)
        s.forward(keep=False)
    _replayed(cold, call, [s.initial, s.h])
    want = scan_exact(f, v, initial, lengths)
    close(values(s.initial), want["last"], want["last_tol"] + stored(want["last"], "f32"), "state")
    close(values(s.h), want["h"], want["h_tol"] + stored(want["h"], "f32"), "h")


def test_clipping(cold):  # noqa: F811
    """The gradients are scaled in place, so each replay starts from fresh ones."""
    from plast_amd import runtime as rt
    rng = np.random.RandomState(2)
    a = rng.randn(100000).astype(np.float32)
    g, fresh, norm = (device(a, "f32") for _ in range(3))
    norm = rt.DeviceTensor((1,))
    p = abi.make_tensor(g.ptr, (a.size,), None, abi.FLOAT32, abi.GPU, True, g.t)
    arr, keep = abi.tensor_array(p)

    def call():
        cold.arena_memcpy_d2d_hip(g.ptr, fresh.ptr, a.nbytes)
        cold.clip_grad_norm_hip(arr, 1, 3.0, norm.p)
    got = _replayed(cold, call, [g, norm])
    exact = np.sqrt((a.astype(np.float64) ** 2).sum())
    want = a * (3.0 / exact)
    close(got[0], want, np.abs(want) * 4 * 2.0 ** -24, "clipped")
