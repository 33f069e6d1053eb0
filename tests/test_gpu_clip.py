"""Clipping by the global norm of all gradients, against 64 bits: the norm is rounded to fp32 once, a clipped gradient by its
factor (64 bits) and its type."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from block_cases import U, around, close, device, give, rounded, stored, values
from plast_amd import abi

pytestmark = pytest.mark.gpu


def _params(grads):
    """Parameters of these gradients (device tensors); their own values are never looked at."""
    out = []
    for g in grads:
        p = abi.make_tensor(g.ptr, g.shape, None, abi.FLOAT32, abi.GPU, True, g.t)
        out.append(p)
    return out


def _clip(params, bound, norm=None):
    from plast_amd.runtime import lib
    arr, keep = abi.tensor_array(*params)
    lib().clip_grad_norm_hip(arr, len(params), bound, C.byref(norm.t) if norm is not None else None)
    lib().check("clip")


def _check(arrays, kinds, ratio, leads=None):
    from plast_amd.runtime import DeviceTensor
    leads = leads or [0] * len(arrays)
    arrays = [rounded(a, k) for a, k in zip(arrays, kinds)]
    grads = [device(a.reshape(-1), k, lead) for a, k, lead in zip(arrays, kinds, leads)]
    exact = np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays))
    bound = float(np.float32(ratio * exact))
    norm = DeviceTensor((1,))
    _clip(_params(grads), bound, norm)
    # a norm below 2^-126 is a subnormal number: fp32's are 2^-149 apart
    close(norm.numpy()[0], exact, exact * U * 1.01 + 2.0 ** -150, "norm")
    scale = bound / exact if exact > bound else 1.0
    for k, (a, g, kind) in enumerate(zip(arrays, grads, kinds)):
        want = a.astype(np.float64).reshape(-1) * scale
        # rounded to fp32 on the way to 16 bits; the norm's 64-bit sum is off by far less
        tol = 0.0 if scale == 1.0 else stored(want, kind) + np.abs(want) * 2 * U + 2.0 ** -149
        close(values(g), want, tol, f"gradient {k} of {a.shape} {kind}")
        assert (around(g, kind) == rounded(77.0, kind)).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes", [[1], [2, 3], [255, 256, 257], [4096], [16384, 16383, 5], [100003], [7] * 90, [1000] * 97, [33] * 300, [5] * 160, [9] * 161, [70] * 330,
                                   [3000001, 1, 65536]])
def test_sizes(sizes, kind):
    rng = np.random.RandomState(len(sizes))
    for ratio in (0.3, 1.5):
        print("clip", kind, sizes[:4], len(sizes), ratio, flush=True)
        _check([rng.randn(n) for n in sizes], [kind] * len(sizes), ratio)


def test_types_and_addresses_together():
    rng = np.random.RandomState(0)
    sizes = [5000, 70001, 3, 40000, 12345, 8192]
    kinds = ["f32", "bf16", "f16", "f16", "bf16", "f32"]
    for leads in ([0] * 6, [1, 1, 1, 3, 5, 2]):
        for ratio in (0.01, 0.999, 1.001):
            _check([rng.randn(n) * (1 + k) for k, n in enumerate(sizes)], kinds, ratio, leads)


def test_extremes():
    """Squares beyond fp32 in both directions, a norm beyond it too, a bound of zero."""
    from plast_amd.runtime import DeviceTensor
    rng = np.random.RandomState(1)
    _check([rng.randn(1000) * 1e30], ["f32"], 1e-3)
    _check([rng.randn(1000) * 1e-30], ["f32"], 0.5)
    _check([rng.randn(1000) * 1e-41], ["f32"], 2.0)
    _check([rng.randn(5000) * 300], ["f16"], 0.5)
    g = device(np.full(1000, 3e38), "f32")
    norm = DeviceTensor((1,))
    _clip(_params([g]), 1.0, norm)
    assert np.isinf(norm.numpy()[0])
    close(values(g), np.full(1000, 1000 ** -0.5), 4 * U, "beyond fp32")
    g = device(rng.randn(500), "f32")
    _clip(_params([g]), 0.0)
    assert not values(g).any()
    _clip(_params([g]), 0.0, norm)   # nothing left
    assert norm.numpy()[0] == 0


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_norm_that_is_no_number_leaves_all_as_it_is(bad, kind):
    from plast_amd.runtime import DeviceTensor
    a, b = np.arange(1, 3001, dtype=np.float32) % 128, np.ones(40000, np.float32)
    b[12345] = bad
    grads = [device(a, kind), device(b, kind)]
    norm = DeviceTensor((1,))
    _clip(_params(grads), 0.1, norm)
    assert np.isnan(norm.numpy()[0]) if np.isnan(bad) else np.isinf(norm.numpy()[0])
    assert np.array_equal(values(grads[0]), a) and np.array_equal(values(grads[1]), b, equal_nan=True)


def test_an_infinite_bound_computes_the_norm():
    from plast_amd import ops
    from plast_amd.runtime import DeviceTensor
    a = np.random.RandomState(2).randn(40, 50).astype(np.float32)
    p = give(DeviceTensor((40, 50)), device(a, "f32"))
    norm = ops.clip_grad_norm([p], float("inf")).numpy()[0]
    exact = np.sqrt((a.astype(np.float64) ** 2).sum())
    close(norm, exact, exact * U * 1.01, "norm")
    assert np.array_equal(values(p.kept_grad), a)


def test_what_is_skipped():
    """NULL parameters, parameters without a gradient, and empty ones."""
    from plast_amd.runtime import DeviceTensor, lib
    a = np.random.RandomState(3).randn(300).astype(np.float32)
    g = device(a, "f32")
    with_grad = _params([g])[0]
    without = abi.make_tensor(g.ptr, (7,), None, abi.FLOAT32, abi.GPU, False, None)
    empty = _params([DeviceTensor((0, 4))])[0]
    arr = (abi.TensorP * 4)(C.pointer(without), C.pointer(with_grad), abi.TensorP(), C.pointer(empty))
    norm = DeviceTensor((1,))
    lib().clip_grad_norm_hip(C.cast(arr, C.c_void_p), 4, 1.0, C.byref(norm.t))
    lib().check()
    exact = np.sqrt((a.astype(np.float64) ** 2).sum())
    close(norm.numpy()[0], exact, exact * U * 1.01, "norm")
    close(values(g), a / exact, np.abs(a / exact) * 4 * U, "gradient")
    L = lib()
    for ptr, n in ((None, 0), (None, 5), (C.cast(arr, C.c_void_p), 0)):
        norm.fill_("uniform", 1, 5.0, 6.0)
        L.clip_grad_norm_hip(ptr, n, 1.0, C.byref(norm.t))
        L.check()
        assert norm.numpy()[0] == 0.0


def test_same_bits_every_time():
    rng = np.random.RandomState(4)
    arrays = [rng.randn(n).astype(np.float32) for n in (100000, 5, 777777)]
    runs = []
    for _ in range(3):
        grads = [device(a, "f32") for a in arrays]
        _clip(_params(grads), 1.0)
        runs.append([values(g) for g in grads])
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("count", [3, 130])
def test_replayed_with_other_work_between(count):
    """A captured clipping replayed over fresh gradients; more than a launch's arguments hold go in several launches there."""
    from plast_amd import runtime as rt
    L = rt.lib()
    rng = np.random.RandomState(5)
    arrays = [rng.randn(int(n)).astype(np.float32) for n in rng.randint(1, 9000, count)]
    grads = [device(a, "f32") for a in arrays]
    params, norm = _params(grads), rt.DeviceTensor((1,))
    _clip(params, 2.0, norm)
    assert L.plast_hip_capture_begin() == 0
    _clip(params, 2.0, norm)
    graph = L.plast_hip_capture_end()
    L.check("capture")
    for rep in range(3):
        fresh = [device(a * (0.01 if rep == 1 else rep + 1), "f32") for a in arrays]
        for g, n in zip(grads, fresh):
            L.arena_memcpy_d2d_hip(g.ptr, n.ptr, int(np.prod(n.shape)) * 4)
        a = rt.DeviceTensor((1000, 1000)).fill_("normal", rep, 0.0, 1.0)
        rt.forward("sum", [a], rt.DeviceTensor((1000,)), abi.KernelParams(0, 0, 0.0))
        assert L.plast_hip_graph_launch(graph) == 0
        got, got_norm = [values(g) for g in grads], norm.numpy()[0]
        exact = np.sqrt(sum((values(n).astype(np.float64) ** 2).sum() for n in fresh))
        close(got_norm, exact, exact * U * 1.01, "norm")
        for g, n in zip(got, fresh):
            want = values(n).astype(np.float64) * min(1.0, 2.0 / exact)
            close(g, want, np.abs(want) * 4 * U + 2.0 ** -149, "gradient")
    L.plast_hip_graph_destroy(graph)


def test_tables_of_many_gradients_in_turn():
    """Two lists of more gradients than a launch's arguments hold, in turn with an optimizer's own table."""
    from plast_amd import runtime as rt
    L = rt.lib()
    rng = np.random.RandomState(6)
    lists = [[rng.randn(50).astype(np.float32) for _ in range(n)] for n in (100, 200)]
    for rep in range(2):
        for arrays in lists:
            _check(arrays, ["f32"] * len(arrays), 0.5)
            grads = [device(a, "f32") for a in arrays]
            ps = [give(rt.DeviceTensor.from_numpy(a), g) for a, g in zip(arrays, grads)]
            arr, keep = abi.tensor_array(*[p.t for p in ps])
            L.sgd_step_hip(C.byref(abi.SGD(1.0)), arr, len(ps))
            L.check()
            assert not any(p.numpy().any() for p in ps)
