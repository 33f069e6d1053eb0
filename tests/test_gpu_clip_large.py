"""Clipping of sets that its launches go through in runs: more than 2048 pieces of 16 KiB, more than the last-level cache, more gradients
than the kernels' arguments hold, in captured graphs too. Against 64 bits, as in test_gpu_clip.py."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from block_cases import DTYPE, U, close, device, give, rounded, stored, values
from plast_amd import abi
from test_gpu_capture_cold import _replayed, cold  # noqa: F401
from test_gpu_clip import _clip, _params
from token_cases import load, store

pytestmark = pytest.mark.gpu


def _noise(n, seed):
    """n values without a period that pieces or workgroups have."""
    return np.resize(np.random.RandomState(seed).randn(100003).astype(np.float32), n)


def _set(sizes, kinds, seed=0):
    """Gradients one behind the other in a buffer for each type, with three elements between, so that their addresses are odd
    ones too. Returns their values, their tensors, the buffers and what these held."""
    from plast_amd.runtime import DeviceTensor
    flat, at = {}, dict.fromkeys(set(kinds), 1)
    places = []
    for n, kind in zip(sizes, kinds):
        places.append(at[kind])
        at[kind] += n + 3
    for i, kind in enumerate(sorted(at)):
        flat[kind] = store(_noise(at[kind], seed + i), kind)
    base = {kind: DeviceTensor.from_numpy(a) for kind, a in flat.items()}
    grads = [DeviceTensor((n,), DTYPE[kind], base=base[kind], offset=p) for n, kind, p in zip(sizes, kinds, places)]
    return [flat[kind][p:p + n] for n, kind, p in zip(sizes, kinds, places)], grads, base, flat, places


def _check(sizes, kinds, ratios, seed=0):
    from plast_amd.runtime import DeviceTensor
    arrays, grads, base, flat, places = _set(sizes, kinds, seed)
    exact = np.sqrt(sum(float((load(a).astype(np.float64) ** 2).sum()) for a in arrays))
    for ratio in ratios:
        print("clip", len(sizes), sum(sizes), ratio, flush=True)
        norm = DeviceTensor((1,))
        bound = float(np.float32(ratio * exact))
        _clip(_params(grads), bound, norm)
        close(norm.numpy()[0], exact, exact * U * 1.01, "norm")
        scale = min(1.0, bound / exact)
        got = {kind: t.numpy() for kind, t in base.items()}
        for kind in flat:  # what lies between the gradients too
            mark = np.zeros(flat[kind].size, bool)
            for n, k, p in zip(sizes, kinds, places):
                if k == kind:
                    mark[p:p + n] = True
            assert np.array_equal(got[kind][~mark], flat[kind][~mark])
            old, new = load(flat[kind])[mark], load(got[kind])[mark]
            if scale == 1.0:
                assert np.array_equal(new, old)
                continue
            for i in range(0, old.size, 1 << 24):
                want = old[i:i + (1 << 24)].astype(np.float64) * scale
                # rounded to fp32 on the way to 16 bits
                close(new[i:i + (1 << 24)], want, stored(want, kind) + np.abs(want) * 2 * U, f"{kind} from {i}")


@pytest.mark.parametrize("sizes, kinds", [
    ([2048 * 4096], ["f32"]), ([2048 * 4096 + 1], ["f32"]), ([2049 * 8192 + 4097], ["bf16"]),           # the last of a piece each, runs of three
    ([3000 * 4096 + 5, 7, 4096, 3], ["f32"] * 4), ([5000017, 8000009, 12345, 4097], ["f32", "f16", "bf16", "f32"]),
    ([1_300_000] * 14, ["f32"] * 14), ([20_000_001, 1, 9_999_999], ["f32", "bf16", "f16"]),             # several turns of the scaling workgroups
])
def test_sets_of_many_pieces(sizes, kinds):
    _check(sizes, kinds, (1.5, 0.3))


def test_runs_over_several_gradients():
    """Gradients of a piece or two, several in a workgroup's run, the types in turn."""
    rng = np.random.RandomState(1)
    sizes = [int(n) for n in rng.randint(1, 9000, 2600)]
    _check(sizes, [("f32", "bf16", "f16")[k % 3] for k in range(len(sizes))], (1.001, 0.5))


def test_sets_beyond_the_last_level_cache():
    _check([40_000_003, 5, 60_000_001, 1_000_000], ["f32", "f16", "f16", "f32"], (1.5, 0.3))


@pytest.mark.parametrize("count", [160, 161, 330])
def test_replayed_tables(count):
    """Tables that the arguments hold no more are laid down in the workspace by every replay: other users of it run in between."""
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
    others = [device(rng.randn(3000).astype(np.float32), "f32") for _ in range(200)]
    for rep in range(3):
        fresh = [device(a * (0.01 if rep == 1 else rep + 1), "f32") for a in arrays]
        for g, n in zip(grads, fresh):
            L.arena_memcpy_d2d_hip(g.ptr, n.ptr, int(np.prod(n.shape)) * 4)
        a = rt.DeviceTensor((1000, 1000)).fill_("normal", rep, 0.0, 1.0)
        rt.forward("sum", [a], rt.DeviceTensor((1000,)), abi.KernelParams(0, 0, 0.0))
        _clip(_params(others), 1e9)
        assert L.plast_hip_graph_launch(graph) == 0
        got, got_norm = [values(g) for g in grads], norm.numpy()[0]
        exact = np.sqrt(sum((values(n).astype(np.float64) ** 2).sum() for n in fresh))
        close(got_norm, exact, exact * U * 1.01, "norm")
        for g, n in zip(got, fresh):
            want = values(n).astype(np.float64) * min(1.0, 2.0 / exact)
            close(g, want, np.abs(want) * 4 * U + 2.0 ** -149, "gradient")
    L.plast_hip_graph_destroy(graph)


def test_long_tables_in_turn_with_an_optimizers():
    from plast_amd import runtime as rt
    L = rt.lib()
    rng = np.random.RandomState(6)
    lists = [[rng.randn(50).astype(np.float32) for _ in range(n)] for n in (200, 400)]
    sgd = abi.SGD(1.0)
    for rep in range(2):
        for arrays in lists:
            grads = [device(a, "f32") for a in arrays]
            ps = [give(rt.DeviceTensor.from_numpy(a), g) for a, g in zip(arrays, grads)]
            exact = np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays))
            _clip([p.t for p in ps], 0.5 * exact)
            arr, keep = abi.tensor_array(*[p.t for p in ps])
            L.sgd_step_hip(C.byref(sgd), arr, len(ps))
            L.check()
            for p, a in zip(ps, arrays):  # a - a / 2, off by a / 2's roundings
                close(p.numpy(), a / 2, np.abs(a) * 3 * U, "stepped")


def test_a_long_table_in_a_cold_capture(cold):  # noqa: F811
    from plast_amd import runtime as rt
    rng = np.random.RandomState(2)
    arrays = [rng.randn(int(n)).astype(np.float32) for n in rng.randint(1, 9000, 170)]
    flat = np.concatenate(arrays)
    g, fresh, norm = rt.DeviceTensor.from_numpy(flat), rt.DeviceTensor.from_numpy(flat), rt.DeviceTensor((1,))
    views, at = [], 0
    for a in arrays:
        views.append(rt.DeviceTensor(a.shape, base=g, offset=at))
        at += a.size
    params = _params(views)
    arr, keep = abi.tensor_array(*params)

    def call():
        cold.arena_memcpy_d2d_hip(g.ptr, fresh.ptr, flat.nbytes)
        cold.clip_grad_norm_hip(arr, len(params), 3.0, norm.p)
    got = _replayed(cold, call, [g, norm])
    exact = np.sqrt((flat.astype(np.float64) ** 2).sum())
    close(got[1][0], exact, exact * U * 1.01, "norm")
    want = flat * (3.0 / exact)
    close(got[0], want, np.abs(want) * 4 * U, "clipped")
