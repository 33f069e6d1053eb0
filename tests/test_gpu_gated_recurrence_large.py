"""The gated recurrence over operands beyond the last-level cache, which are read past it: forward beyond 192 MiB of gates and values,
backward of these and the upstream gradient. Some channels, the first, last and those beside a tile's end among them, against 64
bits; all of them against calls of half of the channels each, which are read through the cache and have the same bits."""
from __future__ import annotations

import numpy as np
import pytest

from block_cases import DTYPE, close, scan_exact, stored
from plast_amd import abi
from plast_amd.abi import KernelParams
from token_cases import load, store

pytestmark = pytest.mark.gpu
PAST = 192 << 20


def _stored(n, kind, seed, plus=0.0, times=1.0):
    """n values without a period that steps or channels have, as a tensor of `kind` is made from."""
    return np.resize(store(np.random.RandomState(seed).randn(1000003).astype(np.float32) * times + plus, kind), n)


# Tiles of every shape that such operands meet: 64 to 256 steps, one and several, forward and backward, the same for half of the channels.
@pytest.mark.parametrize("shape, kind", [((4, 2050, 3137), "f32"), ((1, 7000, 3840), "f32"), ((1, 22000, 1160), "f32"), ((1, 50000, 508), "f32"),
                                         ((60, 200, 2200), "f32"), ((64, 50, 8200), "f32"), ((4, 4099, 3201), "bf16"), ((16, 128, 25000), "bf16"),
                                         ((1, 26000, 2002), "f16")])
def test_past_the_caches(shape, kind):
    B, T, D = shape
    n, item = B * T * D, 4 if kind == "f32" else 2
    assert 2 * n * item > PAST and 3 * n // 2 * item < PAST * 0.9
    add = D % 2 == 1
    print(f"recurrence past the caches {kind} {shape} add={add}", flush=True)
    host = {name: _stored(n, kind, k, *how).reshape(shape) for k, (name, how) in enumerate(
        (("f", (2.0, 1.5)), ("v", (0.5,)), ("dy", ()), ("df", (0.0, 0.1)), ("dv", (0.0, 0.1))))}
    rng = np.random.RandomState(B + T + D)
    host.update({name: rng.randn(B, D).astype(np.float32) for name in ("initial", "dlast", "dinitial")})
    lengths = np.full(B, T, np.int32)
    if B > 1:
        lengths[B // 2:] = T - T // 3
    got = _call(host, lengths, kind, add)

    channels = np.unique(np.concatenate([[0, 1, 62, 63, 64, 65, D // 2, D - 66, D - 3, D - 2, D - 1], rng.randint(0, D, 10)]))
    some = {name: np.ascontiguousarray(a[..., channels]) for name, a in host.items()}
    f, v, dy, df, dv = (load(some[k]) for k in ("f", "v", "dy", "df", "dv"))
    want = scan_exact(f, v, some["initial"], lengths, dy, some["dlast"])
    for name, old in (("h", None), ("last", None), ("df", df), ("dv", dv), ("dinitial", some["dinitial"])):
        ref, size, k = want[name], np.abs(want[name]), "f32" if name in ("last", "dinitial") else kind
        if add and old is not None:
            ref, size = ref + old, np.abs(ref + old) + np.abs(old)
        close(load(got[name][..., channels]), ref, want[name + "_tol"] + stored(size, k), f"{name} of channels {channels}")

    for part in (slice(0, D // 2), slice(D // 2, D)):
        half = _call({name: np.ascontiguousarray(a[..., part]) for name, a in host.items()}, lengths, kind, add)
        for name, a in half.items():
            assert np.array_equal(a, got[name][..., part]), (name, part)


def _call(host, lengths, kind, add):
    """The results of both passes, as they are stored."""
    from plast_amd.runtime import DeviceTensor, backward, forward
    shape = B, T, D = host["f"].shape
    dev = {name: DeviceTensor.from_numpy(a) for name, a in host.items()}
    assert dev["f"].dtype == DTYPE[kind]
    last, states = DeviceTensor((B, D)), DeviceTensor((B, -(-T // abi.RECURRENCE_CHUNK), D))
    h, steps = DeviceTensor(shape, DTYPE[kind]), DeviceTensor.from_numpy(lengths)

    def struct(t, grad):
        return abi.make_tensor(t.ptr, t.shape, None, t.dtype, abi.GPU, True, dev[grad].t)
    ins = [struct(dev["f"], "df"), struct(dev["v"], "dv"), struct(dev["initial"], "dinitial"), steps.t, struct(last, "dlast"), states.t]
    out = struct(h, "dy")
    forward("gated_recurrence", ins, out, KernelParams(1, 0, 0.0))
    backward("gated_recurrence", ins, out, KernelParams(1, 0 if add else 1, 0.0))
    return {"h": h.numpy(), "last": last.numpy(), **{k: dev[k].numpy() for k in ("df", "dv", "dinitial")}}
