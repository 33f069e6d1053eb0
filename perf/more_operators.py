"""The operators that a recurrent language model's blocks need beside the row and optimizer kernels, each
as one pass at one size: layer norm (`norm`), the same with its gradients (`norm_train`), the gated linear
recurrence over a batch of sequences or over one token of each (`scan`), the same with its gradients
(`scan_train`), and the clipping of all gradients by their global norm (`clip`).

With `own` false, `run` computes them from elementary torch operations in 32 bits, rounded once at the
end; with `own` true it makes the calls a program makes of `plast_amd`, asynchronously
(plast_hip_set_sync(0)) and into its own buffers. `exact` computes the same in 64 bits.

Layer norm over rows x of `width` elements, with weight w and bias b:
    mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  n = (x - mu) r,  y = n w + b,
    dx = r (g - mean g - n mean(g n)) with g = dy w,  dw = sum over rows of dy n,  db = of dy.
Gated linear recurrence, each channel by itself, a = sigmoid(f):
    h[t] = a[t] h[t-1] + (1 - a[t]) v[t],  h[-1] the initial state, `last` the state after the sequence's end;
    dh[t] = dy[t] + a[t+1] dh[t+1], with the gradient of `last` added at the sequence's last position,
    dv = (1 - a) dh,  df = dh (h[t-1] - v) a (1 - a),  dinitial = a[0] dh[0].
Positions from a sequence's length on are padding: h and all gradients are 0 there.
Clipping: norm = sqrt of the sum of all squares; where it is above the bound, every gradient times
bound / norm.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
FALL = 1.0 - 2.0 ** -12  # of the bound from one clipping to the next


# ----------------------------------------------------------------------------- the cases

def listed():
    return [
        # The norm in front of a block while a batch of sequences decodes: a row each. Latency.
        {"name": "norm_64x4096_bf16", "kind": "norm", "batch": 64, "len": 1, "width": 4096, "pitch": 4096,
         "type": "bf16"},
        # Prompt processing in fp32, at the rows of the bias-gradient benchmark.
        {"name": "norm_16384x4096_f32", "kind": "norm", "batch": 4, "len": 4096, "width": 4096, "pitch": 4096,
         "type": "f32"},
        # Training a wide model in 16 bits: forward and all three gradients.
        {"name": "train_norm_16384x4096_bf16", "kind": "norm_train", "batch": 8, "len": 2048, "width": 4096,
         "pitch": 4096, "type": "bf16"},
        # Many short rows of an odd width.
        {"name": "train_norm_30011x333_f32", "kind": "norm_train", "batch": 30011, "len": 1, "width": 333,
         "pitch": 333, "type": "f32"},
        # Rows that are slices of a wider buffer, few of them and long.
        {"name": "train_norm_512x20000_f16", "kind": "norm_train", "batch": 2, "len": 256, "width": 20000,
         "pitch": 20480, "type": "f16"},
        # One token of each sequence of a decode batch. Latency.
        {"name": "scan_64x1x4096_bf16", "kind": "scan", "batch": 64, "len": 1, "width": 4096, "type": "bf16",
         "ragged": False, "packed": True, "resets": 0.0},
        # A long prompt: one sequence, gates and values halves of one projection.
        {"name": "scan_1x65536x1024_bf16", "kind": "scan", "batch": 1, "len": 65536, "width": 1024, "type": "bf16",
         "ragged": False, "packed": True, "resets": 0.0},
        # Training on documents packed one behind the other, their starts marked by closed gates.
        {"name": "train_scan_8x4096x2048_bf16", "kind": "scan_train", "batch": 8, "len": 4096, "width": 2048,
         "type": "bf16", "ragged": False, "packed": True, "resets": 0.002},
        # Sequences of several lengths in one batch, odd extents.
        {"name": "train_scan_5x3001x1003_f32", "kind": "scan_train", "batch": 5, "len": 3001, "width": 1003,
         "type": "f32", "ragged": True, "packed": False, "resets": 0.0},
        # The four tensors of a small MLP. Latency.
        {"name": "clip_mlp_f32", "kind": "clip", "count": 2, "rows": 256, "cols": 256, "extra": 2, "type": "f32",
         "ratio": 0.5},
        # The weights and biases of the deep MLP that the Adam benchmark has, above the bound.
        {"name": "clip_24x1024x1024_f32", "kind": "clip", "count": 24, "rows": 1024, "cols": 1024, "extra": 24,
         "type": "f32", "ratio": 0.5},
        # A large layer's projections within the bound: the norm alone.
        {"name": "clip_4x4096x16384_within", "kind": "clip", "count": 4, "rows": 4096, "cols": 16384, "extra": 4,
         "type": "f32", "ratio": 2.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _extent(rng, lo, hi):
    """An extent over [lo, hi], half of them as they fall and half rounded to a usual multiple."""
    n = _log_int(rng, lo, hi)
    m = rng.choice([1, 1, 1, 8, 32, 128])
    return max(lo, min(hi, n // m * m if n >= m else n))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "scan", "scan_train", "clip"])
    if kind == "clip":
        rows, cols = _extent(rng, 1, 8192), _extent(rng, 1, 16384)
        count = _log_int(rng, 1, max(1, min(200, (1 << 28) // (rows * cols))))
        return {"kind": kind, "count": count, "rows": rows, "cols": cols, "extra": rng.choice([0, 1, count]),
                "type": rng.choice(["f32", "f32", "bf16", "f16"]), "ratio": rng.choice([0.01, 0.5, 0.999, 2.0])}
    width = _extent(rng, 4, 65536 if kind.startswith("norm") else 16384)
    rows = _extent(rng, 1, min(131072, (1 << 26) // width))
    if kind.startswith("norm"):
        length = rng.choice([1, rows, max(1, rows // 4)])
        return {"kind": kind, "batch": max(1, rows // length), "len": length, "width": width,
                "pitch": rng.choice([width, width, (width + 63) // 64 * 64, 3 * width]),
                "type": rng.choice(["f32", "bf16", "f16"])}
    batch = _log_int(rng, 1, min(rows, 512))
    return {"kind": kind, "batch": batch, "len": max(1, rows // batch), "width": width,
            "type": rng.choice(["f32", "bf16", "f16"]), "ragged": rng.random() < 0.4,
            "packed": rng.random() < 0.5, "resets": rng.choice([0.0, 0.0, 0.002, 0.1])}


# ----------------------------------------------------------------------------- inputs

def _extents(case):
    """Shapes of a clip case's gradients: matrices, then vectors of their columns."""
    return [(case["rows"], case["cols"])] * case["count"] + [(case["cols"],)] * case["extra"]


def _numel(case):
    return case["rows"] * case["cols"] * case["count"] + case["cols"] * case["extra"]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": dict(case)}

    def noise(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    kind = TYPES[case["type"]]
    if case["kind"] == "clip":
        # one allocation, as a trainer's flat gradient buffer has it, the tensors views of it
        s["flat"] = (noise(_numel(case)) * 1e-3).to(kind)
        s["grads"], at = [], 0
        for shape in _extents(case):
            n = math.prod(shape)
            s["grads"].append(s["flat"][at:at + n].view(shape))
            at += n
        s["bound"] = case["ratio"] * 1e-3 * math.sqrt(_numel(case))
        s["norm"] = torch.empty(1, device=DEV, dtype=torch.float32)
        return s
    b, length, width = case["batch"], case["len"], case["width"]
    if case["kind"].startswith("norm"):
        full = torch.empty((b, length, case["pitch"]), device=DEV, dtype=kind)
        x = full[:, :, :width]
        # a residual stream: channels of their own offsets, a few of them large
        offset = 0.3 * noise(width) + 8.0 * (torch.rand(width, generator=gen, device=DEV) < 0.002).float()
        x.copy_(noise(b, length, width) + offset)
        s["full"], s["x"] = full, x
        s["w"], s["b"] = 1.0 + 0.1 * noise(width), 0.1 * noise(width)
        s["y"] = torch.empty((b, length, width), device=DEV, dtype=kind)
        s["stats"] = torch.empty((b * length, 2), device=DEV, dtype=torch.float32)
        if case["kind"] == "norm_train":
            s["dy"] = (noise(b, length, width) * 0.1).to(kind)
            s["dx"] = torch.empty_like(s["dy"])
            s["dw"], s["db"] = torch.empty_like(s["w"]), torch.empty_like(s["b"])
        return s
    # channels that remember from two steps to some hundreds
    keep = 5.5 * torch.rand(width, generator=gen, device=DEV)
    if case["packed"]:
        both = torch.empty((b, length, 2 * width), device=DEV, dtype=kind)
        s["both"], s["f"], s["v"] = both, both[:, :, :width], both[:, :, width:]
    else:
        s["f"] = torch.empty((b, length, width), device=DEV, dtype=kind)
        s["v"] = torch.empty((b, length, width), device=DEV, dtype=kind)
    s["f"].copy_(noise(b, length, width) + keep)
    s["v"].copy_(noise(b, length, width) + 0.5)
    if case["resets"] > 0:
        start = torch.rand((b, length, 1), generator=gen, device=DEV) < case["resets"]
        s["f"].masked_fill_(start, -math.inf)
    s["initial"] = noise(b, width)
    lengths = torch.full((b,), length, device=DEV, dtype=torch.int32)
    if case["ragged"]:
        lengths = (lengths * (0.25 + 0.75 * torch.rand(b, generator=gen, device=DEV))).round().to(torch.int32)
    s["lengths"] = lengths
    s["h"] = torch.empty((b, length, width), device=DEV, dtype=kind)
    s["last"] = torch.empty((b, width), device=DEV, dtype=torch.float32)
    if case["kind"] == "scan_train":
        s["dy"] = (noise(b, length, width) * 0.1).to(kind)
        s["dlast"] = noise(b, width) * 0.1
        s["df"], s["dv"] = torch.empty_like(s["h"]), torch.empty_like(s["h"])
        s["dinitial"] = torch.empty_like(s["last"])
    return s


# ----------------------------------------------------------------------------- the plain forms

def _plain_norm(s):
    x = s["x"].float()
    d = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    n = d * r
    got = {"y": (n * s["w"] + s["b"]).to(s["y"].dtype)}
    if s["case"]["kind"] == "norm_train":
        dy = s["dy"].float()
        g = dy * s["w"]
        got["dx"] = (r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))).to(s["dx"].dtype)
        got["dw"], got["db"] = (dy * n).sum((0, 1)), dy.sum((0, 1))
    return got


def _plain_runs(a, b):
    """b[t] + a[t] b[t-1] + a[t] a[t-1] b[t-2] + ...: runs of twice the length in every step."""
    step = 1
    while step < b.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_scan(s):
    f, v = s["f"].float(), s["v"].float()
    length = f.shape[1]
    ends = s["lengths"].long()[:, None, None]
    live = torch.arange(length, device=DEV)[None, :, None] < ends
    # beyond the end a state stays as it is
    a = torch.where(live, 1.0 / (1.0 + torch.exp(-f)), 1.0)
    z = torch.where(live, 1.0 / (1.0 + torch.exp(f)), 0.0)
    u = z * v
    u[:, 0] += a[:, 0] * s["initial"]
    h = _plain_runs(a, u)
    got = {"h": torch.where(live, h, 0.0).to(s["h"].dtype), "last": h[:, -1]}
    if s["case"]["kind"] == "scan_train":
        dy = torch.where(live, s["dy"].float(), 0.0)
        dy[:, -1] += s["dlast"]
        following = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
        dh = _plain_runs(following.flip(1), dy.flip(1)).flip(1)
        before = torch.cat([s["initial"][:, None], h[:, :-1]], 1)
        got["df"] = (dh * (before - v) * a * z).to(s["df"].dtype)
        got["dv"] = (z * dh).to(s["dv"].dtype)
        got["dinitial"] = a[:, 0] * dh[:, 0]
    return got


def _bound(s):
    """This pass's bound on the norm. It falls a little every time, so that gradients clipped by the pass
    before are above it again."""
    bound = s["bound"]
    if s["case"]["ratio"] < 1.0:
        s["bound"] = bound * FALL
    return bound


def _plain_clip(s):
    bound = _bound(s)
    g = s["flat"].float()
    norm = torch.sqrt((g * g).sum())
    s["flat"].copy_(g * torch.where(norm > bound, bound / norm, 1.0))
    return {"norm": norm.reshape(1), "grads": s["flat"]}


# ----------------------------------------------------------------------------- the library's calls

def _struct(t, requires_grad=False, grad=None):
    from plast_amd import abi
    kind = {torch.float32: abi.FLOAT32, torch.bfloat16: abi.BFLOAT16, torch.float16: abi.FLOAT16,
            torch.int32: abi.INT32}[t.dtype]
    return abi.make_tensor(t.data_ptr(), t.shape, t.stride(), kind, abi.GPU, requires_grad, grad)


def _calls(s):
    """What a program sets up once around its buffers: the tensors' structs and, for a backward pass of the
    recurrence, the buffer of the states that its forward pass leaves."""
    from plast_amd import abi
    from plast_amd.runtime import lib
    lib().plast_hip_set_sync(0)
    c, q = s["case"], {}

    def given(name, grad=None):
        q[grad] = _struct(s[grad]) if grad in s else None
        return _struct(s[name], q[grad] is not None, q[grad])

    if c["kind"] == "clip":
        q["grads"] = [_struct(g) for g in s["grads"]]
        q["params"] = [_struct(g, True, t) for g, t in zip(s["grads"], q["grads"])]  # only their gradients are used
        q["list"], q["keep"] = abi.tensor_array(*q["params"])
        q["norm"] = _struct(s["norm"])
    elif c["kind"].startswith("norm"):
        q["ins"] = [given("x", "dx"), given("w", "dw"), given("b", "db"), _struct(s["stats"])]
        q["out"] = given("y", "dy")
        q["params"] = abi.KernelParams(0, 1, EPS)
    else:
        train = c["kind"] == "scan_train"
        q["ins"] = [given("f", "df"), given("v", "dv"), given("initial", "dinitial"), _struct(s["lengths"]),
                    given("last", "dlast")]
        if train:
            chunks = -(-c["len"] // abi.RECURRENCE_CHUNK)
            s["states"] = torch.empty((c["batch"], chunks, c["width"]), device=DEV, dtype=torch.float32)
            q["ins"].append(_struct(s["states"]))
        q["out"] = given("h", "dy")
        q["params"] = abi.KernelParams(int(train), 1, 0.0)
    return q


def _own(s):
    import ctypes as ct

    from plast_amd.runtime import backward, forward, lib
    if "calls" not in s:
        s["calls"] = _calls(s)
    q, c = s["calls"], s["case"]
    if c["kind"] == "clip":
        lib().clip_grad_norm_hip(q["list"], len(s["grads"]), _bound(s), ct.byref(q["norm"]))
        lib().check("clip_grad_norm")
        return {"norm": s["norm"], "grads": s["flat"]}
    norm = c["kind"].startswith("norm")
    op = "layer_norm" if norm else "gated_recurrence"
    forward(op, q["ins"], q["out"], q["params"])
    got = {"y": s["y"]} if norm else {"h": s["h"], "last": s["last"]}
    if c["kind"].endswith("train"):
        backward(op, q["ins"], q["out"], q["params"])
        got.update({k: s[k] for k in (("dx", "dw", "db") if norm else ("df", "dv", "dinitial"))})
    return got


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "clip":
        return _plain_clip(state)
    return _plain_norm(state) if kind.startswith("norm") else _plain_scan(state)


# ----------------------------------------------------------------------------- what a pass needs

def work(case):
    item = TYPES[case["type"]].itemsize
    if case["kind"] == "clip":
        n = _numel(case)
        return {"bytes": n * item * (2 if case["ratio"] < 1.0 else 1), "flops": n * (3 if case["ratio"] < 1.0 else 2)}
    train = case["kind"].endswith("train")
    b, width = case["batch"], case["width"]
    n = b * case["len"] * width
    if case["kind"].startswith("norm"):
        # x (and dy) read, y (and dx) written
        return {"bytes": n * item * (4 if train else 2) + width * (16 if train else 8), "flops": n * (20 if train else 8)}
    # gates and values (and dy) read, states (and two gradients) written
    return {"bytes": n * item * (6 if train else 3) + b * width * (16 if train else 8), "flops": n * (20 if train else 8)}


# ----------------------------------------------------------------------------- in 64 bits

def _exact_norm(s):
    rows, width = s["case"]["batch"] * s["case"]["len"], s["case"]["width"]
    train = s["case"]["kind"] == "norm_train"
    f64 = {"device": DEV, "dtype": torch.float64}
    x, out = s["x"].reshape(rows, width), {"y": torch.empty((rows, width), **f64)}
    w, b = s["w"].double(), s["b"].double()
    if train:
        dy = s["dy"].reshape(rows, width)
        out["dx"] = torch.empty((rows, width), **f64)
        out["dw"], out["db"] = torch.zeros(width, **f64), torch.zeros(width, **f64)
    step = max(1, (1 << 25) // width)
    for r in range(0, rows, step):
        z = x[r:r + step].double()
        var, mu = torch.var_mean(z, dim=1, correction=0, keepdim=True)
        z = (z - mu) * torch.rsqrt(var + EPS)
        out["y"][r:r + step] = b + w * z
        if train:
            u = dy[r:r + step].double()
            out["db"] += u.sum(0)
            out["dw"] += (u * z).sum(0)
            # the projection of the upstream gradient off the row's ones and its normalised values
            u = u * w
            along = (u * z).sum(1, keepdim=True) / width
            out["dx"][r:r + step] = (u - u.sum(1, keepdim=True) / width - along * z) * torch.rsqrt(var + EPS)
    return {k: t.reshape(s["x"].shape) if t.dim() == 2 else t for k, t in out.items()}


def _exact_scan(s):
    b, length, width = s["h"].shape
    f64 = {"device": DEV, "dtype": torch.float64}
    train = s["case"]["kind"] == "scan_train"
    ends = s["lengths"].long().tolist()
    order = sorted(range(b), key=lambda i: -ends[i])
    h, last = torch.zeros((b, length + 1, width), **f64), torch.empty((b, width), **f64)
    h[:, 0] = s["initial"].double()
    a = torch.sigmoid(s["f"].double())
    into = torch.sigmoid(-s["f"].double()) * s["v"].double()
    for t in range(length):
        torch.addcmul(into[:, t], a[:, t], h[:, t], out=h[:, t + 1])
    for i in range(b):
        last[i] = h[i, ends[i]]
        h[i, ends[i] + 1:] = 0.0
    out = {"h": h[:, 1:], "last": last}
    if train:
        dh = torch.zeros((b, length, width), **f64)
        carry = torch.zeros((b, width), **f64)
        alive = 0
        dy, dlast = s["dy"].double(), s["dlast"].double()
        for t in range(length - 1, -1, -1):
            while alive < b and ends[order[alive]] > t:
                carry[order[alive]] = dlast[order[alive]]
                alive += 1
            if alive == b:
                carry += dy[:, t]
                dh[:, t] = carry
                carry *= a[:, t]
            else:
                at = order[:alive]
                dh[at, t] = carry[at] + dy[at, t]
                carry[at] = a[at, t] * dh[at, t]
        for i in range(alive, b):
            carry[order[i]] = dlast[order[i]]
        rest = torch.sigmoid(-s["f"].double())
        out["dv"] = rest * dh
        out["df"] = out["dv"] * a * (h[:, :-1] - s["v"].double())
        out["dinitial"] = carry
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("norm"):
        return _exact_norm(s)
    if case["kind"].startswith("scan"):
        if case["ragged"] and case["kind"] == "scan_train" and case["len"] > 16384:
            return None
        return _exact_scan(s)
    norm = torch.linalg.vector_norm(s["flat"].double())
    scale = min(1.0, s["bound"] / float(norm))
    return {"norm": norm.reshape(1), "grads": s["flat"].double() * scale}
