"""The operators of a language-model training step that this library adds to its reductions and
optimizers, each as one pass at one size: log-probabilities of given tokens with entropy and top
alternatives (`score`), the same with its gradient (`train`), both in one pass over the logits
(`step`), the Newton-Schulz orthogonalisation of a matrix (`orth`) and the optimizer step that is
built on it (`muon`).

With `own` false, `run` computes them from elementary torch operations in 32 bits, rounded once at
the end; with `own` true it makes the calls a program makes of `plast_amd`, asynchronously
(plast_hip_set_sync(0)) and into its own buffers. `exact` computes the same in 64 bits.

A row's distribution is softmax(x / temperature) over its `vocab` logits:
    logp = log p[token],  entropy = -sum p log p,  alternatives: the `top` largest logits in
    descending order, ties to the lowest index, with their log p.
A row whose token is negative is padding: it is not looked at, and gets logp 0, entropy 0, a zero
gradient and alternatives (-1, -inf). A row whose logits are all -inf has no distribution: logp -inf,
entropy 0, a zero gradient.
The gradient, for upstream gradients u of logp and h of the entropy H:
    dx[j] = (u * ((j == token) - p[j]) - h * p[j] * (log p[j] + H)) / temperature.
Newton-Schulz: X = G / (|G| + eps), Frobenius norm, on the side with fewer rows; `steps` times
    A = X X^T,  X = a X + (b A + c A A) X.
Muon: m = beta m + (1 - beta) g,  u = (1 - beta) g + beta m,  O = Newton-Schulz(u),
    p = p (1 - lr decay) - lr sqrt(max(1, rows / cols)) O.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
A, B, C, EPS = 3.4445, -4.7750, 2.0315, 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.01


# ----------------------------------------------------------------------------- the cases

def listed():
    return [
        # One sequence decoding: the sampled token's log-probability and twenty alternatives for the
        # reply, at the sampling temperature. Latency.
        {"name": "score_1x131072_bf16_top20", "kind": "score", "batch": 1, "len": 1, "pad": 0,
         "vocab": 131072, "pitch": 131072, "type": "bf16", "top": 20, "masked": 0.0, "temp": 0.7},
        # A decode batch under a grammar: most of an odd vocabulary is masked with -inf.
        {"name": "score_64x50001_f16_top5", "kind": "score", "batch": 64, "len": 1, "pad": 0,
         "vocab": 50001, "pitch": 50001, "type": "f16", "top": 5, "masked": 0.9, "temp": 1.0},
        # Prompt scoring: positions predict the next token, so the last one is left out of the view,
        # and the ends of the sequences are padding.
        {"name": "score_8x1023x32000_f32", "kind": "score", "batch": 8, "len": 1023, "pad": 100,
         "vocab": 32000, "pitch": 32000, "type": "f32", "top": 0, "masked": 0.0, "temp": 1.0},
        # Log-probabilities with alternatives over a corpus, a large vocabulary.
        {"name": "score_4x1024x131072_bf16_top8", "kind": "score", "batch": 4, "len": 1024, "pad": 0,
         "vocab": 131072, "pitch": 131072, "type": "bf16", "top": 8, "masked": 0.0, "temp": 1.0},
        # A policy-gradient step whose loss needs the log-probabilities first: forward, backward.
        {"name": "train_4x512x32000_f32", "kind": "train", "batch": 4, "len": 512, "pad": 64,
         "vocab": 32000, "pitch": 32000, "type": "f32", "top": 0, "masked": 0.0, "temp": 1.0},
        # The same over a batch of 16-bit logits whose rows are padded to a whole multiple of 64.
        {"name": "train_8x1024x49999_bf16", "kind": "train", "batch": 8, "len": 1024, "pad": 128,
         "vocab": 49999, "pitch": 50048, "type": "bf16", "top": 0, "masked": 0.0, "temp": 0.8},
        # Upstream gradients known beforehand (on-policy advantages): one call, at the sizes of the
        # cross-entropy step's benchmark.
        {"name": "step_32768x32000_f32", "kind": "step", "batch": 1, "len": 32768, "pad": 0,
         "vocab": 32000, "pitch": 32000, "type": "f32", "top": 0, "masked": 0.0, "temp": 1.0},
        # A policy over a handful of actions, some of them illegal in each state.
        {"name": "step_60000x18_f32", "kind": "step", "batch": 60000, "len": 1, "pad": 0,
         "vocab": 18, "pitch": 18, "type": "f32", "top": 0, "masked": 0.3, "temp": 1.0},
        # One small weight: the iterations are a chain of short products. Latency.
        {"name": "orth_256x256_f32", "kind": "orth", "count": 1, "rows": 256, "cols": 256,
         "type": "f32", "steps": 5},
        # Tall weights of odd extents, stacked over layers, in 16 bits.
        {"name": "orth_6x2605x1001_bf16", "kind": "orth", "count": 6, "rows": 2605, "cols": 1001,
         "type": "bf16", "steps": 5},
        # An optimizer step over the weights of the deep MLP that the Adam benchmark has.
        {"name": "muon_24x1024x1024", "kind": "muon", "count": 24, "rows": 1024, "cols": 1024,
         "steps": 5},
        # One large weight: the arithmetic of a wide layer's projection.
        {"name": "muon_1x4096x16384", "kind": "muon", "count": 1, "rows": 4096, "cols": 16384,
         "steps": 5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _extent(rng, lo, hi):
    """An extent over [lo, hi], half of them as they fall and half rounded to a usual multiple."""
    n = _log_int(rng, lo, hi)
    m = rng.choice([1, 1, 1, 8, 32, 128])
    return max(lo, min(hi, n // m * m if n >= m else n))


def draw(rng):
    kind = rng.choice(["score", "train", "step", "orth", "muon"])
    if kind in ("score", "train", "step"):
        vocab = _extent(rng, 10, 131072)
        rows = _extent(rng, 1, min(65536, (1 << 28) // vocab))
        length = rng.choice([1, rows, max(1, rows // 4)])
        masked = rng.choice([0.0, 0.0, 0.3, 0.9])
        return {"kind": kind, "batch": max(1, rows // length), "len": length,
                "pad": rng.choice([0, length // 8]), "vocab": vocab,
                "pitch": rng.choice([vocab, (vocab + 63) // 64 * 64]),
                "type": rng.choice(["f32", "bf16", "f16"]),
                "top": rng.choice([0, 1, 5, 20, 32]) if kind == "score" else 0,
                "masked": masked, "temp": rng.choice([1.0, 1.0, 0.6, 1.5])}
    rows = _extent(rng, 32, 4096)
    cols = _extent(rng, 32, 8192)
    if rng.random() < 0.4:
        rows, cols = cols, rows
    small, large = min(rows, cols), max(rows, cols)
    count = _log_int(rng, 1, max(1, min(24, (1 << 35) // (small * small * large))))
    case = {"kind": kind, "count": count, "rows": rows, "cols": cols, "steps": 5}
    if kind == "orth":
        case["type"] = rng.choice(["f32", "f32", "bf16", "f16"])
    return case


# ----------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": dict(case)}
    if case["kind"] in ("orth", "muon"):
        shape = (case["count"], case["rows"], case["cols"])
        # a gradient: a few strong directions over noise
        g = torch.randn(shape, generator=gen, device=DEV)
        left = torch.randn((shape[0], shape[1], 8), generator=gen, device=DEV)
        right = torch.randn((shape[0], 8, shape[2]), generator=gen, device=DEV)
        g += left @ right
        g *= 1e-3
        if case["kind"] == "orth":
            s["g"] = g.to(TYPES[case["type"]])
            s["out"] = torch.empty_like(s["g"])
        else:
            # parameters of their own, as a model's layers have them
            s["g"] = list(g.unbind(0))
            s["p"] = [0.02 * torch.randn(shape[1:], generator=gen, device=DEV) for _ in s["g"]]
            s["m"] = [1e-3 * torch.randn(shape[1:], generator=gen, device=DEV) for _ in s["g"]]
        return s
    n, length, vocab = case["batch"] * case["len"], case["len"], case["vocab"]
    kind = TYPES[case["type"]]
    # sequences hold one position more than the view where there are several positions
    full = torch.empty((case["batch"], length + (1 if length > 1 else 0), case["pitch"]),
                       device=DEV, dtype=kind)
    x = full[:, :length, :vocab]
    for b in range(0, case["batch"], max(1, case["batch"] // 16)):
        part = x[b:b + max(1, case["batch"] // 16)]
        part.copy_(2.0 * torch.randn(part.shape, generator=gen, device=DEV))
    tokens = torch.randint(0, vocab, (case["batch"], length), generator=gen, device=DEV)
    # half of the given tokens are likely ones
    at = tokens.unsqueeze(-1)
    likely = (torch.rand(at.shape, generator=gen, device=DEV) < 0.5).float()
    x.scatter_(2, at, (x.gather(2, at).float() + 8.0 * likely).to(kind))
    if case["masked"] > 0:
        for b in range(0, case["batch"], max(1, case["batch"] // 16)):
            part = x[b:b + max(1, case["batch"] // 16)]
            part.masked_fill_(torch.rand(part.shape, generator=gen, device=DEV) < case["masked"],
                              -math.inf)
        if n >= 8:
            x[case["batch"] // 2, length // 2] = -math.inf
    if case["pad"]:
        tokens[:, length - case["pad"]:] = -1
    s["full"], s["x"], s["tokens"] = full, x, tokens.reshape(-1).to(torch.int32)
    f32 = {"device": DEV, "dtype": torch.float32}
    s["logp"], s["entropy"] = torch.empty(n, **f32), torch.empty(n, **f32)
    if case["kind"] == "score":
        s["stats"] = torch.empty((n, 2), **f32)
        s["top_logp"] = torch.empty((n, case["top"]), **f32)
        s["top_ids"] = torch.empty((n, case["top"]), device=DEV, dtype=torch.int32)
        return s
    s["stats"] = torch.empty((n, 2), **f32)
    s["dlogp"] = torch.randn(n, generator=gen, device=DEV) / n
    s["dentropy"] = (-0.01 / n) * torch.rand(n, generator=gen, device=DEV)
    s["dx"] = torch.empty((case["batch"], length, vocab), device=DEV, dtype=kind)
    return s


# ----------------------------------------------------------------------------- the plain forms

def _plain_rows(s):
    """log p of every logit, p, logp, entropy, and the rows that are padding or empty."""
    c, tokens = s["case"], s["tokens"].long()
    x = s["x"].reshape(-1, c["vocab"]).float()
    pad = tokens < 0
    peak = x.max(1, keepdim=True).values
    empty = peak[:, 0] == -math.inf
    d = (x - torch.where(peak == -math.inf, 0.0, peak)) / c["temp"]
    lp = d - torch.exp(d).sum(1, keepdim=True).log()
    lp = torch.where(empty[:, None], -math.inf, lp)
    p = torch.exp(lp)
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    logp = lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    logp, entropy = torch.where(pad, 0.0, logp), torch.where(pad, 0.0, entropy)
    return x, lp, p, logp, entropy, pad, empty


def _plain_score(s):
    top = s["case"]["top"]
    x, lp, _, logp, entropy, pad, _ = _plain_rows(s)
    if not top:
        return {"logp": logp, "entropy": entropy}
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    top_logp = torch.where(pad[:, None], -math.inf, lp.gather(1, ids))
    ids = torch.where(pad[:, None], -1, ids).to(torch.int32)
    short = top - ids.shape[1]
    if short > 0:
        ids = torch.nn.functional.pad(ids, (0, short), value=-1)
        top_logp = torch.nn.functional.pad(top_logp, (0, short), value=-math.inf)
    return {"logp": logp, "entropy": entropy, "top_logp": top_logp, "top_ids": ids}


def _plain_gradient(s):
    c, tokens = s["case"], s["tokens"].long()
    _, lp, p, logp, entropy, pad, empty = _plain_rows(s)
    u, h = s["dlogp"][:, None], s["dentropy"][:, None]
    dx = -u * p - torch.where(p > 0, h * p * (lp + entropy[:, None]), 0.0)
    dx.scatter_add_(1, tokens.clamp(min=0)[:, None], u)
    dx = torch.where((pad | empty)[:, None], 0.0, dx / c["temp"])
    return {"logp": logp, "entropy": entropy, "dx": dx.to(s["x"].dtype).reshape(s["dx"].shape)}


def _plain_orth(g, steps):
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(steps):
        a = x @ x.transpose(-2, -1).contiguous()
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.transpose(-2, -1) if tall else x


def _plain_muon(s):
    g, m = torch.stack(s["g"]), torch.stack(s["m"])
    m = BETA * m + (1 - BETA) * g
    o = _plain_orth((1 - BETA) * g + BETA * m, s["case"]["steps"])
    scale = LR * math.sqrt(max(1.0, g.shape[1] / g.shape[2]))
    for k, p in enumerate(s["p"]):
        p.copy_(p * (1 - LR * DECAY) - scale * o[k])
        s["m"][k].copy_(m[k])
    return {"p": s["p"], "m": s["m"]}


# ----------------------------------------------------------------------------- the library's calls

def _struct(t, requires_grad=False, grad=None):
    from plast_amd import abi
    kind = {torch.float32: abi.FLOAT32, torch.bfloat16: abi.BFLOAT16, torch.float16: abi.FLOAT16,
            torch.int32: abi.INT32}[t.dtype]
    return abi.make_tensor(t.data_ptr(), t.shape, t.stride(), kind, abi.GPU, requires_grad, grad)


def _calls(s):
    """What a program sets up once around its buffers: the tensors' structs, the optimizer."""
    import ctypes as ct

    from plast_amd import abi
    from plast_amd.runtime import lib
    lib().plast_hip_set_sync(0)
    c, q = s["case"], {}
    if c["kind"] == "orth":
        q["g"], q["out"] = _struct(s["g"]), _struct(s["out"])
        q["rule"] = abi.NewtonSchulz(A, B, C, EPS, c["steps"])
    elif c["kind"] == "muon":
        q["grads"] = [_struct(t) for t in s["g"]]
        q["params"] = [_struct(t, True, g) for t, g in zip(s["p"], q["grads"])]
        q["moments"] = [_struct(t) for t in s["m"]]
        q["list"], q["keep"] = abi.tensor_array(*q["params"])
        q["held"], q["keep_m"] = abi.tensor_array(*q["moments"])
        rule = abi.NewtonSchulz(A, B, C, EPS, c["steps"])
        q["muon"] = abi.Muon(lr=LR, momentum=BETA, weight_decay=DECAY, nesterov=1, rule=rule,
                             m=ct.cast(q["held"], abi.TensorPP))
    else:
        q["dlogp"] = _struct(s["dlogp"]) if "dlogp" in s else None
        q["dentropy"] = _struct(s["dentropy"]) if "dlogp" in s else None
        q["dx"] = _struct(s["dx"]) if "dx" in s else None
        q["x"] = _struct(s["x"], "dx" in s, q["dx"])
        q["tokens"], q["stats"] = _struct(s["tokens"]), _struct(s["stats"])
        q["entropy"] = _struct(s["entropy"], "dx" in s, q["dentropy"])
        q["logp"] = _struct(s["logp"], "dx" in s, q["dlogp"])
        ins = [q["x"], q["tokens"], q["stats"], q["entropy"]]
        if c["kind"] == "score" and c["top"]:
            ins += [_struct(s["top_logp"]), _struct(s["top_ids"])]
        q["ins"] = ins
        q["params"] = abi.KernelParams(c["top"], 1, c["temp"])
    return q


def _own(s):
    import ctypes as ct

    from plast_amd.runtime import backward, forward, lib
    if "calls" not in s:
        s["calls"] = _calls(s)
    q, c = s["calls"], s["case"]
    if c["kind"] == "orth":
        lib().newton_schulz_hip(ct.byref(q["g"]), ct.byref(q["out"]), ct.byref(q["rule"]))
        lib().check("newton_schulz")
        return {"out": s["out"]}
    if c["kind"] == "muon":
        lib().muon_step_hip(ct.byref(q["muon"]), q["list"], len(s["p"]))
        lib().check("muon_step")
        return {"p": s["p"], "m": s["m"]}
    if c["kind"] == "step":
        lib().token_logprob_step_hip(ct.byref(q["x"]), ct.byref(q["tokens"]), ct.byref(q["dlogp"]),
                                     ct.byref(q["dentropy"]), ct.byref(q["logp"]),
                                     ct.byref(q["entropy"]), ct.byref(q["dx"]), c["temp"])
        lib().check("token_logprob_step")
        return {"logp": s["logp"], "entropy": s["entropy"], "dx": s["dx"]}
    forward("token_logprob", q["ins"], q["logp"], q["params"])
    got = {"logp": s["logp"], "entropy": s["entropy"]}
    if c["kind"] == "train":
        backward("token_logprob", q["ins"], q["logp"], q["params"])
        got["dx"] = s["dx"]
    elif c["top"]:
        got["top_logp"], got["top_ids"] = s["top_logp"], s["top_ids"]
    return got


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "orth":
        return {"out": _plain_orth(state["g"], state["case"]["steps"]).to(state["g"].dtype)}
    if kind == "muon":
        return _plain_muon(state)
    return _plain_score(state) if kind == "score" else _plain_gradient(state)


# ----------------------------------------------------------------------------- what a pass needs

def work(case):
    if case["kind"] in ("orth", "muon"):
        m, n = sorted((case["rows"], case["cols"]))
        # the two symmetric products count their half
        flops = case["steps"] * (2 * m * m * n + m * m * (n + m)) * case["count"]
        size = case["rows"] * case["cols"] * case["count"]
        return {"bytes": size * (20 if case["kind"] == "muon" else
                                 2 * TYPES[case["type"]].itemsize), "flops": flops}
    rows = case["batch"] * case["len"]
    live = case["batch"] * (case["len"] - case["pad"])
    item = TYPES[case["type"]].itemsize
    read = live * case["vocab"] * item + rows * 4
    wrote = rows * (8 + 8 * case["top"])
    if case["kind"] != "score":
        read, wrote = read + rows * 8, wrote + rows * case["vocab"] * item
    return {"bytes": read + wrote, "flops": 5 * live * case["vocab"]}


# ----------------------------------------------------------------------------- in 64 bits

def _exact_orth(g, steps):
    x = g.double()
    if x.shape[-2] > x.shape[-1]:
        return _exact_orth(g.transpose(-2, -1), steps).transpose(-2, -1)
    x = x / (torch.linalg.norm(x, dim=(-2, -1), keepdim=True) + EPS)
    for _ in range(steps):
        xt = x.transpose(-2, -1).contiguous()
        ax = torch.matmul(torch.matmul(x, xt), x)
        aax = torch.matmul(torch.matmul(x, xt), ax)
        x = A * x + B * ax + C * aax
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "orth":
        return {"out": torch.stack([_exact_orth(g, case["steps"]) for g in s["g"]])}
    if case["kind"] == "muon":
        p, m = [], []
        for w, g, v in zip(s["p"], s["g"], s["m"]):
            g, v = g.double(), v.double()
            m.append(v + (1 - BETA) * (g - v))
            o = _exact_orth(g + BETA * (m[-1] - g), case["steps"])
            scale = max(1.0, case["rows"] / case["cols"]) ** 0.5
            p.append(w.double() - LR * (DECAY * w.double() + scale * o))
        return {"p": p, "m": m}
    n, vocab = s["logp"].shape[0], case["vocab"]
    x = s["x"].reshape(n, vocab)
    grad = case["kind"] != "score"
    out = {"logp": torch.empty(n, device=DEV, dtype=torch.float64)}
    out["entropy"] = torch.empty_like(out["logp"])
    if grad:
        out["dx"] = torch.zeros((n, vocab), device=DEV, dtype=torch.float64)
    elif case["top"]:
        out["top_logp"] = torch.full((n, case["top"]), -math.inf, device=DEV, dtype=torch.float64)
        out["top_ids"] = None
    step = max(1, (1 << 26) // vocab)
    for r in range(0, n, step):
        z = x[r:r + step].double() / case["temp"]
        tok = s["tokens"][r:r + step].long()
        live = tok >= 0
        total = torch.logsumexp(z, 1)
        some = total > -math.inf
        lp = torch.where(some[:, None], z - total[:, None], -math.inf)
        p = torch.softmax(z, 1).nan_to_num(0.0)
        plogp = torch.special.xlogy(p, p)
        ent = -plogp.sum(1)
        rows = torch.arange(len(tok), device=DEV)
        out["logp"][r:r + step] = torch.where(live, lp[rows, tok.clamp(min=0)], 0.0)
        out["entropy"][r:r + step] = torch.where(live, ent, 0.0)
        if grad:
            u, h = s["dlogp"][r:r + step].double(), s["dentropy"][r:r + step].double()
            d = -p * (u - 0.0)[:, None] - h[:, None] * (plogp + p * ent[:, None])
            d[rows, tok.clamp(min=0)] += u
            out["dx"][r:r + step] = d * ((live & some) / case["temp"])[:, None]
        elif case["top"]:
            k = min(case["top"], vocab)
            best = torch.topk(lp, k, dim=1).values
            out["top_logp"][r:r + step, :k] = torch.where(live[:, None], best, -math.inf)
    if grad:
        out["dx"] = out["dx"].reshape(s["dx"].shape)
    return out
