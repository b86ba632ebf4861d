"""Cases of the mixture-of-experts operators: what runs between the attention layers of the hybrid stack.

Four operators, each a public call of ``router_ia.kernels``:

    route    moe_route       router logits -> the experts of each token and their weights
    quant    quant_fp8       activations -> e4m3 values with one power-of-two scale per 128 of a row
    linear   linear_fp8_x8   product of such activations with block-FP8 weights (one scale per 128 x 128)
    experts  moe_experts     the gated MLPs of the chosen experts, summed with the router's weights

The plain forms below are elementary torch operations in 32 bits, in 64 where a choice between
experts or a rounding to 8 bits hangs on the last digits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
BLOCK = 128
_PKG = str(Path(__file__).resolve().parents[1] / "router-ia_amd")


def _kernels():
    """The framework's entry points (imported where the framework's own operators are asked for)."""
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from router_ia import kernels

    return kernels


def listed():
    return [
        # One chat's decode step: the router of one layer, top 8 of 256, weights renormalised.
        {"name": "route_1", "kind": "route", "tokens": 1, "experts": 256, "top_k": 8, "dtype": "fp32",
         "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_score": "max", "renorm": True,
         "scale": 1.0, "shared": False, "masked": 0.0},
        # A batch of prompts with padding, routed with a balance bias inside the best 4 of 8 groups, and an
        # expert that every token visits.
        {"name": "route_4099_groups", "kind": "route", "tokens": 4099, "experts": 256, "top_k": 8, "dtype": "fp32",
         "scoring": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_score": "top2", "renorm": True,
         "scale": 2.5, "shared": True, "masked": 0.1},
        # Every token of a long prompt, logits as a 16-bit product leaves them (ties are common).
        {"name": "route_16384", "kind": "route", "tokens": 16384, "experts": 256, "top_k": 8, "dtype": "bf16",
         "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_score": "max", "renorm": True,
         "scale": 1.0, "shared": False, "masked": 0.0},
        # The normed hidden states of a serving batch of odd size.
        {"name": "quant_129", "kind": "quant", "rows": 129, "cols": 2048, "dtype": "fp16"},
        # The attention outputs of a long prompt, before the output projection.
        {"name": "quant_16384", "kind": "quant", "rows": 16384, "cols": 4096, "dtype": "bf16"},
        # One chat's decode step: a DeltaNet layer's input projection.
        {"name": "linear_1", "kind": "linear", "rows": 1, "n": 8192, "k": 2048, "dtype": "fp16"},
        # A short prompt through an output projection.
        {"name": "linear_333", "kind": "linear", "rows": 333, "n": 2048, "k": 4096, "dtype": "fp32"},
        # A long prompt through a DeltaNet layer's input projection.
        {"name": "linear_16384", "kind": "linear", "rows": 16384, "n": 8192, "k": 2048, "dtype": "bf16"},
        # One chat's decode step: the eight experts of one token.
        {"name": "experts_1", "kind": "experts", "tokens": 1, "experts": 256, "top_k": 8, "hidden": 2048,
         "inter": 512, "dtype": "fp16", "masked": 0.0},
        # A small serving batch with idle rows.
        {"name": "experts_21", "kind": "experts", "tokens": 21, "experts": 256, "top_k": 8, "hidden": 2048,
         "inter": 512, "dtype": "bf16", "masked": 0.1},
        # A full serving batch: nearly every expert has a few tokens.
        {"name": "experts_128", "kind": "experts", "tokens": 128, "experts": 256, "top_k": 8, "hidden": 2048,
         "inter": 512, "dtype": "fp16", "masked": 0.0},
        # A long prompt: some hundred tokens for every expert.
        {"name": "experts_16384", "kind": "experts", "tokens": 16384, "experts": 256, "top_k": 8, "hidden": 2048,
         "inter": 512, "dtype": "bf16", "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], odd ones as often as even ones."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["route", "quant", "linear", "linear", "experts", "experts"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_int(rng, max(2, 8 // groups), 512 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, top_groups * (experts // groups)))
        return {"kind": kind, "tokens": _log_int(rng, 1, 16384), "experts": experts, "top_k": top_k,
                "dtype": rng.choice(["fp32", "bf16", "fp16"]), "scoring": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "group_score": rng.choice(["max", "top2"]), "renorm": rng.random() < 0.7,
                "scale": rng.choice([1.0, 2.5]), "shared": rng.random() < 0.3,
                "masked": rng.choice([0.0, 0.0, 0.1])}
    if kind == "quant":
        return {"kind": kind, "rows": _log_int(rng, 1, 16384), "cols": BLOCK * _log_int(rng, 1, 32),
                "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    if kind == "linear":
        n, k = 16 * _log_int(rng, 2, 512), BLOCK * _log_int(rng, 1, 32)
        # no more products than the long prompt's, and no more results than fit its time
        most = min(16384, 2 ** 38 // (n * k), 2 ** 27 // n)
        return {"kind": kind, "rows": _log_int(rng, 1, most), "n": n, "k": k,
                "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    hidden, inter = BLOCK * _log_int(rng, 2, 24), BLOCK * _log_int(rng, 1, 8)
    # the weights of the largest listed case at most
    experts = min(256, 2 ** 28 // (hidden * inter), _log_int(rng, 8, 256))
    top_k = rng.randint(1, min(8, experts))
    most = min(16384, 2 ** 36 // (top_k * hidden * inter))
    return {"kind": kind, "tokens": _log_int(rng, 1, most), "experts": experts, "top_k": top_k, "hidden": hidden,
            "inter": inter, "dtype": rng.choice(["bf16", "fp16"]), "masked": rng.choice([0.0, 0.0, 0.1])}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _activations(g, rows, cols, dtype):
    """Normed hidden states: unit normal, a few channels ten times as large."""
    loud = 1.0 + 9.0 * (torch.rand((cols,), generator=g, device=DEV) < 0.01).float()
    return (torch.randn((rows, cols), generator=g, device=DEV) * loud).to(dtype)


def _weights(g, *shape):
    """e4m3 weights as a block-FP8 checkpoint holds them, and their scales: N(0, 0.02), the largest of a block at 448."""
    w = torch.randn(shape, generator=g, device=DEV)
    w = w.mul_(100.0).clamp_(-E4M3_MAX, E4M3_MAX).to(E4M3)
    blocks = shape[:-2] + ((shape[-2] + BLOCK - 1) // BLOCK, shape[-1] // BLOCK)
    return w, 2e-4 * (0.8 + 0.4 * torch.rand(blocks, generator=g, device=DEV))


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "route":
        t, e = case["tokens"], case["experts"]
        logits = torch.randn((t, e + int(case["shared"])), generator=g, device=DEV) * 1.5
        if case["masked"]:  # padding rows, and experts that are switched off for some tokens
            logits.masked_fill_(torch.rand((t, 1), generator=g, device=DEV) < case["masked"], -math.inf)
            logits[:, :e].masked_fill_(torch.rand((t, e), generator=g, device=DEV) < 0.02, -math.inf)
        bias = torch.randn((e,), generator=g, device=DEV) * 0.1 if case["bias"] else None
        return {"case": case, "logits": logits.to(dtype), "bias": bias}
    if kind == "quant":
        return {"case": case, "x": _activations(g, case["rows"], case["cols"], dtype)}
    if kind == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        x = _activations(g, m, k, torch.float32)
        top = x.reshape(m, k // BLOCK, BLOCK).abs().amax(-1)
        scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)))
        x8 = (x / scale.repeat_interleave(BLOCK, 1)).clamp_(-E4M3_MAX, E4M3_MAX).to(E4M3)
        w, s = _weights(g, n, k)
        return {"case": case, "x8": x8, "x_scale": scale, "w": w, "s": s}
    t, e, k, h, i = (case[q] for q in ("tokens", "experts", "top_k", "hidden", "inter"))
    w13, s13 = _weights(g, e, 2 * i, h)
    w2, s2 = _weights(g, e, h, i)
    # some experts are asked for more often than others
    logits = torch.randn((t, e), generator=g, device=DEV) + 0.25 * torch.randn((e,), generator=g, device=DEV)
    top, ids = torch.topk(logits, k, dim=-1)
    weights = torch.softmax(top, -1)
    if case["masked"]:
        idle = torch.rand((t, 1), generator=g, device=DEV) < case["masked"]
        ids = ids.masked_fill(idle, -1)
        weights = weights.masked_fill(idle, 0.0)
    return {"case": case, "x": _activations(g, t, h, dtype), "ids": ids.to(torch.int32), "weights": weights,
            "w13": w13, "s13": s13, "w2": w2, "s2": s2}


# ----------------------------------------------------------------------------- plain forms
def _expand(s, n):
    """One scale per 128 x 128 block -> one per element of [.., n, k]."""
    return s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)


def _plain_quant(x):
    """e4m3 values and scales: the smallest power of two that brings a block's largest finite value to 448 or less."""
    x = x.float()
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = torch.where(torch.isfinite(b), b, torch.zeros_like(b)).abs().amax(-1)
    mant, expo = torch.frexp(top)  # top = mant 2^expo, mant in [0.5, 1); 448 = 0.875 2^9
    expo = torch.where(mant > 0.875, expo - 8, expo - 9).clamp(min=-126)
    scale = torch.where(top > 0, torch.exp2(expo.double()).float(), torch.ones_like(top))
    q = b / scale[..., None]  # exact, but for results below e4m3's smallest
    q = torch.where(torch.isfinite(q), q, torch.full_like(q, math.nan)).to(E4M3)
    return q.reshape(x.shape), scale


def _plain_route(s):
    c, logits, bias = s["case"], s["logits"], s["bias"]
    t, e, k, groups = logits.shape[0], c["experts"], c["top_k"], c["groups"]
    x = logits[:, :e].double()
    if c["scoring"] == "softmax":
        top = x.amax(-1, keepdim=True)
        score = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        total = score.sum(-1, keepdim=True)
        score = score / torch.where(total == 0, torch.ones_like(total), total)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score + bias.double() if bias is not None else score
    choice = choice.masked_fill(x == -math.inf, -math.inf)
    if groups > 1:
        per = choice.reshape(t, groups, e // groups)
        best = torch.sort(per, dim=-1, descending=True).values
        rank = best[..., 0] if c["group_score"] == "max" or e == groups else best[..., 0] + best[..., 1]
        keep = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, : c["top_groups"]]
        open_ = torch.zeros((t, groups), dtype=torch.bool, device=x.device).scatter_(1, keep, True)
        choice = per.masked_fill(~open_[..., None], -math.inf).reshape(t, e)
    order = torch.sort(choice, dim=-1, descending=True, stable=True)
    ids, taken = order.indices[:, :k], order.values[:, :k] != -math.inf
    w = torch.gather(score, 1, ids) * taken
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total == 0, torch.ones_like(total), total)
    w = w * c["scale"]
    ids = torch.where(taken, ids, torch.full_like(ids, -1))
    if c["shared"]:
        gate = logits[:, e:].double()
        w = torch.cat([w, 1.0 / (1.0 + torch.exp(-gate))], 1)
        ids = torch.cat([ids, torch.where(gate == -math.inf, -1, e)], 1)
    return w.float(), ids.to(torch.int32)


def _plain_linear(s):
    x = s["x8"].float() * s["x_scale"].repeat_interleave(BLOCK, 1)
    w = s["w"].float() * _expand(s["s"], s["w"].shape[0])
    return (x @ w.t().contiguous()).to(DTYPES[s["case"]["dtype"]])


def _plain_experts(s):
    c, x = s["case"], s["x"]
    t, e, k, h, i = (c[q] for q in ("tokens", "experts", "top_k", "hidden", "inter"))
    ids, weights = s["ids"].long().reshape(-1), s["weights"].reshape(-1)
    used = ids >= 0
    q, scale = _plain_quant(x)
    xq = (q.float() * scale.repeat_interleave(BLOCK, 1))
    token = torch.arange(t, device=x.device).repeat_interleave(k)
    if t * k <= e:  # each pair's own weights
        bank, home, place = ids.clamp(min=0), torch.arange(t * k, device=x.device), 0
        rows = (xq[token] * used[:, None])[:, None]
    else:  # the pairs in the order of their experts, each expert's padded to the longest
        bank, home = slice(None), ids.clamp(min=0)
        counts = torch.bincount(ids[used], minlength=e)
        order = torch.sort(torch.where(used, ids, e), stable=True).indices
        rank = torch.empty_like(order).scatter_(0, order, torch.arange(t * k, device=x.device))
        place = torch.where(used, rank - (counts.cumsum(0) - counts)[home], 0)
        rows = torch.zeros((e, max(1, int(counts.max())), h), device=x.device)
        rows[home[used], place[used]] = xq[token[used]]
    w13 = (s["w13"][bank].float() * _expand(s["s13"][bank], 2 * i)).transpose(1, 2).contiguous()
    up = torch.bmm(rows, w13)
    del w13, rows
    gate, up = up[..., :i], up[..., i:]
    a, scale = _plain_quant(gate / (1.0 + torch.exp(-gate)) * up)
    a = a.float() * scale.repeat_interleave(BLOCK, -1)
    del gate, up
    w2 = (s["w2"][bank].float() * _expand(s["s2"][bank], h)).transpose(1, 2).contiguous()
    y = torch.bmm(a, w2)[home, place] * (weights * used)[:, None]
    return y.reshape(t, k, h).sum(1).to(x.dtype)


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        K = _kernels()
        if kind == "route":
            return K.moe_route(s["logits"], c["top_k"], scoring=c["scoring"], bias=s["bias"],
                               num_groups=c["groups"], top_groups=c["top_groups"], group_score=c["group_score"],
                               renormalize=c["renorm"], scale=c["scale"], shared_expert=c["shared"])
        if kind == "quant":
            return K.quant_fp8(s["x"])
        if kind == "linear":
            return K.linear_fp8_x8(s["x8"], s["x_scale"], s["w"], s["s"], out_dtype=DTYPES[c["dtype"]])
        return K.moe_experts(s["x"], s["ids"], s["weights"], s["w13"], s["s13"], s["w2"], s["s2"])
    if kind == "route":
        return _plain_route(s)
    if kind == "quant":
        return _plain_quant(s["x"])
    if kind == "linear":
        return _plain_linear(s)
    return _plain_experts(s)


# ----------------------------------------------------------------------------- required work
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def work(case):
    b = _BYTES[case["dtype"]]
    if case["kind"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        s = int(case["shared"])
        return {"bytes": t * ((e + s) * b + (k + s) * 8) + 4 * e * case["bias"], "flops": t * e * 4}
    if case["kind"] == "quant":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (b + 1) + n // BLOCK * 4, "flops": 2 * n}
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * k + m * (k // BLOCK) * 4 + n * k + -(-n // BLOCK) * (k // BLOCK) * 4 + m * n * b,
                "flops": 2 * m * n * k}
    t, e, k, h, i = (case[q] for q in ("tokens", "experts", "top_k", "hidden", "inter"))
    t_used = t * (1.0 - case["masked"])
    some = e * (1.0 - (1.0 - k / e) ** t_used)  # experts with a token, were all asked for alike
    weights = some * 3 * h * i * (1 + 4 / BLOCK ** 2)
    return {"bytes": weights + 2 * t * h * b + t * k * 8, "flops": 6.0 * t_used * k * h * i}


# ----------------------------------------------------------------------------- definitions in 64 bits
def _round_e4m3(v):
    """The e4m3 value nearest to v (64 bits, |v| <= 448): 4 significant bits, ties to even, steps of 2^-9 at the least."""
    expo = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20)))
    step = torch.exp2(torch.clamp(expo, min=-6.0) - 3.0)
    return torch.round(v / step) * step


def _exact_quant(v):
    v = v.double()
    blocks = v.unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.clamp(torch.ceil(torch.log2(top / E4M3_MAX)), min=-126.0))
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    return _round_e4m3(blocks / scale).flatten(-2), scale.squeeze(-1)


def _exact_route(case, s):
    e, k, groups = case["experts"], case["top_k"], case["groups"]
    weights, ids = [], []
    for logits in s["logits"].double().split(1024):
        x = logits[:, :e]
        off = x == -math.inf
        if case["scoring"] == "softmax":
            p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        else:
            p = torch.sigmoid(x)
        c = p if s["bias"] is None else p + s["bias"].double()
        c = c.masked_fill(off, -math.inf)
        index = torch.arange(e, device=x.device)

        def beaten_by(v, at):  # how many come before each: the larger ones, and equal ones of a lower index
            a, b = v[:, None, :], v[:, :, None]
            return ((a > b) | ((a == b) & (at[None, None, :] < at[None, :, None]))).sum(-1)

        if groups > 1:
            g = c.unflatten(1, (groups, -1))
            if case["group_score"] == "max" or g.shape[-1] == 1:
                gs = g.amax(-1)
            else:
                gs = torch.topk(g, 2, dim=-1).values.sum(-1)
            shut = beaten_by(gs, index[:groups]) >= case["top_groups"]
            c = c.masked_fill(shut.repeat_interleave(e // groups, 1), -math.inf)
        rank = beaten_by(c, index)
        pick = torch.argsort(rank, dim=-1)[:, :k]
        live = torch.gather(c, 1, pick) > -math.inf
        w = torch.where(live, torch.gather(p, 1, pick), 0.0)
        if case["renorm"]:
            w = torch.nan_to_num(w / w.sum(-1, keepdim=True), nan=0.0)
        w, pick = w * case["scale"], torch.where(live, pick, -1)
        if case["shared"]:
            w = torch.cat([w, torch.sigmoid(logits[:, e:])], 1)
            pick = torch.cat([pick, torch.where(logits[:, e:] > -math.inf, e, -1)], 1)
        weights.append(w)
        ids.append(pick.to(torch.int32))
    return torch.cat(weights), torch.cat(ids)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, s)
    if case["kind"] == "quant":
        return _exact_quant(s["x"])

    def wide(w, scale):  # w [n, k] with its block scales, in 64 bits
        n, k = w.shape
        at = torch.arange(n, device=w.device)[:, None] // BLOCK, torch.arange(k, device=w.device)[None] // BLOCK
        return w.double() * scale.double()[at]

    if case["kind"] == "linear":
        m, k = s["x8"].shape
        x = (s["x8"].double().unflatten(1, (-1, BLOCK)) * s["x_scale"].double()[..., None]).flatten(1)
        return x @ wide(s["w"], s["s"]).T
    q, scale = _exact_quant(s["x"])
    x = (q.unflatten(1, (-1, BLOCK)) * scale[..., None]).flatten(1)
    i = case["inter"]
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        rows, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if rows.numel() == 0:
            continue
        z = x[rows] @ wide(s["w13"][e], s["s13"][e]).T
        a = z[:, :i] * torch.sigmoid(z[:, :i]) * z[:, i:]
        a, scale = _exact_quant(a)
        a = (a.unflatten(1, (-1, BLOCK)) * scale[..., None]).flatten(1)
        out.index_add_(0, rows, a @ wide(s["w2"][e], s["s2"][e]).T * s["weights"][rows, slot].double()[:, None])
    return out
