"""GPU parity: expert routing, e4m3 activations, FP8 x FP8 products and the experts' MLPs.

Every operator is compared with its definition in 64 bits, computed here on the
CPU from the same inputs.  Tolerances count roundings: half a step of the
output's type (eps / 2 relative), and for fp32 sums of n terms the error of
their order, n * 2^-24 of the sum of the terms' magnitudes at most.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import pytest
import torch

from conftest import announce
from router_ia import kernels as K

pytestmark = pytest.mark.gpu

BLOCK = 128
E4M3 = torch.float8_e4m3fn


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


# ----------------------------------------------------------------------------- definitions in 64 bits
def quant64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 values as float64, scales): the smallest power of two s with |x| / s <= 448 for the finite x of a block."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    top = torch.where(torch.isfinite(b), b, 0.0).abs().amax(-1)
    s = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-126.0))
    s = torch.where(top > 0, s, 1.0)
    v = b / s[..., None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0) - 3.0)
    q = torch.where(torch.isfinite(v), torch.round(v / step) * step, math.nan)
    return q.flatten(-2), s


def widen(w: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """Block-scaled e4m3 weights [.., n, k] in 64 bits."""
    n, k = w.shape[-2:]
    return w.double() * s.double().repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def rows64(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return (q.double().unflatten(-1, (-1, BLOCK)) * s.double()[..., None]).flatten(-2)


def route64(logits, k, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_score="top2",
            renormalize=True, scale=1.0, shared_expert=False):
    e = logits.shape[1] - int(shared_expert)
    out_w, out_i = [], []
    for row in logits.double():
        x = [float(v) for v in row[:e]]
        if scoring == "softmax":
            m = max(x)
            p = [math.exp(v - m) if v > -math.inf else 0.0 for v in x]
            z = sum(p)
            p = [v / z if z else 0.0 for v in p]
        else:
            p = [1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0 for v in x]
        c = [a + (float(bias[i]) if bias is not None else 0.0) if x[i] > -math.inf else -math.inf
             for i, a in enumerate(p)]
        per = e // num_groups
        rank = []
        for g in range(num_groups):
            best = sorted(c[g * per:(g + 1) * per], reverse=True)
            rank.append(best[0] if group_score == "max" or per == 1 else best[0] + best[1])
        keep = sorted(range(num_groups), key=lambda g: (-rank[g], g))[:top_groups]
        order = sorted((i for i in range(e) if i // per in keep and c[i] > -math.inf), key=lambda i: (-c[i], i))[:k]
        w = [p[i] for i in order]
        if renormalize and sum(w):
            w = [v / sum(w) for v in w]
        w = [v * scale for v in w] + [0.0] * (k - len(order))
        order = order + [-1] * (k - len(order))
        if shared_expert:
            gate = float(row[e])
            w.append(1.0 / (1.0 + math.exp(-gate)) if gate > -700 else 0.0)
            order.append(e if gate > -math.inf else -1)
        out_w.append(w)
        out_i.append(order)
    return torch.tensor(out_w, dtype=torch.float64), torch.tensor(out_i, dtype=torch.int32)


class Mags(NamedTuple):
    terms: torch.Tensor
    products: torch.Tensor


def experts64(x, ids, weights, w13, s13, w2, s2):
    """The sum over the slots and, for the tolerance, Mags: of the slots' terms, and of the products they sum."""
    e, i = w13.shape[0], w2.shape[2]
    xq = rows64(*quant64(x))
    out = torch.zeros(x.shape, dtype=torch.float64)
    mag = Mags(torch.zeros_like(out), torch.zeros_like(out))
    for j in range(e):
        rows, slot = torch.nonzero(ids == j, as_tuple=True)
        if rows.numel() == 0:
            continue
        z = xq[rows] @ widen(w13[j], s13[j]).T
        a = z[:, :i] * torch.sigmoid(z[:, :i]) * z[:, i:]
        aq, down, pw = rows64(*quant64(a)), widen(w2[j], s2[j]).T, weights[rows, slot].double()[:, None]
        term = aq @ down * pw
        out.index_add_(0, rows, term)
        mag.terms.index_add_(0, rows, term.abs())
        mag.products.index_add_(0, rows, aq.abs() @ down.abs() * pw.abs())
    return out, mag


# ----------------------------------------------------------------------------- inputs
def gen(seed):
    return torch.Generator().manual_seed(seed)


def e4m3_weight(seed, *shape):
    g = gen(seed)
    w = (torch.randn(shape, generator=g) * 100.0).clamp(-448, 448).to(E4M3)
    blocks = shape[:-2] + ((shape[-2] + BLOCK - 1) // BLOCK, shape[-1] // BLOCK)
    return w, 2e-4 * (0.5 + torch.rand(blocks, generator=g))


# ----------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 128), (3, 384), (129, 2048), (517, 896)])
def test_quant_matches_definition_bit_for_bit(gpu, m, k, dtype):
    announce(f"quant_fp8: {m} x {k} {dtype}")
    x = torch.randn((m, k + 8), generator=gen(m + k)) * torch.exp(3 * torch.randn((m, 1), generator=gen(k)))
    x = x.to(dtype)
    q, s = K.quant_fp8(x.to(gpu)[:, :k])  # rows of a wider buffer
    x = x[:, :k]
    want_q, want_s = quant64(x)
    assert torch.equal(s.cpu().double(), want_s)
    assert torch.equal(q.cpu().double(), want_q)


def test_quant_edges(gpu):
    """Zero blocks, the largest and smallest fp32, exact 448 multiples, ties, infinities and NaN."""
    announce("quant_fp8: edge values")
    x = torch.zeros((10, 128))
    x[1, 0] = 448.0                      # scale 1 exactly
    x[2, 0] = 448.0000305                # the next fp32: scale 2
    x[3] = torch.linspace(-3e38, 3e38, 128)
    x[4, :4] = torch.tensor([1e-45, 2e-45, -1e-44, 0.0])  # smallest fp32 values: scale 2^-126
    x[5, :8] = torch.tensor([448.0, 17.0, 19.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, -2.0 ** -10])  # ties
    x[6, :4] = torch.tensor([math.inf, -math.inf, 3.0, math.nan])
    x[7] = math.nan
    x[8, 5] = -math.inf
    x[9] = torch.randn(128, generator=gen(9)) * 1e-30
    q, s = K.quant_fp8(x.to(gpu))
    want_q, want_s = quant64(x)
    assert torch.equal(s.cpu().double(), want_s)
    torch.testing.assert_close(q.cpu().double(), want_q, rtol=0, atol=0, equal_nan=True)


# ----------------------------------------------------------------------------- dense product
LINEAR = [  # (m, n, k)
    (1, 16, 128), (1, 8192, 2048), (2, 48, 256), (5, 400, 1152), (16, 512, 2048), (17, 2048, 4096), (33, 144, 128),
    (64, 1040, 640), (100, 2048, 512), (129, 272, 2048), (200, 1536, 384), (300, 2048, 4096), (513, 784, 896),
    (1025, 4112, 256), (40, 96, 128), (70, 80, 384), (4001, 4080, 384),
    (1500, 3088, 512), (2001, 8176, 1152),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear_x8_matches_definition(gpu, m, n, k, dtype):
    announce(f"linear_fp8_x8: {m} x {n} x {k} -> {dtype}")
    x = torch.randn((m, k), generator=gen(m)) * (1 + 9 * (torch.rand((k,), generator=gen(k)) < 0.02))
    q, s = quant64(x)
    s = s * (0.5 + torch.rand(s.shape, generator=gen(n)))  # any fp32 scales are taken
    q, s = q.to(E4M3), s.float()
    w, ws = e4m3_weight(n + k, n, k)
    # rows of wider buffers
    qd = torch.nn.functional.pad(q.view(torch.uint8), (0, 16)).to(gpu)[:, :k].view(E4M3)
    sd = torch.nn.functional.pad(s, (0, 3)).to(gpu)[:, : k // BLOCK]
    y = K.linear_fp8_x8(qd, sd, w.to(gpu), ws.to(gpu), out_dtype=dtype)
    xw, ww = rows64(q, s), widen(w, ws)
    want, mag = xw @ ww.T, xw.abs() @ ww.abs().T
    # k products summed in fp32 in some order, two scalings per block, and the rounding of the result
    tol = half_step(dtype) * want.abs() + (k + 4) * 2.0 ** -24 * mag
    if dtype != torch.float32:
        # 16-bit results may come from the matrix cores' e4m3 products, which cut each product of a group of 16
        # 13 bits below the group's largest: 16 * 2^-13 of the largest, itself at most the group's magnitudes
        tol = tol + 2.0 ** -9 * mag
    err = (y.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"{(err / tol).max().item():.3g} of the tolerance"


def test_linear_x8_accumulate_strided_out_and_stream(gpu):
    announce("linear_fp8_x8: accumulate into a strided fp32 out, another stream")
    m, n, k = 37, 272, 256
    q, s = quant64(torch.randn((m, k), generator=gen(1)))
    w, ws = e4m3_weight(2, n, k)
    base = torch.randn((m, n + 12), generator=gen(3))
    out = base.to(gpu)
    args = q.to(E4M3).to(gpu), s.float().to(gpu), w.to(gpu), ws.to(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.linear_fp8_x8(*args, out=out[:, 5:5 + n], accumulate=True)
    side.synchronize()
    want = base.double()
    want[:, 5:5 + n] += rows64(q, s) @ widen(w, ws).T
    mag = rows64(q, s).abs() @ widen(w, ws).abs().T
    got = out.cpu().double()
    assert torch.equal(got[:, :5], base[:, :5].double()) and torch.equal(got[:, 5 + n:], base[:, 5 + n:].double())
    tol = 2.0 ** -24 * want[:, 5:5 + n].abs() + (k + 4) * 2.0 ** -24 * mag
    assert bool(((got - want)[:, 5:5 + n].abs() <= tol).all())


def test_linear_x8_nan_stays_in_its_row(gpu):
    announce("linear_fp8_x8: a NaN value shows in its row alone")
    x = torch.randn((20, 256), generator=gen(1))
    x[7, 130] = math.nan
    q, s = K.quant_fp8(x.to(gpu))
    w, ws = e4m3_weight(2, 64, 256)
    y = K.linear_fp8_x8(q, s, w.to(gpu), ws.to(gpu)).cpu()
    bad = torch.isnan(y)
    assert bool(bad[7].all()) and not bool(bad[torch.arange(20) != 7].any())


# ----------------------------------------------------------------------------- routing
ROUTES = [
    dict(t=1, e=256, k=8),
    dict(t=5, e=8, k=8),
    dict(t=67, e=60, k=4, renormalize=False),
    dict(t=33, e=100, k=7, scoring="sigmoid", scale=2.5),
    dict(t=40, e=256, k=8, scoring="sigmoid", bias=True, num_groups=8, top_groups=4, shared_expert=True),
    dict(t=30, e=160, k=6, num_groups=8, top_groups=3, group_score="max"),
    dict(t=30, e=160, k=6, num_groups=8, top_groups=3, group_score="top2"),
    dict(t=30, e=24, k=3, num_groups=24, top_groups=5, bias=True),
    dict(t=30, e=512, k=16, bias=True, scale=0.5, renormalize=False),
    dict(t=9, e=1000, k=32, num_groups=4, top_groups=2, bias=True, shared_expert=True),
    dict(t=9, e=1, k=1),
    # groups of 1, 4 and 8 lanes of a wave that takes four tokens; of no whole lanes, or no power of two of them
    dict(t=50, e=256, k=16, bias=True, num_groups=16, top_groups=3),
    dict(t=50, e=128, k=6, num_groups=4, top_groups=2, group_score="top2", renormalize=False),
    dict(t=50, e=256, k=8, scoring="sigmoid", num_groups=2, top_groups=1, group_score="max", renormalize=False),
    dict(t=50, e=48, k=4, bias=True, num_groups=3, top_groups=2, group_score="max", shared_expert=True),
    dict(t=50, e=64, k=5, scoring="sigmoid", bias=True, num_groups=2, top_groups=2, scale=3.0),
    dict(t=50, e=256, k=8, bias=True, num_groups=64, top_groups=9),
    dict(t=50, e=96, k=3, bias=True, num_groups=2, top_groups=1),
    dict(t=50, e=256, k=8, scoring="softmax", num_groups=2, top_groups=1, group_score="max", renormalize=False),
    # groups of 1, 4, 8, 16 and 32 lanes of a wave that takes one token
    dict(t=20, e=60, k=7, scoring="sigmoid", bias=True, num_groups=60, top_groups=20),
    dict(t=20, e=256, k=20, bias=True, num_groups=16, top_groups=5),
    dict(t=20, e=512, k=9, bias=True, num_groups=8, top_groups=3),
    dict(t=20, e=1024, k=11, scoring="sigmoid", bias=True, num_groups=4, top_groups=2),
    dict(t=20, e=1024, k=32, num_groups=2, top_groups=1, group_score="max"),
]


# tokens from which scores are compared in 64 bits at once, in fp32 first again, and by a wave of four tokens
SOME, MORE, MANY = 32 + 3, 3200 + 3, 32768 + 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", ROUTES, ids=lambda c: f"t{c['t']}_e{c['e']}_k{c['k']}")
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("many", [0, SOME, MORE, MANY])
def test_route_matches_definition(gpu, case, dtype, masked, many):
    c = dict(case)
    t, e, k = c.pop("t"), c.pop("e"), c.pop("k")
    announce(f"moe_route: {t} tokens, {k} of {e} {dtype} {c} masked {masked}")
    cols = e + int(c.get("shared_expert", False))
    x = (torch.randn((t, cols), generator=gen(e + t)) * 1.5).to(dtype)
    if masked:
        x.masked_fill_(torch.rand((t, cols), generator=gen(e)) < 0.6, -math.inf)
        x[0] = -math.inf
    if c.pop("bias", False):
        c["bias"] = torch.randn((e,), generator=gen(3)) * 0.2
    want_w, want_i = route64(x, k, **c)
    if many:  # the same tokens again and again
        x, want_w, want_i = (v.repeat(many // t + 1, 1)[:many] for v in (x, want_w, want_i))
    if "bias" in c:
        c["bias"] = c["bias"].to(gpu)
    wide = torch.nn.functional.pad(x, (0, 5)).to(gpu)[:, :cols]
    w, i = K.moe_route(wide, k, **c)
    assert torch.equal(i.cpu(), want_i)
    # computed in 64 bits (or fp32 with a handful of roundings), rounded once to fp32
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=16 * 2.0 ** -24, atol=1e-38)


def test_route_ties_go_to_the_lowest_index(gpu):
    announce("moe_route: ties")
    x = torch.zeros((3, 130))
    x[1, 100:] = 1.0
    x[2, ::2] = -0.0
    w, i = K.moe_route(x.to(gpu), 5)
    assert i.cpu().tolist() == [[0, 1, 2, 3, 4], [100, 101, 102, 103, 104], [0, 1, 2, 3, 4]]
    torch.testing.assert_close(w.cpu(), torch.full((3, 5), 0.2), rtol=2.0 ** -23, atol=0)
    _, i = K.moe_route(torch.zeros((1, 64), device=gpu), 3, scoring="sigmoid", num_groups=8, top_groups=2,
                       bias=torch.zeros(64, device=gpu))
    assert i.cpu().tolist() == [[0, 1, 2]]


@pytest.mark.parametrize("many", [0, SOME, MORE, MANY])
def test_route_near_ties_follow_64_bits(gpu, many):
    """A bias that brings unlike scores within 1e-9 of each other: fp32 could not order them."""
    announce("moe_route: scores and biases that nearly cancel")
    g = gen(5)
    x = torch.randn((64, 128), generator=g)
    p = torch.sigmoid(x[0].double())
    bias = (1.0 - p).float()  # token 0: every choice within fp32 roundings of 1
    want_w, want_i = route64(x, 8, scoring="sigmoid", bias=bias)
    if many:
        x, want_w, want_i = (v.repeat(many // 64 + 1, 1)[:many] for v in (x, want_w, want_i))
    w, i = K.moe_route(x.to(gpu), 8, scoring="sigmoid", bias=bias.to(gpu))
    assert torch.equal(i.cpu(), want_i)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=16 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("many", [0, SOME, MORE, MANY])
@pytest.mark.parametrize("groups", [1, 8])
def test_route_near_ties_in_one_place(gpu, groups, many):
    """The chosen experts and the next one, 1e-9 apart, are neighbours; every other token is far from a tie."""
    announce(f"moe_route: near ties in experts 16 to 31, {groups} groups")
    x = torch.randn((37, 256), generator=gen(6))
    p = torch.sigmoid(x[5].double())
    bias = torch.full((256,), -3.0)
    bias[16:32] = (1.0 - p[16:32]).float()
    c = dict(scoring="sigmoid", num_groups=groups, top_groups=max(groups // 2, 1))
    want_w, want_i = route64(x, 8, bias=bias, **c)
    if many:
        x, want_w, want_i = (v.repeat(many // 37 + 1, 1)[:many] for v in (x, want_w, want_i))
    w, i = K.moe_route(x.to(gpu), 8, bias=bias.to(gpu), **c)
    assert torch.equal(i.cpu(), want_i)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=16 * 2.0 ** -24, atol=0)


def test_route_extreme_logits(gpu):
    announce("moe_route: saturated, infinite and NaN logits")
    x = torch.zeros((6, 16))
    x[0] = -200.0
    x[0, 3] = -190.0
    x[1] = torch.linspace(50.0, 80.0, 16)      # sigmoids that round to 1: the logits rank
    x[2, 2], x[2, 9] = math.nan, 5.0
    x[3, 4] = math.inf
    x[4] = -3e38
    x[5] = 3e38
    w, i = K.moe_route(x.to(gpu), 2, scoring="softmax")
    w, i = w.cpu(), i.cpu()
    assert i[0].tolist() == [3, 0] and i[1].tolist() == [15, 14] and i[4].tolist() == [0, 1] and i[5].tolist() == [0, 1]
    assert i[2].tolist() == [2, 9] and bool(torch.isnan(w[2]).all())
    assert i[3, 0] == 4 and bool(torch.isnan(w[3]).any())
    torch.testing.assert_close(w[0], torch.tensor([1.0, math.exp(-10.0)]) / (1 + math.exp(-10.0)), rtol=1e-6, atol=0)
    w, i = K.moe_route(x.to(gpu), 2, scoring="sigmoid")
    assert i[1].tolist() == [15, 14] and i[0].tolist() == [3, 0]
    torch.testing.assert_close(w[0].cpu(), torch.tensor([1.0, math.exp(-10.0)]) / (1 + math.exp(-10.0)), rtol=1e-6, atol=0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("many", [SOME, MORE, MANY])
def test_route_extreme_logits_of_many_tokens(gpu, scoring, groups, many):
    """Tokens with infinities and NaN choose the same experts in a large batch as in a small one."""
    announce(f"moe_route: infinite and NaN logits, {scoring}, {groups} groups, {many} tokens")
    x = torch.randn((7, 64), generator=gen(8))
    x[0, 40], x[0, 9] = math.nan, 5.0
    x[1, 4] = math.inf
    x[2, 3:] = -math.inf
    x[3] = math.nan
    x[4, 7], x[4, 50] = 3e38, -3e38
    x[5] = -200.0
    c = dict(scoring=scoring, bias=torch.linspace(0, 0.5, 64).to(gpu), num_groups=groups, top_groups=1)
    want_w, want_i = K.moe_route(x.to(gpu), 4, **c)
    w, i = K.moe_route(x.repeat(many // 7 + 1, 1)[:many].to(gpu), 4, **c)
    assert torch.equal(i, want_i.repeat(many // 7 + 1, 1)[:many])
    # both sum and divide in fp32, in orders of their own
    torch.testing.assert_close(w, want_w.repeat(many // 7 + 1, 1)[:many], rtol=32 * 2.0 ** -24, atol=0, equal_nan=True)


# ----------------------------------------------------------------------------- experts
EXPERTS = [  # (tokens, experts, top_k, hidden, inter)
    (1, 8, 2, 256, 128), (1, 16, 8, 2048, 512), (2, 4, 1, 128, 128), (3, 5, 5, 384, 256), (7, 16, 3, 512, 640),
    (17, 3, 2, 256, 128), (40, 33, 4, 256, 384), (130, 6, 2, 640, 256), (200, 2, 2, 256, 128), (300, 40, 6, 512, 128),
    (700, 3, 2, 256, 256), (2100, 5, 2, 256, 128), (400, 20, 1, 384, 256), (900, 24, 2, 640, 128),
    # tiles of 256 pairs, the last features' half empty; more experts than a planning workgroup has threads
    (2048, 16, 2, 256, 1024), (1500, 12, 3, 384, 1408), (300, 700, 3, 128, 128), (2000, 1024, 4, 128, 128), (5000, 300, 2, 128, 128),
    (1700, 40, 3, 256, 1024),  # tiles of 64 pairs, more than two a CU
]


def expert_inputs(t, e, k, h, i, dtype, seed):
    g = gen(seed)
    x = torch.randn((t, h), generator=g).to(dtype)
    ids = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(t)]).to(torch.int32)
    weights = torch.rand((t, k), generator=g) + 0.05
    w13, s13 = e4m3_weight(seed + 1, e, 2 * i, h)
    w2, s2 = e4m3_weight(seed + 2, e, h, i)
    return x, ids, weights, w13, s13, w2, s2


def expert_tolerance(out, mag, i, dtype, slack):
    """Roundings of the slots' terms and of the sum to out's type, and the fp32 sums' own.

    Terms are kept to 11 bits or more, or in out's type's step; a sum of i
    products in fp32, its scalings and the sum over the slots are off by at
    most (i + 16) 2^-24 of the products' magnitudes.

    The hidden values are e4m3: where an fp32 sum of another order lies on the
    other side of a rounding border, one value moves by a step, 2^-3 of itself
    at most.  `slack` bounds what such moves add, relative to the row's size.
    """
    size = out.abs().amax(-1, keepdim=True)
    return half_step(dtype) * (out.abs() + mag.terms) + (i + 16) * 2.0 ** -24 * mag.products + slack * size


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,e,k,h,i", EXPERTS)
def test_experts_match_definition(gpu, t, e, k, h, i, dtype):
    announce(f"moe_experts: {t} tokens, {k} of {e}, {h} x {i} {dtype}")
    a = expert_inputs(t, e, k, h, i, dtype, t + h)
    if t > 2:
        a[1][1] = -1              # a token without experts
        a[1][2, 0] = e            # ids past the experts add nothing
    want, mag = experts64(*a)
    out = K.moe_experts(*(v.to(gpu) for v in a)).cpu().double()
    assert out.shape == want.shape
    if t > 2:
        assert not bool(out[1].any())
    # one value of `i` moved by 2^-3 of itself changes a term by 2^-3 / sqrt(i) of its size, typically;
    # the largest values are 4 sigma, and two may move in a row
    err, tol = (out - want).abs(), expert_tolerance(want, mag, i, dtype, 0.125 * 4 * 2 / math.sqrt(i))
    assert bool((err <= tol).all()), f"{(err / tol).max().item():.3g} of the tolerance"
    if dtype != torch.float32:
        return
    # with an fp32 out every sum is in fp32, and such moves are rare: two fp32 sums of one value differ by some 2^-22 of it, its borders lie 2^-3 apart, so one
    # of 2^19 / (4 sizes of safety) values moves; every other row lies within the roundings alone
    tight = expert_tolerance(want, mag, i, dtype, 0.0)
    moved = int((err > tight).any(-1).sum())
    assert moved <= 1 + math.ceil(t * k * i * 2.0 ** -17), f"{moved} of {t} rows"


def device(a, gpu):
    return [v.to(gpu) for v in a]


def check_experts(out, want, mag, i, dtype):
    err = (out.cpu().double() - want).abs()
    tol = expert_tolerance(want, mag, i, dtype, 0.125 * 4 * 2 / math.sqrt(i))
    assert bool((err <= tol).all()), f"{(err / tol).max().item():.3g} of the tolerance"


@pytest.mark.parametrize("t", [1, 9, 150])
def test_experts_accumulate_strided_and_on_another_stream(gpu, t):
    """16-bit x into an fp32 residual stream: rows of wider buffers, a workspace of the caller's, another stream."""
    announce(f"moe_experts: {t} tokens, accumulate")
    e, k, h, i = 6, 2, 384, 256
    x, ids, weights, *w = expert_inputs(t, e, k, h, i, torch.float16, 77 + t)
    want, mag = experts64(x, ids, weights, *w)
    base = torch.randn((t, h + 12), generator=gen(5))
    out = base.to(gpu)
    wide_x = torch.nn.functional.pad(x, (0, 8)).to(gpu)[:, :h]
    wide_ids = torch.nn.functional.pad(ids, (0, 3)).to(gpu)[:, :k]
    wide_w = torch.nn.functional.pad(weights, (0, 5)).to(gpu)[:, :k]
    w = device(w, gpu)
    ws = torch.empty(K.moe_experts_workspace_bytes(t, k, e, h, i) + 7, dtype=torch.uint8, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.moe_experts(wide_x, wide_ids, wide_w, *w, out=out[:, 4:4 + h], accumulate=True, workspace=ws)
    side.synchronize()
    assert got.data_ptr() == out[:, 4:].data_ptr()
    out = out.cpu()
    assert torch.equal(out[:, :4], base[:, :4]) and torch.equal(out[:, 4 + h:], base[:, 4 + h:])
    # the terms are fp16 (x's type), their sum and the residual fp32
    err = (out[:, 4:4 + h].double() - base[:, 4:4 + h].double() - want).abs()
    tol = expert_tolerance(want, mag, i, torch.float16, 0.125 * 4 * 2 / math.sqrt(i)) + 2.0 ** -23 * out[:, 4:4 + h].abs()
    assert bool((err <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("t", [2, 70, 1200])
def test_experts_all_tokens_to_one_expert_and_twice(gpu, t, dtype):
    """The whole batch on one expert (the others' tiles empty), some rows naming it in both slots."""
    announce(f"moe_experts: {t} tokens on one expert of 7")
    e, k, h, i = 7, 2, 256, 128
    x, ids, weights, *w = expert_inputs(t, e, k, h, i, dtype, 3)
    ids[:] = 5
    ids[1::2, 1] = -7
    want, mag = experts64(x, ids, weights, *w)
    out = K.moe_experts(*device((x, ids, weights, *w), gpu))
    check_experts(out, want, mag, i, dtype)


@pytest.mark.parametrize("t", [3, 90])
def test_experts_without_any(gpu, t):
    """No slot names an expert: zeros, also over what out held; with accumulate out stays."""
    announce("moe_experts: every id out of range")
    e, k, h, i = 4, 3, 256, 128
    x, ids, weights, *w = device(expert_inputs(t, e, k, h, i, torch.bfloat16, 9), gpu)
    ids.fill_(-1)
    ids[:, 1] = e
    ids[:, 2] = 2 ** 31 - 1
    out = torch.full((t, h), math.nan, dtype=torch.bfloat16, device=gpu)
    K.moe_experts(x, ids, weights, *w, out=out)
    assert not bool(out.any())
    keep = torch.randn((t, h), device=gpu)
    out = keep.clone()
    K.moe_experts(x, ids, weights, *w, out=out, accumulate=True)
    assert torch.equal(out, keep)


@pytest.mark.parametrize("t,e,i", [(4, 5, 128), (60, 16, 128), (300, 8, 128), (2048, 16, 1024)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_experts_overflow_stays_in_its_token(gpu, t, e, i, dtype):
    """Hidden values that overflow are NaN in e4m3; infinite weights and terms stay infinite or NaN; other tokens keep theirs."""
    announce(f"moe_experts: overflow in the hidden values and an infinite weight, {t} tokens {dtype}")
    k, h = 2, 256
    x, ids, weights, *w = expert_inputs(t, e, k, h, i, dtype, 33 + t)
    rest = torch.tensor([r for r in range(t) if r not in (1, 2)])
    want, mag = experts64(x[rest], ids[rest], weights[rest], *w)
    x[1] *= 1e25
    weights[2, 0] = math.inf
    ids[1:3, 0] = 1  # (one expert that is there)
    out = K.moe_experts(*device((x, ids, weights, *w), gpu)).cpu()
    assert bool(torch.isnan(out[1]).all()) and not bool(torch.isfinite(out[2]).any())
    check_experts(out[rest], want, mag, i, dtype)


@pytest.mark.parametrize("t", [4, 100])
def test_experts_nan_and_infinity_stay_in_their_token(gpu, t):
    announce("moe_experts: NaN and infinite activations")
    e, k, h, i = 5, 2, 256, 128
    x, ids, weights, *w = expert_inputs(t, e, k, h, i, torch.float16, 21)
    x[1, 7], x[3, 200] = math.nan, math.inf
    out = K.moe_experts(*device((x, ids, weights, *w), gpu)).cpu()
    bad = torch.isnan(out)
    assert bool(bad[1].all()) and bool(bad[3].all())
    rest = torch.tensor([r for r in range(t) if r not in (1, 3)])
    assert not bool(bad[rest].any())
    want, mag = experts64(x[rest], ids[rest], weights[rest], *w)
    check_experts(out[rest], want, mag, i, torch.float16)


def test_experts_same_inputs_same_bits(gpu):
    """Which place a pair gets in its expert's tiles is left to the order of the counting: the results are not."""
    announce("moe_experts: repeated calls")
    for t, e, k, i in ((8, 16, 4, 256), (900, 6, 2, 256), (3000, 6, 2, 256), (3000, 12, 2, 1408), (9000, 6, 4, 256)):
        a = device(expert_inputs(t, e, k, 256, i, torch.bfloat16, t), gpu)
        first = K.moe_experts(*a)
        for _ in range(4):
            assert torch.equal(K.moe_experts(*a), first)


def test_two_streams_at_once(gpu):
    """Calls that overlap on two streams, each with its own workspace, give what they give alone."""
    announce("moe_experts and moe_route: two streams")
    a = [device(expert_inputs(t, 12, 3, 512, 256, torch.float16, t), gpu) for t in (300, 257)]
    logits = [torch.randn((5000, 200), generator=gen(s)).to(gpu) for s in (1, 2)]
    alone = [K.moe_experts(*v) for v in a], [K.moe_route(v, 6) for v in logits]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [], []
    for _ in range(5):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[0].append((j, K.moe_experts(*a[j])))
                got[1].append((j, K.moe_route(logits[j], 6)))
    torch.cuda.synchronize()
    for j, y in got[0]:
        assert torch.equal(y, alone[0][j])
    for j, (w, i) in got[1]:
        assert torch.equal(w, alone[1][j][0]) and torch.equal(i, alone[1][j][1])


@pytest.mark.parametrize("t", [1, 60])
def test_a_run_of_all_four_recorded_twice(gpu, t):
    """Route, experts, quantise and project, recorded as two HIP graphs and replayed between eager calls."""
    announce(f"operators in a row, {t} tokens, two graphs")
    e, k, h, i = 10, 3, 512, 256
    w13, s13, w2, s2 = device((*e4m3_weight(1, e, 2 * i, h), *e4m3_weight(2, e, h, i)), gpu)
    wp, sp = device(e4m3_weight(3, 272, h), gpu)

    def block(x, logits):
        weights, ids = K.moe_route(logits, k)
        y = K.moe_experts(x, ids, weights, w13, s13, w2, s2)
        return K.linear_fp8_x8(*K.quant_fp8(y), wp, sp, out_dtype=torch.float32)

    def inputs(seed):
        g = gen(seed)
        return torch.randn((t, h), generator=g).half().to(gpu), torch.randn((t, e), generator=g).to(gpu)

    x, logits = inputs(0)
    block(x, logits)  # every kernel is loaded before the first recording
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(x, logits)
        graphs.append((graph, out))
    for seed in (1, 2, 3):
        fresh = inputs(seed)
        want = block(*fresh)
        for graph, out in graphs:
            x.copy_(fresh[0])
            logits.copy_(fresh[1])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            block(*inputs(seed + 10))  # the program's own calls between the replays


def test_wide_rows_past_32_bit_offsets(gpu):
    """Rows of a buffer of more than 2^32 bytes: offsets in 64 bits."""
    announce("quant_fp8, linear_fp8_x8, moe_experts and moe_route: rows 16 MiB apart")
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    t, h = 300, 256
    x = torch.randn((t, h), generator=gen(4)).half().to(gpu)
    far = torch.empty((t, 1 << 23), dtype=torch.float16, device=gpu)
    far[:, :h] = x
    q, s = K.quant_fp8(x)
    qf, sf = K.quant_fp8(far[:, :h])
    assert torch.equal(q.view(torch.uint8), qf.view(torch.uint8)) and torch.equal(s, sf)
    a = device(expert_inputs(t, 4, 2, h, 128, torch.float16, 8), gpu)
    want = K.moe_experts(x, *a[1:])
    assert torch.equal(K.moe_experts(far[:, :h], *a[1:]), want)
    K.moe_experts(x, *a[1:], out=far[:, h:2 * h])
    assert torch.equal(far[:, h:2 * h], want)
    w, i = K.moe_route(x, 8)
    wf, i_f = K.moe_route(far[:, :h], 8)
    assert torch.equal(w, wf) and torch.equal(i, i_f)
    wp, sp = device(e4m3_weight(6, 64, h), gpu)
    y = K.linear_fp8_x8(q, s, wp, sp)
    K.linear_fp8_x8(q, s, wp, sp, out=far[:, :64])
    assert torch.equal(far[:, :64], y)
    q8 = far.view(torch.uint8)[:, 2048:2048 + h]
    q8.copy_(q.view(torch.uint8))
    if q8.stride(0) <= 1 << 23:
        assert torch.equal(K.linear_fp8_x8(q8, s, wp, sp), y)
    else:
        with pytest.raises(RuntimeError, match="8 MiB"):
            K.linear_fp8_x8(q8, s, wp, sp)
