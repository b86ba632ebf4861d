"""Refusals of the routing, quantisation, FP8 x FP8 and expert entry points: host checks alone, nothing is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch

from router_ia import _native as nat
from router_ia import kernels as K

A = 0x10000  # an aligned address that no check dereferences


def refused(rc: int, text: str, code: int = 1) -> None:
    message = nat.load().ria_last_error().decode()
    assert rc == code and text in message, (rc, message)


def quant(rows=4, cols=256, x=A, dtype=0, stride=256, out=A, scale=A):
    return nat.load().ria_quant_fp8(rows, cols, x, dtype, stride, out, scale, None)


def test_quant_refusals() -> None:
    refused(quant(cols=200), "multiple of 128")
    refused(quant(cols=0), "multiple of 128")
    refused(quant(rows=-1), "cols")
    refused(quant(dtype=3), "dtype")
    refused(quant(x=None), "null")
    refused(quant(out=None), "null")
    refused(quant(scale=None), "null")
    refused(quant(x=A + 8), "16-byte")
    refused(quant(stride=255), "row stride")
    refused(quant(stride=260), "multiple of 8")
    refused(quant(out=A + 4), "out must be")
    assert quant(rows=0, x=None) == 0


def linear(m=4, n=32, k=256, x=A, xs=256, s=A, ss=2, w=A, ws=A, y=A, dt=1, ys=32, add=0):
    return nat.load().ria_linear_fp8_x8(m, n, k, x, xs, s, ss, w, ws, y, dt, ys, add, None)


def test_linear_refusals() -> None:
    refused(linear(n=24), "multiple of 16")
    refused(linear(n=0), "multiple of 16")
    refused(linear(m=-1), "N must")
    refused(linear(k=200), "multiple of 128")
    refused(linear(k=32768 + 128), "multiple of 128")
    refused(linear(dt=7), "dtype")
    refused(linear(add=1), "y_add")
    for name in ("x", "s", "w", "ws", "y"):
        refused(linear(**{name: None}), "null")
    refused(linear(x=A + 8), "16-byte")
    refused(linear(xs=240), "row stride")
    refused(linear(xs=264), "multiple of 16")
    refused(linear(ss=1), "x_scale")
    refused(linear(ys=31), "y row stride")
    refused(linear(w=A + 8), "weight")
    assert linear(m=0, x=None) == 0


def route(t=4, e=64, k=8, logits=A, dt=2, ls=64, scoring=0, bias=None, groups=1, top=1, gs=0, renorm=1, scale=1.0,
          shared=0, w=A, wstride=8, ids=A, istride=8):
    return nat.load().ria_moe_route(t, e, k, logits, dt, ls, scoring, bias, groups, top, gs, renorm, scale, shared, w,
                                    wstride, ids, istride, None)


def test_route_refusals() -> None:
    refused(route(e=0), "experts")
    refused(route(e=1025, ls=1025), "experts")
    refused(route(t=-1), "experts")
    refused(route(k=0), "top_k")
    refused(route(k=33), "top_k")
    refused(route(e=4, k=5), "top_k")
    refused(route(groups=8, top=1, k=9), "top_k")  # more than the open groups hold
    refused(route(groups=3), "groups")
    refused(route(groups=0), "groups")
    refused(route(e=65, ls=65, groups=65), "groups")
    refused(route(groups=8, top=9), "top_groups")
    refused(route(groups=8, top=0), "top_groups")
    refused(route(scoring=2), "scoring")
    refused(route(gs=2), "group score")
    refused(route(dt=5), "dtype")
    for name in ("logits", "w", "ids"):
        refused(route(**{name: None}), "null")
    refused(route(ls=63), "row stride")
    refused(route(wstride=7), "row stride")
    refused(route(shared=1), "row stride")
    assert route(t=0, logits=None) == 0


def experts(**kw):
    d = dict(tokens=3, top_k=2, experts=4, hidden=256, inter=128, x=A, x_dtype=1, x_row_stride=256, ids=A,
             ids_row_stride=2, weights=A, weights_row_stride=2, w13=A, w13_scale_inv=A, w2=A, w2_scale_inv=A, out=A,
             out_dtype=1, out_row_stride=256, accumulate=0, workspace=A, workspace_bytes=1 << 30)
    d.update(kw)
    return nat.load().ria_moe_experts(ctypes.byref(nat.MoeExpertsDesc(**d)), None)


def test_experts_refusals() -> None:
    assert nat.load().ria_moe_experts(None, None) == 1
    refused(experts(top_k=0), "sizes")
    refused(experts(experts=0), "sizes")
    refused(experts(experts=1025), "sizes")
    refused(experts(tokens=-1), "sizes")
    refused(experts(hidden=200), "hidden")
    refused(experts(inter=100), "inter")
    refused(experts(tokens=1 << 29, top_k=4), "pairs")
    refused(experts(x_dtype=9), "dtype")
    refused(experts(out_dtype=9), "dtype")
    refused(experts(accumulate=1), "accumulating")
    for name in ("x", "ids", "weights", "w13", "w13_scale_inv", "w2", "w2_scale_inv", "out", "workspace"):
        refused(experts(**{name: None}), "null")
    refused(experts(x=A + 2), "16-byte")
    refused(experts(x_row_stride=255), "row stride")
    refused(experts(x_row_stride=260), "multiple of 8")
    refused(experts(ids_row_stride=1), "row stride")
    refused(experts(weights_row_stride=1), "row stride")
    refused(experts(out_row_stride=128), "row stride")
    refused(experts(w13=A + 8), "weights")
    refused(experts(workspace=A + 16), "256-byte")
    need = K.moe_experts_workspace_bytes(3, 2, 4, 256, 128)
    refused(experts(workspace_bytes=need - 1), "workspace", code=3)
    assert experts(tokens=0, x=None) == 0


def test_workspace_sizes() -> None:
    small, large = (K.moe_experts_workspace_bytes(t, 8, 256, 2048, 512) for t in (1, 4096))
    assert 0 < small < large
    assert K.moe_experts_workspace_bytes(4096, 8, 256, 2048, 512, torch.float32) > large
    with pytest.raises(ValueError, match="sizes refused"):
        K.moe_experts_workspace_bytes(1, 8, 256, 2000, 512)


def test_tensors_off_the_gpu_are_refused() -> None:
    w = torch.zeros((32, 128), dtype=torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.quant_fp8(torch.zeros((2, 128)))
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.linear_fp8_x8(w, torch.ones((32, 1)), w, torch.ones((1, 1)))
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.moe_route(torch.zeros((2, 16)), 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.moe_experts(torch.zeros((2, 128)), torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)),
                      torch.zeros((1, 256, 128), dtype=torch.float8_e4m3fn), torch.ones((1, 2, 1)),
                      torch.zeros((1, 128, 128), dtype=torch.float8_e4m3fn), torch.ones((1, 1, 1)))


def test_block_refusals() -> None:
    from router_ia.moe_block import MoeBlock, MoeLayerWeights

    z = torch.zeros
    w = MoeLayerWeights(z(128), z(5, 128), z(5, 256, 128), z(5, 2, 1), z(5, 128, 128), z(5, 1, 1), True)
    with pytest.raises(ValueError, match="top_k"):
        MoeBlock([w], 5)
    block = MoeBlock([w], 4)
    with pytest.raises(ValueError, match="fp32"):
        block(0, z((2, 128), dtype=torch.float16))
    with pytest.raises(RuntimeError, match="no CPU path"):
        block(0, z((2, 128)))
