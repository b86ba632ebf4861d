"""GPU parity: the mixture-of-experts block (router_ia.moe_block) alone and as the forward loop's mlp."""

from __future__ import annotations

import pytest
import torch

from conftest import announce
from router_ia import batched_forward as BF
from router_ia import kernels as K
from router_ia import workloads as W
from router_ia.batched_state import BatchedAttentionState
from router_ia.moe_block import MoeBlock, MoeLayerWeights
from test_gpu_moe import expert_tolerance, experts64, route64

pytestmark = pytest.mark.gpu

EXPERTS, TOP_K, INTER = 12, 3, 128


def moe_layers(n, gpu, shared=True):
    return [MoeLayerWeights.from_checkpoint(W.synthetic_moe_layer(900 + m, EXPERTS, INTER, shared=shared), EXPERTS, gpu)
            for m in range(n)]


def test_weights_from_checkpoint(gpu):
    announce("MoeLayerWeights.from_checkpoint: order of the experts and of their rows")
    ckpt = W.synthetic_moe_layer(3, 4, 128, hidden=256)
    w = MoeLayerWeights.from_checkpoint(ckpt, 4, gpu)
    assert w.shared and tuple(w.w13.shape) == (5, 256, 256) and tuple(w.w2.shape) == (5, 256, 128)
    assert tuple(w.s13.shape) == (5, 2, 2) and tuple(w.s2.shape) == (5, 2, 1) and tuple(w.gate.shape) == (5, 256)
    up = ckpt["mlp.experts.2.up_proj.weight"]
    assert torch.equal(w.w13[2, 128:].cpu().view(torch.uint8), up.view(torch.uint8))
    assert torch.equal(w.w2[4].cpu().view(torch.uint8), ckpt["mlp.shared_expert.down_proj.weight"].view(torch.uint8))
    assert torch.equal(w.s13[1].cpu()[0], ckpt["mlp.experts.1.gate_proj.weight_scale_inv"][0])
    ckpt.update({k: v for k, v in W.synthetic_moe_layer(4, 4, 256, hidden=256).items() if "shared_expert." in k})
    with pytest.raises(ValueError, match="sizes differ"):
        MoeLayerWeights.from_checkpoint(ckpt, 4, gpu)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_block_matches_definition(gpu, rows, shared):
    announce(f"MoeBlock: {rows} rows, shared expert {shared}")
    (w,) = moe_layers(1, gpu, shared)
    block = MoeBlock([w], TOP_K)
    x = torch.randn((rows, 2048), generator=torch.Generator().manual_seed(rows))
    got = block(0, x.clone().to(gpu)).cpu().double()
    # from the normed rows and logits on (both checked elsewhere), in 64 bits
    h = K.rmsnorm(x.to(gpu), w.norm, out=torch.empty((rows, 2048), dtype=torch.float16, device=gpu))
    logits = torch.nn.functional.linear(h, w.gate)
    weights, ids = route64(logits.cpu(), TOP_K, shared_expert=shared)
    want, mag = experts64(h.cpu(), ids, weights.float(), w.w13.cpu(), w.s13.cpu(), w.w2.cpu(), w.s2.cpu())
    tol = expert_tolerance(want, mag, INTER, torch.float16, 0.125 * 4 * 2 / INTER ** 0.5) + 2.0 ** -23 * got.abs()
    assert bool(((got - x.double() - want).abs() <= tol).all())


def setup(gpu, lengths):
    st = BatchedAttentionState(len(lengths), 700, num_linear_layers=3, num_full_layers=1, device=gpu,
                               page_shuffle_seed=5)
    st.set_positions(lengths)
    g = torch.Generator(device=gpu)
    g.manual_seed(71)
    st.linear_states.normal_(0.0, 0.02, generator=g)
    st.conv_rings.normal_(0.0, 1.0, generator=g)
    st.kv.k.normal_(0.0, 1.0, generator=g)
    st.kv.v.normal_(0.0, 1.0, generator=g)
    return BF.BatchedForward(st, [BF.layer_weights(W.synthetic_layer(700 + m, m), m, gpu) for m in range(4)])


@pytest.mark.parametrize("rows", [2, 20])
def test_forward_loop_with_the_block(gpu, rows):
    """step(x, mlp=block) is the layers and the blocks in turn, and a recorded step replays to the same bits."""
    announce(f"BatchedForward with MoeBlock, {rows} rows: eager, by hand, recorded")
    lengths = [37 + 11 * r for r in range(rows)]
    block = MoeBlock(moe_layers(4, gpu), TOP_K)
    inputs = [torch.randn((rows, 2048), generator=torch.Generator().manual_seed(s)).to(gpu) for s in range(5)]

    fwd = setup(gpu, lengths)
    eager = [fwd.step(x.clone(), mlp=block).clone() for x in inputs]

    by_hand = setup(gpu, lengths)
    for x, want in zip(inputs, eager):
        x = x.clone()
        for m in range(4):
            x = block(m, by_hand.layer(m, x))
        by_hand.state.advance()
        assert torch.equal(x, want)

    recorded = setup(gpu, lengths)
    assert torch.equal(recorded.step(inputs[0].clone(), mlp=block), eager[0])
    graph = recorded.capture(4, mlp=block)
    for x, want in zip(inputs[1:], eager[1:]):
        graph.x.copy_(x)
        y = graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        block(0, x.clone())  # the program's own calls between the replays
