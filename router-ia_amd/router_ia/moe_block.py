"""The mixture-of-experts block between the attention layers, for ``BatchedForward``.

The reference's ``batched_moe_step`` (v2/src/router_ia/qwen36_chat_batch.py:127-178)
norms the residual stream, routes each token (qwen36_router.py:96), fetches the
chosen experts and runs them one by one on the host's orders.  Here a layer is
four launches or five and nothing returns to the host:

    h = fp16(rmsnorm(x))                      ria_rmsnorm
    logits = h [gate | shared gate]^T         one library product
    weights, ids                              ria_moe_route (shared expert in the last slot)
    x += sum of the experts' gated MLPs       ria_moe_experts (both products in e4m3)

The shared expert is the experts' last, one that every token visits with the
weight sigmoid(shared gate).  A ``MoeBlock`` is the ``mlp`` callable of
``BatchedForward.step`` and ``capture``, and takes a prompt's rows as well.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import kernels as K


@dataclass
class MoeLayerWeights:
    """One layer's experts as the kernels read them; ``shared``: the last expert and gate row are the shared ones."""
    norm: torch.Tensor      # [hidden] fp32, (1 + w) RMSNorm (post_attention_layernorm)
    gate: torch.Tensor      # [experts (+ 1), hidden] fp16 router rows
    w13: torch.Tensor       # [experts (+ 1), 2 inter, hidden] e4m3, gate rows first
    s13: torch.Tensor       # fp32 scales per 128x128 block
    w2: torch.Tensor        # [experts (+ 1), hidden, inter] e4m3
    s2: torch.Tensor
    shared: bool

    @classmethod
    def from_checkpoint(cls, ckpt: dict[str, torch.Tensor], num_experts: int,
                        device: torch.device | str | None = None) -> "MoeLayerWeights":
        """From a layer's checkpoint tensors (keys: the suffixes after the layer prefix).

        ``mlp.experts.{e}.{gate,up,down}_proj.weight`` with their
        ``.weight_scale_inv``, ``mlp.gate.weight`` and, where the model has
        one, ``mlp.shared_expert.*`` and ``mlp.shared_expert_gate.weight``.
        """
        shared = "mlp.shared_expert.gate_proj.weight" in ckpt
        prefixes = [f"mlp.experts.{e}." for e in range(num_experts)] + (["mlp.shared_expert."] if shared else [])
        sizes = {tuple(ckpt[p + "gate_proj.weight"].shape) for p in prefixes}
        if len(sizes) != 1:
            raise ValueError(f"the experts' sizes differ (the shared one's among them): {sorted(sizes)}")

        def put(t: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
            return t.to(device=device, dtype=dtype).contiguous()

        def stack(names: list[str], suffix: str, dtype: torch.dtype | None = None) -> torch.Tensor:
            rows = []
            for p in prefixes:
                parts = [ckpt[p + n + suffix] for n in names]
                raw = [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in parts]
                rows.append(torch.cat(raw, 0))
            out = put(torch.stack(rows), dtype)
            return out.view(torch.float8_e4m3fn) if out.dtype == torch.uint8 else out

        gates = [ckpt["mlp.gate.weight"]] + ([ckpt["mlp.shared_expert_gate.weight"]] if shared else [])
        return cls(put(ckpt["post_attention_layernorm.weight"], torch.float32), put(torch.cat(gates, 0), torch.float16),
                   stack(["gate_proj", "up_proj"], ".weight"),
                   stack(["gate_proj", "up_proj"], ".weight_scale_inv", torch.float32),
                   stack(["down_proj"], ".weight"), stack(["down_proj"], ".weight_scale_inv", torch.float32), shared)


class MoeBlock:
    """The blocks of all layers: ``block(model_layer, x)`` adds the layer's experts to x [rows, hidden] fp32 in place."""

    def __init__(self, layers: list[MoeLayerWeights], top_k: int, *, scoring: str = "softmax",
                 renormalize: bool = True, scale: float = 1.0):
        """top_k routed experts a token; scoring, renormalize and scale as ``kernels.moe_route`` takes them."""
        for w in layers:
            if not 1 <= top_k <= w.w13.shape[0] - int(w.shared):
                raise ValueError(f"top_k {top_k} of {w.w13.shape[0] - int(w.shared)} experts")
        self.layers = layers
        self.top_k = int(top_k)
        self.scoring, self.renormalize, self.scale = scoring, bool(renormalize), float(scale)

    def __call__(self, model_layer: int, x: torch.Tensor) -> torch.Tensor:
        # every buffer is the allocator's, per call: calls on several streams and captured graphs share none
        w = self.layers[model_layer]
        if x.dtype != torch.float32 or x.dim() != 2:
            raise ValueError(f"x must be fp32 [rows, hidden], got {x.dtype} {tuple(x.shape)}")
        h = K.rmsnorm(x, w.norm, out=torch.empty(x.shape, dtype=torch.float16, device=x.device))
        logits = torch.nn.functional.linear(h, w.gate)
        weights, ids = K.moe_route(logits, self.top_k, scoring=self.scoring, renormalize=self.renormalize,
                                   scale=self.scale, shared_expert=w.shared)
        return K.moe_experts(h, ids, weights, w.w13, w.s13, w.w2, w.s2, out=x, accumulate=True)
