"""Routed-expert FFN on the W8A8 formats: the mixture-of-experts sibling of the dense
quantized FFN (fc1 -> SwiGLU -> fc2).  No counterpart in the reference, whose blocks
are dense.

* ``quantize_expert_weights``  per-output-channel codes of every expert's matrix, tiled
                               where the shape allows
* ``QuantizedExperts``         the experts one GPU holds; forward on routed tokens
* ``QuantizedMoE``             the layer with its router

Expert parallelism: a rank holds the experts [first_expert, first_expert + E) and
returns the part of the sum that falls on them; the parts of all ranks add up to the
layer's output (an all-reduce, or the reduce-scatter that follows anyway).
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


def quantize_expert_weights(weights: torch.Tensor, fmt: int) -> tuple[torch.Tensor, torch.Tensor, bool]:
    """Codes [E, n, k], fp32 scales [E, n] and whether the codes are tiled, of bf16
    expert matrices [E, n, k]: the per-output-channel weight quantizer of the dense
    linears, expert by expert.  Tiled when n % 16 == 0 and k % 128 == 0."""
    if weights.ndim != 3 or weights.dtype != torch.bfloat16:
        raise TypeError(f"quantize_expert_weights: expected bf16 [experts, n, k], got {weights.dtype} "
                        f"{tuple(weights.shape)}")
    experts, n, k = (int(v) for v in weights.shape)
    if experts < 1 or n % 16 or k % 16:
        raise ValueError(f"quantize_expert_weights: n={n} and k={k} must be multiples of 16")
    tiled = ops.can_tile(n, k)
    codes = torch.empty((experts, n, k), device=weights.device, dtype=ops.code_dtype(fmt))
    scales = torch.empty((experts, n), device=weights.device, dtype=torch.float32)
    for e in range(experts):
        quantize = ops.quant_rows_tiled if tiled else ops.quant_rows
        quantize(weights[e].contiguous(), fmt, ops.ROUND_DIV, codes=codes[e], scales=scales[e].view(n, 1))
    if tiled:
        ops.mark_tiled(codes)
    return codes, scales, tiled


class QuantizedExperts(nn.Module):
    """The experts [first_expert, first_expert + E) of a layer: ``w13 [E, 2 f, d]``
    (rows [gate | up]) and ``w2 [E, d, f]`` as e4m3fn or int8 codes with per-channel scales."""

    def __init__(self, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor, *,
                 w13_tiled: bool, w2_tiled: bool, first_expert: int = 0) -> None:
        super().__init__()
        if w13.ndim != 3 or tuple(w2.shape) != (w13.shape[0], w13.shape[2], w13.shape[1] // 2):
            raise ValueError(f"expert weights must be [E, 2 f, d] and [E, d, f], got {tuple(w13.shape)} and "
                             f"{tuple(w2.shape)}")
        self.register_buffer("w13", w13)
        self.register_buffer("w13_scale", w13_scale)
        self.register_buffer("w2", w2)
        self.register_buffer("w2_scale", w2_scale)
        self.w13_tiled, self.w2_tiled, self.first_expert = bool(w13_tiled), bool(w2_tiled), int(first_expert)

    @classmethod
    def from_weights(cls, w13: torch.Tensor, w2: torch.Tensor, fmt: int, *, first_expert: int = 0) -> QuantizedExperts:
        """From bf16 weights [E, 2 f, d] (rows [gate | up]) and [E, d, f]."""
        q13, s13, t13 = quantize_expert_weights(w13, fmt)
        q2, s2, t2 = quantize_expert_weights(w2, fmt)
        return cls(q13, s13, q2, s2, w13_tiled=t13, w2_tiled=t2, first_expert=first_expert)

    def forward(self, x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """bf16 ``x [..., d]``, routed ids and weights [tokens, top_k]; the sum over the experts held here."""
        flat = x.reshape(-1, x.shape[-1])
        return ops.expert_ffn(flat, experts, weights, self.w13, self.w13_scale, self.w2, self.w2_scale,
                              first_expert=self.first_expert, w13_tiled=self.w13_tiled,
                              w2_tiled=self.w2_tiled).reshape(x.shape)


class QuantizedMoE(nn.Module):
    """A routed-expert layer: router (a plain linear, in its weight's dtype), top-k and experts."""

    def __init__(self, router: torch.Tensor, experts: QuantizedExperts, *, top_k: int, scoring: str = "softmax",
                 renormalize: bool = True, scale: float = 1.0) -> None:
        super().__init__()
        self.router = nn.Parameter(router, requires_grad=False)
        self.experts = experts
        self.top_k, self.scoring, self.renormalize, self.scale = int(top_k), scoring, bool(renormalize), float(scale)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        flat = x.reshape(-1, x.shape[-1])
        logits = F.linear(flat.to(self.router.dtype), self.router)
        ids, weights = ops.route_experts(logits, self.top_k, scoring=self.scoring, renormalize=self.renormalize,
                                         scale=self.scale)
        return self.experts(flat, ids, weights).reshape(x.shape)


__all__ = ["QuantizedExperts", "QuantizedMoE", "quantize_expert_weights"]
