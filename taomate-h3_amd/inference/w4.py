"""Linears with 4-bit weights and group scales, the sibling of the W8A8 linears for decode, where a
linear's time is its weights' bytes.  Forward only.  No counterpart in the reference.

* ``W4Linear``                        a linear on packed 4-bit weights, from full weights or a checkpoint's codes
* ``set_module_w4_weight_``           the same on a module that keeps its class: a parallel linear of the
                                      reference, whose forward goes through ``distributed.linear._module_linear``
* ``quantize_h3_block_linears_w4_``   the DiT block linears that a policy selects, in place

Activations stay bf16 or fp16, whatever their number: one token's products and a prefill's run on
the same packed weights (``ops.w4_mm``).  The scales keep their dtype when a model is converted to another:
the codes were made for them.
"""

from __future__ import annotations

from typing import Any

import torch
import torch.nn as nn

from .. import ops
from .buffers import FixedDtypeModule
from .fp8 import _block_candidates, resolve_h3_dynamic_fp8_policy


def quantize_w4_weight(weight: torch.Tensor, *, group: int = 128, zeros: bool = False) -> ops.W4Weight:
    """Packed 4-bit weights of ``weight [n, k]`` (bf16, fp16 or fp32; k a multiple of 16)."""
    return ops.pack_w4(*ops.quantize_w4(weight.detach(), group, zeros=zeros), group=group)


def w4_linear(inputs: torch.Tensor, weight: ops.W4Weight, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``inputs [..., k]`` times the transposed weights: [..., n] in the inputs' dtype."""
    flat = inputs.reshape(-1, int(inputs.shape[-1]))
    if flat.stride(-1) != 1 or flat.data_ptr() % 16 or (
            flat.shape[0] > 1 and (flat.stride(0) % 8 or flat.stride(0) < flat.shape[1])):
        flat = flat.clone(memory_format=torch.contiguous_format)  # contiguous() keeps an unaligned start
    if bias is not None and bias.dtype != inputs.dtype:
        bias = bias.to(inputs.dtype)
    return ops.w4_mm(flat, weight, bias=bias).reshape(*inputs.shape[:-1], weight.n)


class W4Linear(FixedDtypeModule):
    """A linear on packed 4-bit weights (``ops.W4Weight``)."""

    FIXED = ("scales",)

    def __init__(self, weight: ops.W4Weight, bias: torch.Tensor | None = None) -> None:
        super().__init__()
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.register_buffer("bias", bias)
        self.out_features, self.in_features, self.group = weight.n, weight.k, weight.group

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None, *, group: int = 128,
                    zeros: bool = False) -> W4Linear:
        """From full weights [n, k]."""
        return cls(quantize_w4_weight(weight, group=group, zeros=zeros), bias)

    @classmethod
    def from_rows(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, *, group: int = 128) -> W4Linear:
        """From a checkpoint's rows: codes uint8 [n, k / 2] (the low nibble first), scales and zeros [n, groups]."""
        return cls(ops.pack_w4(codes, scales, zeros, group=group), bias)

    @property
    def weight(self) -> ops.W4Weight:
        return ops.W4Weight(self.codes, self.scales, self.zeros, self.out_features, self.in_features, self.group)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return w4_linear(x, self.weight, self.bias)


class _W4Groups(FixedDtypeModule):
    """Scales and zero points beside the codes of a module that is not a W4Linear."""

    FIXED = ("scales",)

    def __init__(self, scales: torch.Tensor, zeros: torch.Tensor | None) -> None:
        super().__init__()
        self.register_buffer("scales", scales)
        self.register_buffer("zeros", zeros)


def set_module_w4_weight_(module: nn.Module, weight: ops.W4Weight) -> None:
    """Gives a linear-like module packed 4-bit weights: ``weight`` becomes their codes, with the scales and
    zero points (a submodule, ``_w4_groups``) and sizes beside it."""
    module.weight = nn.Parameter(weight.codes, requires_grad=False)
    module._w4_groups = _W4Groups(weight.scales, weight.zeros)
    module._w4_sizes = (weight.n, weight.k, weight.group)


def module_w4_weight(module: nn.Module) -> ops.W4Weight | None:
    """The packed weights that ``set_module_w4_weight_`` gave the module, or None."""
    sizes = getattr(module, "_w4_sizes", None)
    return None if sizes is None else ops.W4Weight(module.weight, module._w4_groups.scales, module._w4_groups.zeros, *sizes)


def quantize_h3_block_linears_w4_(transformer: Any, *, policy: str | None = None, group: int = 128,
                                  zeros: bool = False) -> dict[str, Any]:
    """4-bit weights for the block linears that a policy of the FP8 linears selects (None: all four projections
    of every block), in place; biases stay as they are."""
    candidates = _block_candidates(transformer, (".attn.qkv_proj", ".attn.out_proj", ".mlp.fc1", ".mlp.fc2"))
    if not candidates:
        raise RuntimeError("no H3 DiT block linears were selected for 4-bit weights")
    selection = resolve_h3_dynamic_fp8_policy([n for n, _ in candidates], policy=policy)
    wanted = set(selection["quantized_linear_names"])
    names, source_bytes, quantized_bytes = [], 0, 0
    for name, module in candidates:
        if name not in wanted:
            continue
        weight = module.weight.detach()
        if weight.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"{name} expected BF16 or FP16 weight before 4-bit conversion")
        packed = quantize_w4_weight(weight, group=group, zeros=zeros)
        source_bytes += int(weight.numel() * weight.element_size())
        quantized_bytes += sum(int(t.numel() * t.element_size()) for t in packed[:3] if t is not None)
        set_module_w4_weight_(module, packed)
        names.append(name)
    if not names:
        raise RuntimeError("4-bit weight policy selected no block linears")
    return {"format": "int4_group_scales", "group": group, "zero_points": bool(zeros), "activations": "unquantized",
            "policy": policy or "all_main_blocks_v1", "linear_count": len(names), "quantized_linear_names": names,
            "bf16_protected_linear_names": selection["bf16_protected_linear_names"],
            "source_weight_bytes": source_bytes, "quantized_weight_bytes": quantized_bytes}


__all__ = ["W4Linear", "module_w4_weight", "quantize_h3_block_linears_w4_", "quantize_w4_weight",
           "set_module_w4_weight_", "w4_linear"]
