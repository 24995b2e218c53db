"""Between a block's qkv product and its attention: head norms with rotary positions, and the paged cache
that keys and values are appended to.  No counterpart in the reference, whose fused norm and rotation is a
Triton kernel with rounding points of its own and whose cache keeps whole chunks.

* ``QKNormRotary``   the norms' weights and the angle tables of a model; on packed qkv rows
* ``PagedKVCache``   one layer's pages (16 or 32 bits, or e4m3fn codes with scales)

A step plans its tokens once (``PagedKVCache.plan``) and appends in every layer with the same plan; nothing waits
for the device, and every call can be captured into a graph.
"""

from __future__ import annotations

import torch

from .. import ops
from .buffers import FixedDtypeModule

SCALES = (None, "static", "rows")


class PagedKVCache:
    """Pages [pages, page_size, kv_heads, head_dim] of one layer's keys and values.

    ``scales`` None: rows of ``dtype``.  "static": e4m3fn codes by ``k_scale`` and ``v_scale`` (fp32, [1] or [kv_heads],
    calibrated).  "rows": e4m3fn codes, each row's scale kept beside it."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
                 scales: str | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                 device: torch.device | str = "cuda") -> None:
        if scales not in SCALES:
            raise ValueError(f"PagedKVCache: scales must be one of {SCALES}, got {scales!r}")
        if (scales == "static") != (k_scale is not None) or (scales == "static") != (v_scale is not None):
            raise ValueError("PagedKVCache: k_scale and v_scale go with static scales")
        shape = (pages, page_size, kv_heads, head_dim)
        kind = dtype if scales is None else torch.float8_e4m3fn
        self.k, self.v = (torch.zeros(shape, device=device, dtype=kind) for _ in range(2))
        self.page_size, self.dtype = int(page_size), dtype
        if scales == "rows":
            k_scale, v_scale = (torch.zeros(shape[:3], device=device, dtype=torch.float32) for _ in range(2))
        self.k_scale, self.v_scale = k_scale, v_scale

    def plan(self, table: torch.Tensor, lengths: torch.Tensor, cu_tokens: torch.Tensor, tokens: int) -> ops.AppendPlan:
        """Positions and slots of a step's tokens (``ops.plan_append``), good for every layer with such pages."""
        return ops.plan_append(table, lengths, cu_tokens, tokens, self.page_size)

    def append(self, k: torch.Tensor, v: torch.Tensor, plan: ops.AppendPlan, **rows) -> torch.Tensor | None:
        """``ops.append_kv`` into these pages at the plan's slots; ``rows``: its norms, tables and q (positions are
        the plan's where tables are given)."""
        if rows.get("cos") is not None:
            rows.setdefault("positions", plan.positions)
        return ops.append_kv(k, v, self.k, self.v, plan.slots, k_scale=self.k_scale, v_scale=self.v_scale, **rows)

    def gather(self, pages: torch.Tensor, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [length, kv_heads, head_dim] of a sequence with the page ids ``pages``, in ``dtype``."""
        if not 0 <= length <= pages.shape[0] * self.page_size:
            raise ValueError(f"PagedKVCache.gather: {pages.shape[0]} pages of {self.page_size} hold no {length} tokens")
        pages = pages[:(length + self.page_size - 1) // self.page_size].long()
        out = []
        for held, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            if scale is None:
                rows = held[pages]
            else:
                rows = held.view(torch.uint8)[pages].view(held.dtype).float()
                rows = (rows * (scale[pages] if scale.ndim == 3 else scale).unsqueeze(-1)).to(self.dtype)
            out.append(rows.flatten(0, 1)[:length])
        return out[0], out[1]


class QKNormRotary(FixedDtypeModule):
    """RMS norms of the query and key heads and rotary positions, on packed qkv rows [tokens, (q_heads +
    2 * kv_heads) * head_dim].  Weights [head_dim] or [heads, head_dim]; None leaves out that norm.  The angle tables
    stay fp32 when a model is converted to another dtype."""

    FIXED = ("cos", "sin")

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, *, positions: int, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, rot_dim: int | None = None,
                 interleaved: bool = False, device: torch.device | str = "cuda", **frequencies) -> None:
        """``positions``: rows of the angle tables; ``frequencies``: base and scaling of ``ops.rotary_frequencies``."""
        super().__init__()
        self.q_heads, self.kv_heads, self.head_dim = int(q_heads), int(kv_heads), int(head_dim)
        self.eps, self.interleaved = float(eps), bool(interleaved)
        self.register_buffer("q_weight", q_weight)
        self.register_buffer("k_weight", k_weight)
        turns, magnitude = ops.rotary_frequencies(head_dim if rot_dim is None else rot_dim, device=device, **frequencies)
        cos, sin = ops.rotary_tables(torch.arange(positions, device=device), turns, magnitude)
        self.register_buffer("cos", cos, persistent=False)
        self.register_buffer("sin", sin, persistent=False)

    def split(self, qkv: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Views [tokens, heads, head_dim] of q, k and v."""
        rows = qkv.unflatten(-1, (self.q_heads + 2 * self.kv_heads, self.head_dim))
        q, k, v = rows.split((self.q_heads, self.kv_heads, self.kv_heads), dim=-2)
        return q, k, v

    def forward(self, qkv: torch.Tensor, positions: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """q and k normed and rotated (new tensors), v as it lies in the packed rows."""
        q, k, v = self.split(qkv)
        q, k = ops.qk_norm_rotary(q, k, self.q_weight, self.k_weight, self.cos, self.sin, positions, eps=self.eps,
                                  interleaved=self.interleaved)
        return q, k, v

    def append(self, qkv: torch.Tensor, cache: PagedKVCache, plan: ops.AppendPlan,
               q_out: torch.Tensor | None = None) -> torch.Tensor:
        """q normed and rotated; k, normed and rotated, and v into the cache, in one launch."""
        q, k, v = self.split(qkv)
        return cache.append(k, v, plan, k_weight=self.k_weight, eps=self.eps, cos=self.cos, sin=self.sin,
                            interleaved=self.interleaved, q=q, q_weight=self.q_weight, q_out=q_out)


__all__ = ["PagedKVCache", "QKNormRotary"]
