"""Plain 64-bit forms of the head norms, the rotation and the paged append, with the tolerances of results
that are computed in binary32 and rounded once.

A value y = a c - b s of normed channels is off by
* half a step of its type where it is stored: eps / 2 of its magnitude (and half of the smallest subnormal),
* binary32 before that: the norm's factor has a sum of d squares (d / 2 V of them in a lane, each one fused
  step, then log2 steps), a product, a sum, the reciprocal root (a unit) and two products; at most 24 + d / 8
  roundings of 2^-24 in all, of which the sum's count half (a root), then two products and a sum: the
  roundings apply to |a c| + |b s|, which cancellation does not shrink.
FP32 = 2^-24 (32 + d / 8) of |a c| + |b s| covers all of it."""

from __future__ import annotations

import numpy as np
import torch


def norm_rotate(x: torch.Tensor, weight=None, cos=None, sin=None, rows=None, *, eps=1e-6, interleaved=False,
                inverse=False):
    """(value, |a c| + |b s|) in float64 of rows x [tokens, heads, d]; cos, sin fp32 tables, rows: int list."""
    y = x.double().cpu().numpy().copy()
    tokens, heads, d = y.shape
    with np.errstate(all="ignore"):
        if weight is not None:
            w = np.broadcast_to(weight.double().cpu().numpy(), (heads, d))
            for t in range(tokens):
                for h in range(heads):
                    y[t, h] = y[t, h] / np.sqrt(np.sum(y[t, h] ** 2) / d + eps) * w[h]
        size = np.abs(y)
        if cos is not None:
            half = cos.shape[1]
            rows = list(range(tokens)) if rows is None else [int(r) for r in rows]
            nan = np.full(half, np.nan)
            ct, st = cos.double().cpu().numpy(), sin.double().cpu().numpy()
            for t, r in enumerate(rows):
                c, s = (ct[r], st[r]) if 0 <= r < len(ct) else (nan, nan)
                s = -s if inverse else s
                first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (
                    slice(0, half), slice(half, 2 * half))
                a, b = y[t, :, first].copy(), y[t, :, second].copy()
                y[t, :, first], y[t, :, second] = a * c - b * s, a * s + b * c
                size[t, :, first] = np.abs(a * c) + np.abs(b * s)
                size[t, :, second] = np.abs(a * s) + np.abs(b * c)
    return torch.from_numpy(y), torch.from_numpy(size)


def fp32_bound(size: torch.Tensor, d: int) -> torch.Tensor:
    return size * ((32 + d / 8) * 2.0 ** -24)


def assert_close(got: torch.Tensor, want: torch.Tensor, size: torch.Tensor, d: int, what: str = "") -> None:
    """got within half a step of its type, and the binary32 bound, of want."""
    info = torch.finfo(got.dtype)
    g = got.detach().cpu().double()
    bound = fp32_bound(size, d)
    bound = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps / 2
    same = (g == want) | (torch.isnan(g) & torch.isnan(want))
    # a value that the type rounds to infinity
    over = want.abs() + bound >= info.max
    bad = ~(same | ((g - want).abs() <= bound) | (over & torch.isinf(g)))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values, first at {bad.nonzero()[0].tolist()}: "
                           f"{g[bad][0].item()!r}, {want[bad][0].item()!r} +- {bound[bad][0].item():.3g}")


def assert_codes(codes: torch.Tensor, scale: torch.Tensor, want: torch.Tensor, size: torch.Tensor, d: int,
                 what: str = "") -> None:
    """e4m3 codes of want / scale, clamped to 448: half a step (2^-4 of the value, 2^-10 in the subnormal
    range) and the binary32 bound with the scale's own two roundings."""
    g = codes.detach().cpu().float().double()
    by = scale.double().cpu()
    q = (want / by).clamp(-448.0, 448.0)
    q = torch.where(torch.isnan(want / by), want / by, q)
    bound = fp32_bound(size, d) / by + q.abs() * 4 * 2.0 ** -24
    bound = bound + torch.maximum((q.abs() + bound) * 2.0 ** -4, torch.tensor(2.0 ** -10))
    ok = ((g - q).abs() <= bound) | (torch.isnan(g) & torch.isnan(q))
    assert ok.all(), f"{what}: {int((~ok).sum())} codes, first {g[~ok][0].item()} for {q[~ok][0].item()}"


def plan(table, lengths, cu, tokens: int, page_size: int):
    """Positions and slots of a step, token by token."""
    table, lengths, cu = (np.asarray(t.cpu()) for t in (table, lengths, cu))
    positions, slots = np.full(tokens, -1, np.int64), np.full(tokens, -1, np.int64)
    for s in range(len(lengths)):
        for t in range(int(cu[s]), min(int(cu[s + 1]), tokens)):
            positions[t] = int(lengths[s]) + t - int(cu[s])
            column = positions[t] // page_size
            if column < table.shape[1] and table[s, column] >= 0:
                slots[t] = int(table[s, column]) * page_size + positions[t] % page_size
    return torch.from_numpy(positions), torch.from_numpy(slots)
