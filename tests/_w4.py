"""Plain 64-bit form of the products with 4-bit weights, the quantizer, the packed layout and the bound of results
that are summed in binary32 and rounded once."""

from __future__ import annotations

import numpy as np
import torch


def unpack_rows(codes: torch.Tensor) -> torch.Tensor:
    """uint8 [n, k / 2] -> integers [n, k], the low nibble first."""
    c = codes.cpu()
    return torch.stack((c & 15, c >> 4), dim=2).flatten(1)


def dequantized(codes, scales, zeros, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights s (u - z) and scales by column, float64 [n, k]."""
    u = unpack_rows(codes).double()
    by = torch.arange(u.shape[1]) // group
    s = scales.cpu().double()[:, by]
    z = 8.0 if zeros is None else zeros.cpu().double()[:, by]
    return s * (u - z), s


def product(x, codes, scales, zeros, group: int, bias=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(value, bound of its binary32 error), float64 [m, n].

    Above 16 rows the weights s (u - z) are rounded once to x's type; binary32 holds them before that (11 + 5
    bits), so the rounding is a definite one.  A matrix instruction takes 16 or 32 products: its own sum has at most
    32 roundings (of 2^-23: it may cut off) of its terms, and one follows onto a sum of at most sum |x w|, k / 16
    times; the parts of a split k and a workgroup's waves add at most 16 more: (k / 16 + 48) 2^-23 sum |x w|.

    Up to 16 rows a group (at most 128 columns of it at a time) is summed as x u, at most 15 |x| a term, with 32 + 4
    roundings as above, and z times the sum of x, as large, with as many, is taken off in one; the scale and the
    sum over the groups are one more rounding each of at most 30 |s x|: (56 + k / min(group, 128)) 2^-23 * 30
    sum |s x|."""
    w, s = dequantized(codes, scales, zeros, group)
    a = x.cpu().double()
    if len(x) > 16:
        w = w.to(x.dtype).double()
        bound = (a.shape[1] / 16 + 48) * 2.0 ** -23 * (a.abs() @ w.abs().T)
    else:
        bound = (56 + a.shape[1] / min(group, 128)) * 2.0 ** -23 * 30.0 * (a.abs() @ s.abs().T)
    y = a @ w.T
    if bias is not None:
        y = y + bias.cpu().double()
        bound = bound + 2.0 ** -23 * y.abs()
    return y, bound


def assert_product(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    info = torch.finfo(got.dtype)
    g = got.detach().cpu().double()
    bound = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps / 2
    bad = ~((g - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}: "
                           f"{g[bad][0].item()!r} for {want[bad][0].item()!r} +- {bound[bad][0].item():.3g}")


def quantize(w: torch.Tensor, group: int, zeros: bool):
    """The quantizer in binary32, operation by operation (numpy: IEEE, no reciprocal of a constant divisor)."""
    kind = torch.float16 if w.dtype == torch.float16 else torch.bfloat16
    a = w.float().cpu().numpy()
    n, k = a.shape
    groups = (k + group - 1) // group
    codes = np.zeros((n, k), np.uint8)
    scales = torch.zeros(n, groups, dtype=kind)
    points = np.full((n, groups), 8, np.uint8)
    for g in range(groups):
        part = a[:, g * group:(g + 1) * group]
        low, high = np.minimum(part.min(1), np.float32(0)), np.maximum(part.max(1), np.float32(0))
        reach = (high - low) / np.float32(15) if zeros else np.maximum(high, -low) / np.float32(7)
        scales[:, g] = torch.from_numpy(reach).to(kind)
        s = scales[:, g].float().numpy()
        live = s > 0
        safe = np.where(live, s, np.float32(1))
        z = np.where(live, np.clip(np.rint(-low / safe), 0, 15), 0) if zeros else np.full(n, 8.0)
        q = np.where(live[:, None], np.rint(part / safe[:, None]), 0)
        codes[:, g * group:(g + 1) * group] = np.clip(q + z[:, None], 0, 15).astype(np.uint8)
        points[:, g] = z.astype(np.uint8)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return torch.from_numpy(packed), scales, torch.from_numpy(points) if zeros else None


def packed_codes(codes: torch.Tensor) -> torch.Tensor:
    """The layout, word by word: word s of lane L of block (r, b) holds the codes 128 b + 32 s + 8 (L / 16) .. + 7 of
    row 16 r + L % 16, k0 .. k3 in the low nibbles of its bytes and k4 .. k7 in the high ones."""
    u = unpack_rows(codes).numpy().astype(np.uint64)
    n, k = u.shape
    rows, cols = -(-n // 16), -(-k // 128)
    full = np.zeros((rows * 16, cols * 128), np.uint64)
    full[:n, :k] = u
    out = np.zeros((rows, cols, 64, 4), np.uint32)
    for lane in range(64):
        for s in range(4):
            base = 32 * s + 8 * (lane // 16)
            e = [full[lane % 16::16, base + i::128] for i in range(8)]
            out[:, :, lane, s] = sum(v << np.uint64(8 * (i & 3) + (i & 4)) for i, v in enumerate(e))
    return torch.from_numpy(out.view(np.uint8).reshape(rows, cols, 1024))


def packed_groups(rows: torch.Tensor) -> torch.Tensor:
    """Scales or zero points [n, groups] -> [ceil(n / 16), ceil(groups / 4), 16, 4], zeros past the ends."""
    n, groups = rows.shape
    full = torch.zeros(-(-n // 16) * 16, -(-groups // 4) * 4, dtype=rows.dtype)
    full[:n, :groups] = rows
    return full.view(-(-n // 16), 16, -1, 4).transpose(1, 2).contiguous()
