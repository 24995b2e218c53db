"""Plain CPU restatements of the routed-expert operators, in 64 bits where the
definition is arithmetic, with the error bounds the GPU results are held to."""

from __future__ import annotations

import numpy as np
import torch

from _util import bits16

HALF_BF16 = 2.0 ** -8   # half a step of bf16, relative: finfo(bf16).eps / 2
U32 = 2.0 ** -24        # half a step of binary32, relative


def route(logits: torch.Tensor, k: int, scoring: str, renorm: bool, scale: float = 1.0):
    """(ids int32, weights float64): a loop over the largest logit left, lowest index first."""
    l = logits.double().numpy().copy()
    l[np.isnan(l)] = -np.inf
    tokens, experts = l.shape
    ids = np.full((tokens, k), -1, np.int32)
    weights = np.zeros((tokens, k))
    for t in range(tokens):
        left = l[t].copy()
        values = []
        for j in range(k):
            e = int(np.argmax(left))  # the first of the largest
            if left[e] == -np.inf:
                break
            ids[t, j] = e
            values.append(left[e])
            left[e] = -np.inf
        if not values:
            continue
        v = np.array(values)
        if scoring == "sigmoid":
            with np.errstate(over="ignore"):
                w = 1.0 / (1.0 + np.exp(-v))
            whole = w.sum() if renorm else 1.0
        else:
            e_of = lambda a: np.where(a == v[0], 1.0, np.exp(np.where(a == v[0], 0.0, a) - np.where(a == v[0], 0.0, v[0])))  # noqa: E731
            w = e_of(v)
            whole = w.sum() if renorm else e_of(l[t][l[t] > -np.inf]).sum()
        weights[t, :len(v)] = w / whole * scale
    return ids, weights


def plan(ids: np.ndarray, experts: int, first: int = 0):
    flat = ids.reshape(-1).astype(np.int64)
    here = [p for p in range(flat.size) if flat[p] >= 0 and first <= flat[p] < first + experts]
    here.sort(key=lambda p: (flat[p], p))
    order = np.full(flat.size, -1, np.int32)
    order[:len(here)] = here
    slots = np.full(flat.size, -1, np.int32)
    for row, p in enumerate(here):
        slots[p] = row
    offsets = np.array([sum(1 for p in here if flat[p] < first + e) for e in range(experts + 1)], np.int32)
    return order, offsets, slots.reshape(ids.shape)


def products(O, fmt: str, qa: np.ndarray, qb: np.ndarray):
    """(sum, bound) of code rows [m, k] x [n, k]: the exact sums.  int8 keeps them (sums
    above 2^24 round once when they become binary32).  e4m3 products run through the FP8
    instruction (its model's distance from the exact sum and the bound on the model's own
    rounding) or as bf16 (exact products, k binary32 additions in some order: at most k
    U32 of the sum of the magnitudes): the larger of the two."""
    if fmt == "int8":
        s = qa.view(np.int8).astype(np.float64) @ qb.view(np.int8).astype(np.float64).T
        return s, np.abs(s) * U32
    a, b = O.e4m3_to_f32(qa).astype(np.float64), O.e4m3_to_f32(qb).astype(np.float64)
    s = a @ b.T  # products of 4-bit significands: binary64 keeps the sums to 2^-53
    model, rest = O.gemm_e4m3_mfma(qa, qb)
    return s, np.maximum(np.abs(s - model) + rest, qa.shape[1] * U32 * (np.abs(a) @ np.abs(b).T))


def scaled(O, fmt, qa, sa, qb, sb):
    """(y, bound) of sa * (sb * products): two binary32 multiplies."""
    s, b = products(O, fmt, qa, qb)
    scale = sa.astype(np.float64)[:, None] * sb.astype(np.float64)[None, :]
    y = s * scale
    return y, b * scale + 2.5 * U32 * np.abs(y)


def swiglu(y: np.ndarray, bound: np.ndarray):
    """(h, bound) of silu(gate) * up from [gate | up] with its bound.

    silu'(g) = s (1 + g (1 - s)) lies in [-0.1, 1.1]; its own evaluation: exp(-g) by
    exp2 of a rounded product (relative error |g| (U32 of the product + U32 of the
    constant) + 2 U32 of exp2), reaching silu with at most that factor, then a sum (U32), a
    reciprocal to one unit in the last place (2 U32) and two products (2 U32): (2 |g| + 7)
    U32, doubled for second-order terms.  The up factor: its own relative bound."""
    half = y.shape[1] // 2
    g, u, bg, bu = y[:, :half], y[:, half:], bound[:, :half], bound[:, half:]
    silu = g / (1.0 + np.exp(-g))
    h = silu * u
    b = 1.1 * bg * np.abs(u) + (np.abs(silu) + 1.1 * bg) * bu + 2 * (2 * np.abs(g) + 7) * U32 * np.abs(h)
    return h, b


def to_bf16(v: np.ndarray) -> np.ndarray:
    """float64 -> the bf16 value nearest (ties to even), as float64 (through binary32 pinned to odd)."""
    f = v.astype(np.float32)
    # round to odd: keeps the second rounding right
    err = v - f.astype(np.float64)
    b = f.view(np.int32).copy()
    away = ((err > 0) == (f > 0)) & (err != 0)
    toward = (err != 0) & ~away
    b = np.where((b & 1) == 0, np.where(away, b | 1, np.where(toward, b - 1, b)), b)
    t = torch.from_numpy(b.astype(np.int32).view(np.float32).copy()).to(torch.bfloat16)
    return t.double().numpy()


def codes_of(x: np.ndarray, fmt: str):
    """(code values float64, scales float32) of bf16 rows, activation form, in binary32 as defined."""
    t = torch.from_numpy(np.ascontiguousarray(x)).float()
    amax = t.abs().amax(dim=1, keepdim=True)
    if fmt == "e4m3":
        s = torch.clamp(amax * (1.0 / 448.0), min=1e-12)
        q = torch.clamp(t / s, -448.0, 448.0).to(torch.float8_e4m3fn)
        return q.double().numpy(), s.numpy().ravel()
    limit = torch.full_like(amax, 127.0)  # a tensor: torch divides a number by a tensor through a rounded reciprocal
    inv = torch.where(amax > 0, limit / amax, torch.zeros_like(amax))
    return torch.clamp(torch.round(t * inv), -128, 127).double().numpy(), (amax / limit).numpy().ravel()


def raw_codes(q: np.ndarray, fmt: str) -> np.ndarray:
    t = torch.from_numpy(q)
    return (t.to(torch.int8) if fmt == "int8" else t.float().to(torch.float8_e4m3fn)).view(torch.uint8).numpy()


def quantize_weights(w: torch.Tensor, O, fmt: str):
    """uint8 codes [E, n, k] and scales [E, n] of bf16 weights, by the oracle."""
    q, s = zip(*(O.quant_rows(bits16(w[e]), "e4m3" if fmt == "e4m3" else "int8") for e in range(w.shape[0])))
    return np.stack([v.view(np.uint8) for v in q]), np.stack([v.ravel() for v in s])


def ffn(O, fmt, x: torch.Tensor, ids: np.ndarray, weights: np.ndarray, q13, s13, q2, s2, first: int = 0):
    """(out float64, bound) of the layer.

    The bound: one bf16 rounding of the result; the binary32 sums and scales; and the
    codes of h that the error of h (through its bf16 rounding) can move to a neighbour:
    every code between those of h - b and h + b is allowed, with the row's scale between
    those of the extremes."""
    tokens, d = x.shape
    experts = q13.shape[0]
    q, s = O.quant_rows(bits16(x), fmt, "rcp" if fmt == "int8" else "div")
    q = q.view(np.uint8)
    out = np.zeros((tokens, d))
    bound = np.zeros((tokens, d))
    decode = (lambda c: c.view(np.int8).astype(np.float64)) if fmt == "int8" else (
        lambda c: O.e4m3_to_f32(c).astype(np.float64))
    for e in range(experts):
        t, j = np.nonzero(ids == first + e)
        if t.size == 0:
            continue
        y, b = scaled(O, fmt, q[t], s.ravel()[t], q13[e], s13[e])
        h, bh = swiglu(y, b)
        mid, lo, hi = to_bf16(h), to_bf16(h - bh), to_bf16(h + bh)
        qh, sh = codes_of(mid, fmt)
        value = qh * sh[:, None]
        # what h can become: the extremes quantized with the extreme scales
        span = np.zeros_like(value)
        top_lo, top_hi = np.minimum(np.abs(lo), np.abs(hi)).max(1), np.maximum(np.abs(lo), np.abs(hi)).max(1)
        for v in (lo, hi):
            for top in (top_lo, top_hi):
                w = np.concatenate((np.clip(v, -top[:, None], top[:, None]), top[:, None]), 1)
                cq, cs = codes_of(w, fmt)
                span = np.maximum(span, np.abs(cq[:, :-1] * cs[:, None] - value))
        p, pb = products(O, fmt, raw_codes(qh, fmt), q2[e])
        scale = sh.astype(np.float64)[:, None] * s2[e].astype(np.float64)[None, :]
        w2 = np.abs(decode(q2[e]) * s2[e].astype(np.float64)[:, None])
        # the instruction's truncation depends on the codes it is given: twice its step where they may differ
        loose = 2.0 ** -9 * (span @ w2.T) if fmt == "e4m3" else 0.0
        c = weights[t, j].astype(np.float64)[:, None]
        yd = p * scale
        np.add.at(out, t, c * yd)
        np.add.at(bound, t, np.abs(c) * (pb * scale + span @ w2.T + loose + (3 + ids.shape[1]) * U32 * np.abs(yd)))
    return out, bound + HALF_BF16 * (np.abs(out) + bound) + 2.0 ** -133
