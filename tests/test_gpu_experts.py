"""Routed-expert operators on the GPU against the CPU restatements of tests/_experts.py."""

from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

import _experts as R
from _util import activations, bits16, to_tiled

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def experts_module():
    return importlib.import_module("taomate_h3_amd.inference.experts")


# ------------------------------------------------------------------ routing

def _logits(t, e, seed, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    l = torch.randn(t, e, generator=gen) * 2
    l[torch.rand(t, e, generator=gen) < 0.1] = -torch.inf
    if t > 3:
        l[1] = -torch.inf
        l[2, : e - 1] = -torch.inf
        l[3, 0] = torch.nan
    return l.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 64, 8), (5, 7, 7), (37, 128, 6), (70, 256, 16), (33, 257, 3),
                                   (9, 1024, 64), (3, 40, 17)])
@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                            ("sigmoid", False)])
def test_route(ops, device, dtype, t, e, k, scoring, renorm):
    logits = _logits(t, e, 7 * t + e, dtype)
    ids, weights = ops.route_experts(logits.to(device), k, scoring=scoring, renormalize=renorm, scale=1.5)
    want_ids, want = R.route(logits, k, scoring, renorm, 1.5)
    assert (ids.cpu().numpy() == want_ids).all()
    # exp: 2 half-steps and the difference's rounding times |l| <= 20; at most e terms summed in
    # binary32, the quotient and the scale
    bound = want * (2 + 40 + e + 4) * R.U32
    assert (np.abs(weights.cpu().numpy() - want) <= bound).all()


def test_route_special_values(ops, device):
    inf, nan = torch.inf, torch.nan
    logits = torch.tensor([[inf, 1.0, inf, 0.0], [nan, nan, nan, nan], [-0.0, 0.0, -0.0, 0.0], [-inf, 3e38, -3e38, nan],
                           [1.0, 1.0, 1.0, 1.0], [-1e-45, 1e-45, 0.0, -0.0]])
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            ids, weights = ops.route_experts(logits.to(device), 3, scoring=scoring, renormalize=renorm)
            want_ids, want = R.route(logits, 3, scoring, renorm)
            assert ids.cpu().tolist() == want_ids.tolist()
            np.testing.assert_allclose(weights.cpu().numpy(), want, rtol=64 * R.U32, atol=1e-38)


def test_route_strided_rows_and_no_tokens(ops, device):
    wide = _logits(20, 50, 3).to(device)
    ids, weights = ops.route_experts(wide[:, 5:37], 4)
    ids2, weights2 = ops.route_experts(wide[:, 5:37].contiguous(), 4)
    assert torch.equal(ids, ids2) and torch.equal(weights, weights2)
    ids, weights = ops.route_experts(wide[:0], 4)
    assert ids.shape == (0, 4) and weights.shape == (0, 4)


@pytest.mark.parametrize("t,k,total,e,first", [(1, 1, 1, 1, 0), (1, 8, 64, 64, 0), (5, 3, 8, 4, 2), (257, 6, 128, 128, 0),
                                               (1000, 8, 64, 16, 48), (4099, 4, 256, 64, 64), (63, 64, 1000, 1000, 0),
                                               (2048, 1, 8, 8, 0), (2049, 1, 1024, 1024, 0), (70001, 8, 128, 128, 0),
                                               (9000, 63, 24, 20, 3)])
def test_plan(ops, device, t, k, total, e, first):
    gen = torch.Generator().manual_seed(t + e)
    ids = torch.randint(-1, total, (t, k), generator=gen, dtype=torch.int32)
    ids[torch.rand(t, k, generator=gen) < 0.01] = 2 ** 31 - 1
    ids[torch.rand(t, k, generator=gen) < 0.01] = -2 ** 31
    plan = ops.plan_experts(ids.to(device), e, first_expert=first)
    order, offsets, slots = R.plan(ids.numpy(), e, first)
    assert (plan.offsets.cpu().numpy() == offsets).all()
    assert (plan.order.cpu().numpy() == order).all()
    assert (plan.slots.cpu().numpy() == slots).all()


def test_plan_of_nothing_and_of_one_expert(ops, device):
    none = ops.plan_experts(torch.full((9, 2), -1, dtype=torch.int32, device=device), 5)
    assert none.offsets.tolist() == [0] * 6 and none.order.tolist() == [-1] * 18 and (none.slots == -1).all()
    empty = ops.plan_experts(torch.empty((0, 2), dtype=torch.int32, device=device), 5)
    assert empty.offsets.tolist() == [0] * 6
    same = ops.plan_experts(torch.full((300, 2), 3, dtype=torch.int32, device=device), 5)  # the same expert twice a token
    assert same.offsets.tolist() == [0, 0, 0, 0, 600, 600]
    assert torch.equal(same.order.cpu(), torch.arange(600, dtype=torch.int32))


def test_plan_unaligned_ids(ops, device):
    ids = torch.randint(0, 6, (1 + 3 * 101,), dtype=torch.int32, device=device)[1:].view(101, 3)
    plan = ops.plan_experts(ids, 6)
    order, offsets, slots = R.plan(ids.cpu().numpy(), 6)
    assert (plan.order.cpu().numpy() == order).all() and (plan.slots.cpu().numpy() == slots).all()


# --------------------------------------------------------- grouped products

def _stack(e, n, k, fmt, seed, oracle):
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn(e, n, k, generator=gen) * k ** -0.5).to(torch.bfloat16)
    return R.quantize_weights(w, oracle, fmt)


def _device_codes(codes: np.ndarray, fmt, device):
    t = torch.from_numpy(np.ascontiguousarray(codes)).to(device)
    return t.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)


def _tile_stack(codes: np.ndarray) -> np.ndarray:
    return np.stack([to_tiled(c) for c in codes])


# experts' row counts: empty ones, one row, tile borders, a long one
_COUNTS = [[0, 1, 0, 5, 16], [17, 0, 33, 3], [0, 0, 7], [65, 0, 31, 32], [300, 1, 0, 255], [1], [513, 128, 400, 700]]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("counts", _COUNTS, ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("n,k,tiled", [(64, 128, True), (32, 256, True), (96, 640, True), (32, 16, False), (160, 272, False),
                                       (288, 384, False)])
@pytest.mark.parametrize("swiglu", [False, True])
def test_grouped(ops, device, oracle, fmt, counts, n, k, tiled, swiglu):
    e, rows = len(counts), sum(counts)
    spare = 5  # rows of the call past the last group
    x = activations(rows + spare, k, seed=rows + n, outlier_channels=2)
    qa, sa = oracle.quant_rows(bits16(x), fmt, "rcp" if fmt == "int8" else "div")
    qa, sa = qa.view(np.uint8), sa.ravel()
    qw, sw = _stack(e, n, k, fmt, n + k, oracle)
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    cols = n // 2 if swiglu else n
    out = torch.full((rows + spare, cols), 7.0, device=device, dtype=torch.bfloat16)
    got = ops.grouped_scaled_mm(_device_codes(qa, fmt, device), _device_codes(_tile_stack(qw) if tiled else qw, fmt, device),
                                torch.from_numpy(sa).to(device), torch.from_numpy(sw).to(device),
                                torch.from_numpy(offsets).to(device), swiglu=swiglu, b_tiled=tiled, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (out[rows:] == 7.0).all()
    got = out.double().cpu().numpy()
    for i in range(e):
        lo, hi = offsets[i], offsets[i + 1]
        if lo == hi:
            continue
        y, b = R.scaled(oracle, fmt, qa[lo:hi], sa[lo:hi], qw[i], sw[i])
        if swiglu:
            y, b = R.swiglu(y, b)
        bound = b + R.HALF_BF16 * (np.abs(y) + b) + 2.0 ** -133
        assert (np.abs(got[lo:hi] - y) <= bound).all(), (i, np.max(np.abs(got[lo:hi] - y) / bound))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("tiled,k", [(True, 384), (False, 336)])
@pytest.mark.parametrize("out", ["bf16", "f32", "swiglu"])
def test_grouped_many_tiles(ops, device, oracle, fmt, tiled, k, out):
    """More 256 x 256 tiles than the chip has workgroups for, whole and half ones, and a last
    column tile that is not full: every row, a sample of the columns."""
    counts = [1100, 0, 129, 2000, 128, 700, 1]
    e, n = len(counts), 5216
    rows = sum(counts)
    x = activations(rows, k, seed=21, outlier_channels=2)
    qa, sa = oracle.quant_rows(bits16(x), fmt, "rcp" if fmt == "int8" else "div")
    qa, sa = qa.view(np.uint8), sa.ravel()
    f = ops.FMT_INT8 if fmt == "int8" else ops.FMT_E4M3FN
    gen = torch.Generator(device=device).manual_seed(5)
    w = (torch.randn(e * n, k, generator=gen, device=device) * 0.05).to(torch.bfloat16)
    qw, sw = ops.quant_rows(w, f)
    stack = ops.quant_rows_tiled(w, f)[0] if tiled else qw
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    got = ops.grouped_scaled_mm(_device_codes(qa, fmt, device), stack.view(e, n, k), torch.from_numpy(sa).to(device),
                                sw.view(e, n), torch.from_numpy(offsets).to(device), swiglu=out == "swiglu", b_tiled=tiled,
                                out_dtype=torch.float32 if out == "f32" else torch.bfloat16).double().cpu().numpy()
    half = n // 2
    sample = np.unique(np.concatenate((np.arange(0, half, 97), [15, 16, 63, 64, 127, 128, 255, 256, half - 1])))
    cols = np.concatenate((sample, half + sample))
    qs = qw.view(e, n, k)[:, cols].contiguous().view(torch.uint8).cpu().numpy()
    ss = sw.view(e, n)[:, cols].cpu().numpy()
    for i in range(e):
        lo, hi = offsets[i], offsets[i + 1]
        if lo == hi:
            continue
        y, b = R.scaled(oracle, fmt, qa[lo:hi], sa[lo:hi], qs[i], ss[i])
        mine = got[lo:hi][:, sample if out == "swiglu" else cols]
        if out == "swiglu":
            y, b = R.swiglu(y, b)
        bound = b + (0.0 if out == "f32" else R.HALF_BF16) * (np.abs(y) + b) + 2.0 ** -133
        assert (np.abs(mine - y) <= bound).all(), (i, np.max(np.abs(mine - y) / bound))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t,k_top,e", [(3, 2, 4), (90, 3, 5), (700, 2, 3)])
def test_grouped_gathers_rows(ops, device, fmt, t, k_top, e):
    """A gathered call equals the call on rows copied into the plan's order, bit for bit,
    and its binary32 output rounds to its bf16 output."""
    gen = torch.Generator().manual_seed(t)
    k, n = 384, 96
    f = ops.FMT_INT8 if fmt == "int8" else ops.FMT_E4M3FN
    ids = torch.randint(-1, e + 1, (t, k_top), generator=gen, dtype=torch.int32).to(device)
    plan = ops.plan_experts(ids, e)
    x = activations(t, k, seed=4).to(device)
    q, s = ops.quant_rows(x, f)
    w, sw = ops.quant_rows(activations(e * n, k, seed=5).to(device), f)
    w, sw = w.view(e, n, k), sw.view(e, n)
    used = int(plan.offsets[-1])
    rows = (plan.order.clamp(min=0) // k_top).long()
    qs, ss = q.view(torch.uint8)[rows].view(q.dtype), s[rows]
    for swiglu in (False, True):
        a = ops.grouped_scaled_mm(q, w, s, sw, plan.offsets, order=plan.order, top_k=k_top, swiglu=swiglu)
        b = ops.grouped_scaled_mm(qs, w, ss, sw, plan.offsets, swiglu=swiglu)
        assert torch.equal(a[:used].view(torch.int16), b[:used].view(torch.int16))
    a = ops.grouped_scaled_mm(q, w, s, sw, plan.offsets, order=plan.order, top_k=k_top)
    wide = ops.grouped_scaled_mm(q, w, s, sw, plan.offsets, order=plan.order, top_k=k_top, out_dtype=torch.float32)
    assert torch.equal(wide[:used].to(torch.bfloat16), a[:used])


def test_grouped_strided_operands(ops, device):
    e, n, k = 3, 64, 256
    wide = activations(40, 512, seed=8).to(device)
    q, s = ops.quant_rows(wide, ops.FMT_INT8)
    w, sw = ops.quant_rows(activations(e * n, k, seed=9).to(device), ops.FMT_INT8)
    offsets = torch.tensor([0, 10, 10, 40], dtype=torch.int32, device=device)
    part = q[:, 128:384]
    buffer = torch.zeros(40, 128, device=device, dtype=torch.bfloat16)
    ops.grouped_scaled_mm(part, w.view(e, n, k), s, sw.view(e, n), offsets, out=buffer[:, 32:96])
    plain = ops.grouped_scaled_mm(part.contiguous(), w.view(e, n, k), s, sw.view(e, n), offsets)
    assert torch.equal(buffer[:, 32:96], plain)
    assert (buffer[:, :32] == 0).all() and (buffer[:, 96:] == 0).all()


@pytest.mark.parametrize("experts,rows", [(1024, 10000), (64, 10000), (2, 10000)])
def test_grouped_offsets_past_32_bits(ops, device, experts, rows):
    """Rows of codes and of outputs that lie past 4 GiB of their tensors, through every kernel (by the
    mean rows of an expert: 9, 156 and 5000): the last rows equal a call on those rows alone."""
    k, n, a_stride, o_stride = 384, 64, 1 << 19, 1 << 18  # 5 GB of codes, 5 GB of outputs
    gen = torch.Generator(device=device).manual_seed(1)
    a = torch.empty(rows, a_stride, device=device, dtype=torch.int8)[:, :k]
    a.copy_(torch.randint(-127, 128, (rows, k), device=device, generator=gen))
    s = torch.rand(rows, device=device, generator=gen)
    w = torch.randint(-127, 128, (experts, n, k), device=device, generator=gen).to(torch.int8)
    sw = torch.rand(experts, n, device=device, generator=gen)
    out = torch.empty(rows, o_stride, device=device, dtype=torch.bfloat16)[:, :n]
    offsets = torch.full((experts + 1,), rows, dtype=torch.int32, device=device)
    offsets[0], offsets[1] = 0, rows - 300
    ops.grouped_scaled_mm(a, w, s, sw, offsets, out=out)
    tail = a[-300:].contiguous()
    want = ops.grouped_scaled_mm(tail, w[1:2].contiguous(), s[-300:].contiguous(), sw[1:2].contiguous(),
                                 torch.tensor([0, 300], dtype=torch.int32, device=device))
    assert torch.equal(out[-300:].contiguous().view(torch.int16), want.view(torch.int16))


def test_grouped_bounds_beyond_the_rows(ops, device):
    """Offsets that claim more rows than the call has, and order entries past the tokens,
    touch nothing beside the call's own rows."""
    q, s = ops.quant_rows(activations(8, 128, seed=1).to(device), ops.FMT_INT8)
    w, sw = ops.quant_rows(activations(64, 128, seed=2).to(device), ops.FMT_INT8)
    out = torch.zeros(8, 32, device=device, dtype=torch.bfloat16)
    for bounds in ([0, 4, 1000], [-5, 3, 8], [0, 8, 2], [1 << 30, 0, 8]):
        offsets = torch.tensor(bounds, dtype=torch.int32, device=device)
        ops.grouped_scaled_mm(q, w.view(2, 32, 128), s, sw.view(2, 32), offsets, out=out)
    order = torch.tensor([0, 7, 8, 100, -1, 2 ** 31 - 1, 1, 2], dtype=torch.int32, device=device)
    offsets = torch.tensor([0, 8, 8], dtype=torch.int32, device=device)
    got = ops.grouped_scaled_mm(q, w.view(2, 32, 128), s, sw.view(2, 32), offsets, order=order)
    rows = ops.grouped_scaled_mm(q, w.view(2, 32, 128), s, sw.view(2, 32), offsets)
    assert torch.equal(got[[0, 1, 6, 7]], rows[[0, 7, 1, 2]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k,cols", [(1, 1, 8), (5, 3, 136), (33, 8, 2048), (7, 9, 24)])
def test_combine(ops, device, dtype, t, k, cols):
    gen = torch.Generator().manual_seed(cols)
    rows = t * k
    y = torch.randn(rows, cols, generator=gen).to(dtype)
    slots = torch.randperm(rows, generator=gen).to(torch.int32).view(t, k)
    slots[torch.rand(t, k, generator=gen) < 0.3] = -1
    slots[0, 0] = rows  # out of range: adds nothing
    w = torch.rand(t, k, generator=gen)
    got = ops.combine_experts(y.to(device), slots.to(device), w.to(device)).double().cpu()
    terms = torch.where(((slots >= 0) & (slots < rows))[:, :, None], y.double()[slots.clamp(0, rows - 1).long()] * w.double()[:, :, None], 0.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    assert ((got - want).abs() <= R.HALF_BF16 * want.abs() + 2 * k * R.U32 * size + 2.0 ** -133).all()


# ------------------------------------------------------------------- layer

def _layer(ops, experts_module, device, oracle, fmt, e, d, f, first=0, seed=11):
    gen = torch.Generator().manual_seed(seed)
    w13 = (torch.randn(e, 2 * f, d, generator=gen) * d ** -0.5).to(torch.bfloat16)
    w2 = (torch.randn(e, d, f, generator=gen) * f ** -0.5).to(torch.bfloat16)
    layer = experts_module.QuantizedExperts.from_weights(
        w13.to(device), w2.to(device), ops.FMT_INT8 if fmt == "int8" else ops.FMT_E4M3FN, first_expert=first)
    return layer, (*R.quantize_weights(w13, oracle, fmt), *R.quantize_weights(w2, oracle, fmt))


def _routed(t, k, total, seed):
    gen = torch.Generator().manual_seed(seed)
    ids, weights = R.route(torch.randn(t, total, generator=gen) * 2, k, "softmax", True)
    if t > 2:
        ids[1], weights[1] = -1, 0.0  # a padded token
    return ids, weights.astype(np.float32)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t,k,total,e,first,d,f", [
    (1, 1, 1, 1, 0, 128, 128), (1, 8, 16, 16, 0, 512, 256), (3, 2, 8, 8, 0, 640, 384), (7, 4, 12, 4, 4, 256, 128),
    (5, 2, 6, 6, 0, 144, 80), (21, 3, 8, 8, 0, 272, 208), (20, 8, 40, 40, 0, 256, 256), (150, 2, 4, 4, 0, 384, 128),
    (400, 4, 8, 4, 2, 256, 256), (64, 1, 2, 2, 0, 128, 1024), (8, 8, 64, 64, 0, 256, 512), (1, 64, 64, 64, 0, 384, 256),
    (2, 32, 300, 300, 0, 256, 128), (16, 4, 40, 20, 20, 16, 16)])
def test_expert_ffn(ops, experts_module, device, oracle, fmt, t, k, total, e, first, d, f):
    layer, packed = _layer(ops, experts_module, device, oracle, fmt, e, d, f, first)
    x = activations(t, d, seed=t + d, outlier_channels=2)
    ids, weights = _routed(t, k, total, t + k)
    got = layer(x.to(device), torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device))
    want, bound = R.ffn(oracle, fmt, x, ids, weights, *packed, first=first)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), np.max(err / bound)
    # the bound itself stays small beside the values: a few bf16 steps, or of a moved code of h
    assert np.linalg.norm(err) <= 0.02 * np.linalg.norm(want)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("f", [128, 256, 384, 512, 640, 896, 1024, 1152])
@pytest.mark.parametrize("hit", [0, 1, 2, 3])
def test_few_pairs_of_few_experts(ops, experts_module, device, oracle, fmt, f, hit):
    """Fewer k-steps than waves (some have none): 0 to 3 experts of a rank hit, after a call that
    leaves other sums in the same LDS."""
    layer, packed = _layer(ops, experts_module, device, oracle, fmt, 16, 128, f)
    gen = torch.Generator().manual_seed(f)
    full = torch.stack([torch.randperm(16, generator=gen)[:8] for _ in range(8)]).to(torch.int32).to(device)
    layer(activations(8, 128, seed=3).to(device) * 1000.0, full, torch.ones(8, 8, device=device))
    ids = np.full((2, 6), -1, np.int32)
    for i in range(hit):
        ids[i % 2, 2 * i] = 5 * i
    weights = np.full((2, 6), 0.5, np.float32)
    x = activations(2, 128, seed=f)
    got = layer(x.to(device), torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device))
    want, bound = R.ffn(oracle, fmt, x, ids, weights, *packed)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t,k,e,d,f", [(1, 4, 8, 512, 384), (6, 8, 16, 256, 640), (40, 2, 8, 384, 256), (300, 4, 8, 256, 384)])
def test_expert_ffn_is_the_chain(ops, experts_module, device, oracle, fmt, t, k, e, d, f):
    """The layer against the operators one by one: the same bits in int8 (its sums are exact); in
    e4m3 the order of the sums may differ, so within the bound of the two."""
    layer, packed = _layer(ops, experts_module, device, oracle, fmt, e, d, f)
    code = ops.FMT_INT8 if fmt == "int8" else ops.FMT_E4M3FN
    rounding = ops.ROUND_RCP_MUL if fmt == "int8" else ops.ROUND_DIV
    x = activations(t, d, seed=2, outlier_channels=2).to(device)
    gen = torch.Generator().manual_seed(t)
    ids, weights = ops.route_experts(torch.randn(t, e, generator=gen).to(device), k)
    got = layer(x, ids, weights)
    plan = ops.plan_experts(ids, e)
    q, s = ops.quant_rows(x, code, rounding)
    h = ops.grouped_scaled_mm(q, layer.w13, s, layer.w13_scale, plan.offsets, order=plan.order, top_k=k, swiglu=True,
                              b_tiled=layer.w13_tiled)
    qh, sh = ops.quant_rows(h, code, rounding)
    y = ops.grouped_scaled_mm(qh, layer.w2, sh, layer.w2_scale, plan.offsets, b_tiled=layer.w2_tiled,
                              out_dtype=torch.float32)
    chain = ops.combine_experts(y, plan.slots, weights)
    if fmt == "int8":
        assert torch.equal(got.view(torch.int16), chain.view(torch.int16))
    else:
        _, bound = R.ffn(oracle, fmt, x.cpu(), ids.cpu().numpy(), weights.cpu().numpy(), *packed)
        assert (np.abs((got.double() - chain.double()).cpu().numpy()) <= 2 * bound).all()


def test_repeated_expert_and_unnormalized_weights(ops, experts_module, device, oracle):
    """The same expert twice in a token's slots, weights of any size and sign."""
    layer, packed = _layer(ops, experts_module, device, oracle, "int8", 4, 256, 128)
    x = activations(9, 256, seed=3)
    ids = np.array([[2, 2, 1], [0, 0, 0], [3, 1, 3], [-1, 2, -1], [1, 1, 2], [0, 3, 3], [2, 2, 2], [1, 0, 1], [-1, -1, -1]],
                   np.int32)
    weights = np.random.default_rng(1).normal(size=ids.shape).astype(np.float32) * 3
    got = layer(x.to(device), torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device))
    want, bound = R.ffn(oracle, "int8", x, ids, weights, *packed)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    assert (got[8] == 0).all()


def test_expert_parallel_parts_add_up(ops, experts_module, device, oracle):
    """The parts of two ranks against the layer of all experts: within both sides' bounds."""
    whole, packed = _layer(ops, experts_module, device, oracle, "int8", 8, 256, 256)
    x = activations(30, 256, seed=6)
    ids, weights = _routed(30, 3, 8, 5)
    args = (x.to(device), torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device))
    total = torch.zeros(30, 256, dtype=torch.float64)
    for first in (0, 4):
        part = experts_module.QuantizedExperts(whole.w13[first:first + 4].clone(), whole.w13_scale[first:first + 4].clone(),
                                               whole.w2[first:first + 4].clone(), whole.w2_scale[first:first + 4].clone(),
                                               w13_tiled=whole.w13_tiled, w2_tiled=whole.w2_tiled, first_expert=first)
        total += part(*args).double().cpu()
    want, bound = R.ffn(oracle, "int8", x, ids, weights, *packed)
    parts = sum(R.ffn(oracle, "int8", x, ids, weights, *(p[f:f + 4] for p in packed), first=f)[1] for f in (0, 4))
    assert (np.abs(total.numpy() - want) <= parts + R.U32 * np.abs(want)).all()


def test_rows_with_infinities_stay_their_own(ops, experts_module, device, oracle):
    """A token that holds an infinity or a NaN changes no other token's result."""
    layer, _ = _layer(ops, experts_module, device, oracle, "e4m3", 4, 256, 128)
    x = activations(12, 256, seed=9).to(device)
    ids, weights = _routed(12, 2, 4, 3)
    ids, weights = torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device)
    clean = layer(x, ids, weights)
    dirty = x.clone()
    dirty[4, 7], dirty[9, 0] = torch.inf, torch.nan
    got = layer(dirty, ids, weights)
    keep = [i for i in range(12) if i not in (4, 9)]
    assert torch.equal(got[keep].view(torch.int16), clean[keep].view(torch.int16))
    assert torch.isnan(got[9]).any()


def test_moe_module_routes_and_sums(ops, experts_module, device, oracle):
    layer, packed = _layer(ops, experts_module, device, oracle, "int8", 8, 256, 128)
    gen = torch.Generator().manual_seed(4)
    router = (torch.randn(8, 256, generator=gen) * 0.1).to(device)
    moe = experts_module.QuantizedMoE(router, layer, top_k=2, scale=2.0)
    x = activations(24, 256, seed=1).to(device)
    got = moe(x.view(2, 12, 256))
    assert got.shape == (2, 12, 256)
    ids, weights = ops.route_experts(torch.nn.functional.linear(x.float(), router), 2, scale=2.0)
    want, bound = R.ffn(oracle, "int8", x.cpu(), ids.cpu().numpy(), weights.cpu().numpy(), *packed)
    assert (np.abs(got.view(24, 256).double().cpu().numpy() - want) <= bound).all()


def test_no_tokens_strided_x_and_out(ops, experts_module, device, oracle):
    layer, _ = _layer(ops, experts_module, device, oracle, "int8", 4, 256, 128)
    empty = layer(torch.empty(0, 256, device=device, dtype=torch.bfloat16),
                  torch.empty(0, 2, device=device, dtype=torch.int32), torch.empty(0, 2, device=device))
    assert empty.shape == (0, 256)
    ids, weights = _routed(5, 2, 4, 3)
    ids, weights = torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device)
    wide = activations(5, 512, seed=5).to(device)
    out = torch.zeros(5, 320, device=device, dtype=torch.bfloat16)
    w = (layer.w13, layer.w13_scale, layer.w2, layer.w2_scale)
    tiles = {"w13_tiled": layer.w13_tiled, "w2_tiled": layer.w2_tiled}
    ops.expert_ffn(wide[:, 128:384], ids, weights, *w, **tiles, out=out[:, 32:288])
    plain = ops.expert_ffn(wide[:, 128:384].contiguous(), ids, weights, *w, **tiles)
    assert torch.equal(out[:, 32:288].view(torch.int16), plain.view(torch.int16))
    assert (out[:, :32] == 0).all() and (out[:, 288:] == 0).all()


@pytest.mark.parametrize("t,k", [(1, 4), (20, 4), (200, 2)])
def test_layer_in_graphs_on_streams(ops, experts_module, device, oracle, t, k):
    """Two captured layers that share the program's pool, replayed with eager calls and new inputs
    between them, on a side stream: every replay gives the eager bits."""
    layer, _ = _layer(ops, experts_module, device, oracle, "e4m3", 8, 256, 384)
    router = torch.randn(8, 256, device=device) * 0.1
    moe = experts_module.QuantizedMoE(router, layer, top_k=k)
    xs = [activations(t, 256, seed=i).to(device) for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moe(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(moe(x))
        graphs.append(g)
    for replay in range(3):
        for i in (0, 1):
            xs[i].copy_(activations(t, 256, seed=10 * replay + i).to(device))
            want = moe(xs[i])
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i].view(torch.int16), want.view(torch.int16)), (replay, i)


def test_two_calls_on_two_streams(ops, experts_module, device, oracle):
    layer, _ = _layer(ops, experts_module, device, oracle, "int8", 8, 256, 384)
    ids, weights = _routed(40, 3, 8, 3)
    ids, weights = torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device)
    xs = [activations(40, 256, seed=i).to(device) for i in range(2)]
    want = [layer(x, ids, weights) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(layer(x, ids, weights))
        torch.cuda.synchronize()
        assert all(torch.equal(g.view(torch.int16), w.view(torch.int16)) for g, w in zip(got, want))


def test_native_wrappers_equal_the_python_bodies(ops, experts_module, device, oracle, monkeypatch):
    """Every call once through the native wrapper and once with it declining: the same bits."""
    layer, _ = _layer(ops, experts_module, device, oracle, "e4m3", 6, 256, 128)
    x = activations(40, 256, seed=4).to(device)
    logits = torch.randn(40, 6, device=device)
    native, taken = ops._native_call, []

    def calls():
        ids, w = ops.route_experts(logits, 3, scoring="sigmoid")
        plan = ops.plan_experts(ids, 6)
        q, s = ops.quant_rows(x, ops.FMT_E4M3FN)
        used = int(plan.offsets[-1])
        h = ops.grouped_scaled_mm(q, layer.w13, s, layer.w13_scale, plan.offsets, order=plan.order, top_k=3, swiglu=True,
                                  b_tiled=True)[:used]
        y = torch.randn(120, 64, device=device, generator=torch.Generator(device=device).manual_seed(1))
        return (ids, w, *plan, h, ops.combine_experts(y, plan.slots, w), layer(x, ids, w), layer(x[:2], ids[:2], w[:2]))

    def hook(enabled):
        def call(name, first, *args):
            out = native(name, first, *args) if enabled else None
            taken.append(out is not None)
            return out
        return call

    results = []
    for enabled in (True, False):
        taken.clear()
        monkeypatch.setattr(ops, "_native_call", hook(enabled))
        results.append(calls())
        assert all(taken) == enabled and any(taken) == enabled
    for a, b in zip(*results):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_in_place_layer(ops, experts_module, device, oracle):
    """The output may be the input: x is read before any of it is written."""
    layer, _ = _layer(ops, experts_module, device, oracle, "int8", 4, 256, 128)
    for t in (3, 50):
        x = activations(t, 256, seed=t).to(device)
        ids, weights = _routed(t, 2, 4, 1)
        ids, weights = torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device)
        want = layer(x, ids, weights)
        ops.expert_ffn(x, ids, weights, layer.w13, layer.w13_scale, layer.w2, layer.w2_scale, w13_tiled=True, w2_tiled=True,
                       out=x)
        assert torch.equal(x.view(torch.int16), want.view(torch.int16))


# --------------------------------------------------------------- refusals

def test_refusals(ops, experts_module, device, oracle):
    layer, _ = _layer(ops, experts_module, device, oracle, "int8", 4, 256, 128)
    x = activations(5, 256, seed=1).to(device)
    ids = torch.zeros(5, 2, dtype=torch.int32, device=device)
    w = torch.ones(5, 2, device=device)
    args = (layer.w13, layer.w13_scale, layer.w2, layer.w2_scale)
    tiles = {"w13_tiled": True, "w2_tiled": True}
    for bad, exc in (((x.float(), ids, w), TypeError), ((x, ids.long(), w), TypeError), ((x, ids[:4], w), ValueError),
                     ((x, ids, w[:, :1]), ValueError), ((x, ids, w.double()), TypeError), ((x[:, :128], ids, w), ValueError)):
        with pytest.raises(exc):
            ops.expert_ffn(*bad, *args, **tiles)
    with pytest.raises(ValueError, match="tiled"):
        ops.expert_ffn(x, ids, w, *args)  # tiled codes passed as rows
    with pytest.raises(ValueError):
        ops.expert_ffn(x, ids, w, layer.w13, layer.w13_scale[:, :-1], layer.w2, layer.w2_scale, **tiles)
    with pytest.raises(TypeError):
        ops.expert_ffn(x, ids, w, layer.w13, layer.w13_scale, layer.w2.view(torch.uint8), layer.w2_scale, **tiles)
    with pytest.raises(RuntimeError, match="first expert"):
        ops.expert_ffn(x, ids, w, *args, **tiles, first_expert=-1)
    with pytest.raises(ValueError):
        ops.route_experts(torch.zeros(4, 8, device=device), 9)
    with pytest.raises(ValueError):
        ops.route_experts(torch.zeros(4, 8, device=device), 2, scoring="tanh")
    with pytest.raises(TypeError):
        ops.route_experts(torch.zeros(4, 8, device=device, dtype=torch.float64), 2)
    for count in (0, -3, 1025, 2 ** 40):
        with pytest.raises(RuntimeError, match="experts"):
            ops.plan_experts(ids, count)
    q, s = ops.quant_rows(x, ops.FMT_INT8)
    offsets = torch.zeros(5, dtype=torch.int32, device=device)
    with pytest.raises(ValueError):
        ops.grouped_scaled_mm(q, layer.w13, s, layer.w13_scale, offsets[:4], b_tiled=True)
    with pytest.raises(TypeError):
        ops.grouped_scaled_mm(q, layer.w13, s, layer.w13_scale, offsets, b_tiled=True, swiglu=True, out_dtype=torch.float32)
    with pytest.raises(ValueError):
        ops.grouped_scaled_mm(q, layer.w13, s, layer.w13_scale, offsets, b_tiled=True,
                              out=torch.empty(4, 256, device=device, dtype=torch.bfloat16))
    y = torch.zeros(10, 256, device=device, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.combine_experts(y, ids, w[:4])
    with pytest.raises(RuntimeError, match="columns"):
        ops.combine_experts(y[:, :12], ids, w)
