"""Routed-expert operators on the GPU: the contract of rows that are not the call's, router
weights far below zero, and every kernel of the grouped products and of the layer by its own
sizes (the sizes that choose it stand at each test)."""

from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

import _experts as R
from _util import activations

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def experts_module():
    return importlib.import_module("taomate_h3_amd.inference.experts")


def _bits(t: torch.Tensor) -> torch.Tensor:
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def _codes(ops, rows, k, fmt, device, seed):
    return ops.quant_rows(activations(rows, k, seed=seed, outlier_channels=2).to(device),
                          ops.FMT_INT8 if fmt == "int8" else ops.FMT_E4M3FN)


def _stack(ops, e, n, k, fmt, device, tiled, seed=5):
    gen = torch.Generator(device=device).manual_seed(seed)
    w = (torch.randn(e * n, k, generator=gen, device=device) * 0.05).to(torch.bfloat16)
    quantize = ops.quant_rows_tiled if tiled else ops.quant_rows
    codes, scales = quantize(w, ops.FMT_INT8 if fmt == "int8" else ops.FMT_E4M3FN)
    return codes.view(e, n, k), scales.view(e, n)


def _offsets(counts, device):
    return torch.from_numpy(np.concatenate(([0], np.cumsum(counts))).astype(np.int32)).to(device)


# Counts of two experts whose mean takes each kernel: streams (to 10 rows), bands of 64 (to 64)
# and of 128 rows (to 384 or 512), 256 x 256 tiles (above).
_EVERY_KERNEL = [[5, 11], [37, 66], [130, 271], [300, 1001]]
_KERNEL_IDS = ["stream", "band64", "band128", "tile"]


# ------------------------------------------------- rows that are not the call's

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("counts", _EVERY_KERNEL, ids=_KERNEL_IDS)
@pytest.mark.parametrize("form", ["bf16", "f32", "swiglu"])
@pytest.mark.parametrize("tiled", [True, False])
def test_rows_of_invalid_order_entries_stay(ops, device, fmt, counts, form, tiled):
    """A row whose order entry names no row of a keeps what out held; so do the rows past the last
    group and everything around out.  The other rows equal the call on sorted rows, bit for bit."""
    k, n, top_k, spare = 384, 96, 2, 3
    rows = sum(counts)
    tokens = rows // 2 + 1
    q, s = _codes(ops, tokens, k, fmt, device, rows)
    w, sw = _stack(ops, 2, n, k, fmt, device, tiled)
    gen = torch.Generator().manual_seed(rows)
    order = torch.randint(0, tokens * top_k, (rows + spare,), generator=gen, dtype=torch.int32)
    bad = torch.rand(rows + spare, generator=gen) < 0.2
    bad[0] = bad[rows - 1] = True
    wrong = torch.tensor([-1, tokens * top_k, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    order[bad] = wrong[torch.randint(0, 4, (int(bad.sum()),), generator=gen)]
    dtype = torch.float32 if form == "f32" else torch.bfloat16
    cols = n // 2 if form == "swiglu" else n
    buffer = torch.full((rows + spare + 20, cols + 32), 7.0, device=device, dtype=dtype)
    out = buffer[10:10 + rows + spare, 16:16 + cols]
    kwargs = {"swiglu": form == "swiglu", "b_tiled": tiled, "out_dtype": dtype}
    ops.grouped_scaled_mm(q, w, s, sw, _offsets(counts, device), order=order.to(device), top_k=top_k, out=out, **kwargs)
    source = (order.clamp(0, tokens * top_k - 1) // top_k).long().to(device)
    want = ops.grouped_scaled_mm(q.view(torch.uint8)[source].view(q.dtype), w, s[source], sw, _offsets(counts, device),
                                 **kwargs)
    good = ~bad
    good[rows:] = False
    assert torch.equal(_bits(out[good.to(device)]), _bits(want[good.to(device)]))
    out[good.to(device)] = 7.0
    assert (buffer == 7.0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("counts", _EVERY_KERNEL, ids=_KERNEL_IDS)
def test_bounds_that_are_no_partition_touch_only_out(ops, device, fmt, counts):
    """Offsets beyond the rows, below zero or falling: nothing around out is written, and a following
    good call is right."""
    k, n = 384, 96
    rows = sum(counts)
    q, s = _codes(ops, rows, k, fmt, device, rows)
    w, sw = _stack(ops, 2, n, k, fmt, device, False)
    buffer = torch.full((rows + 600, n + 32), 7.0, device=device, dtype=torch.bfloat16)
    out = buffer[300:300 + rows, 16:16 + n]
    for bounds in ([0, rows // 2, 10 * rows], [-5, 3, rows], [0, rows, 2], [1 << 30, 0, rows], [rows, rows, rows],
                   [-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1]):
        ops.grouped_scaled_mm(q, w, s, sw, torch.tensor(bounds, dtype=torch.int32, device=device), out=out)
        whole = buffer.clone()
        whole[300:300 + rows, 16:16 + n] = 7.0
        assert (whole == 7.0).all(), bounds
    ops.grouped_scaled_mm(q, w, s, sw, _offsets(counts, device), out=out)
    want = ops.grouped_scaled_mm(q, w, s, sw, _offsets(counts, device))
    assert torch.equal(_bits(out), _bits(want))


# ------------------------------------------------------------ sigmoid shares

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("spare", [0, 4096])  # a wave or 16 lanes a token
def test_renormalized_sigmoid_far_below_zero(ops, device, dtype, spare):
    """Scores of logits below -88 underflow binary32; their shares do not."""
    inf = torch.inf
    rows = torch.tensor([[-100.0, -101.0, -102.5, -100.0], [-88.0, -89.0, -90.0, -95.0], [-1000.0, -1001.0, -1003.0, -inf],
                         [-60000.0, -60000.0, -60032.0, -inf], [-inf, -200.0, -inf, -inf], [-19.0, -18.5, -40.0, -20.0],
                         [-17.0, -17.5, -40.0, -60.0], [-18.0, -18.0, -18.0, -18.0], [0.0, -100.0, -120.0, -1.0]]).to(dtype)
    logits = torch.cat((rows, torch.zeros(spare, 4, dtype=dtype)))
    ids, weights = ops.route_experts(logits.to(device), 3, scoring="sigmoid", renormalize=True, scale=2.0)
    got = weights[:len(rows)].double().cpu()
    want_ids, _ = R.route(rows, 3, "sigmoid", False)
    assert (ids[:len(rows)].cpu().numpy() == want_ids).all()
    taken = torch.from_numpy(want_ids >= 0)
    l = torch.where(taken, rows.double().gather(1, torch.from_numpy(want_ids).clamp(min=0).long()), -inf)
    log_score = torch.where(taken, -torch.logaddexp(torch.zeros(()).double(), -l), -inf)
    want = 2.0 * torch.softmax(log_score, 1)
    # A score by the hardware exp of x: (|x| + 2) 2^-23 of it, x the logit, or its distance from the
    # largest where that one is far below zero; the sum as a whole the same again; 3 additions, the
    # quotient, the scale and 1 + exp(l): 8 half-steps.  Scores below 2^-126 may become zero: of a
    # sum of at least 2^-26, doubled by the scale, 2^-99.
    far = l[:, :1] < -18.0
    x = torch.where(taken, torch.where(far, l[:, :1] - l, l.abs()), 0.0).amax(1, keepdim=True)
    bound = want * (2 * 2 * (x + 2) + 8) * R.U32 + 2.0 ** -99
    assert ((got - want).abs() <= bound).all(), (got, want)
    assert (got[~taken] == 0).all()


# ------------------------------------------------------- grouped: every kernel

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("tiled,k", [(True, 384), (False, 336)])
@pytest.mark.parametrize("form", ["bf16", "f32", "swiglu"])
def test_gathered_rows_over_many_tiles(ops, device, fmt, tiled, k, form):
    """More 256 x 256 tiles than the chip has workgroups for (mean 579 rows): a tile's order is fetched
    while another runs.  Bit for bit the call on sorted rows."""
    counts, n, top_k = [1100, 0, 129, 2000, 128, 700, 1], 5216, 3
    rows, tokens = sum(counts), 1500
    q, s = _codes(ops, tokens, k, fmt, device, 3)
    w, sw = _stack(ops, len(counts), n, k, fmt, device, tiled)
    gen = torch.Generator().manual_seed(k)
    order = torch.randint(0, tokens * top_k, (rows,), generator=gen, dtype=torch.int32).to(device)
    source = (order // top_k).long()
    kwargs = {"swiglu": form == "swiglu", "b_tiled": tiled,
              "out_dtype": torch.float32 if form == "f32" else torch.bfloat16}
    got = ops.grouped_scaled_mm(q, w, s, sw, _offsets(counts, device), order=order, top_k=top_k, **kwargs)
    want = ops.grouped_scaled_mm(q.view(torch.uint8)[source].view(q.dtype), w, s[source], sw, _offsets(counts, device),
                                 **kwargs)
    assert torch.equal(_bits(got), _bits(want))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("e", [65, 130])
@pytest.mark.parametrize("mean", [4, 30, 150, 600], ids=_KERNEL_IDS)
@pytest.mark.parametrize("form", ["bf16", "swiglu"])
def test_more_experts_than_lanes(ops, device, fmt, e, mean, form):
    """65 and 130 experts, some empty, in one call equal the same experts in calls of at most 64, bit
    for bit (each part's mean takes the same kernel as the whole's)."""
    k, n = 384, 96
    pattern = np.array([0, 2, 1, 0, 1, 2, 1, 1])  # mean 1; the counts of a part stay near the mean
    counts = pattern[np.arange(e) % 8] * mean + np.array([0, 1, 0, 0, 1, 0, 0, 1])[np.arange(e) % 8]
    rows = int(counts.sum())
    q, s = _codes(ops, rows, k, fmt, device, e)
    w, sw = _stack(ops, e, n, k, fmt, device, True)
    kwargs = {"swiglu": form == "swiglu", "b_tiled": True}
    got = ops.grouped_scaled_mm(q, w, s, sw, _offsets(counts, device), **kwargs)
    starts = np.concatenate(([0], np.cumsum(counts)))
    for lo in range(0, e, 40):
        hi = min(lo + 40, e)
        a, b = int(starts[lo]), int(starts[hi])
        want = ops.grouped_scaled_mm(q[a:b], w[lo:hi].contiguous(), s[a:b], sw[lo:hi].contiguous(),
                                     _offsets(counts[lo:hi], device), **kwargs)
        assert torch.equal(_bits(got[a:b]), _bits(want)), lo


@pytest.mark.parametrize("counts", _EVERY_KERNEL, ids=_KERNEL_IDS)
def test_swiglu_of_far_negative_gates(ops, device, counts):
    """Gates down to -88.7, where exp(-g) still is a binary32 number and its reciprocal no normal one,
    beside up values that bring the product back to size."""
    k, rows = 272, sum(counts)
    gates = torch.tensor([-88.7, -88.5, -88.0, -87.6, -87.4, -87.3, -86.0, -60.0, -1.0, 0.0, 1e-30, 3.0, 90.0])
    g = gates[torch.arange(rows) % len(gates)]
    q = torch.zeros(rows, k, dtype=torch.int8)
    q[:, 0] = 1
    w = torch.zeros(2, 96, k, dtype=torch.int8)
    w[:, :, 0] = 1
    sw = torch.cat((torch.ones(48), torch.full((24,), -1e30), torch.full((24,), 3.0))).expand(2, 96).contiguous()
    got = ops.grouped_scaled_mm(q.to(device), w.to(device), g.to(device), sw.to(device), _offsets(counts, device),
                                swiglu=True).double().cpu().numpy()
    y = g.double().numpy()[:, None] * sw[0].double().numpy()[None, :]
    y_bound = 2.5 * R.U32 * np.abs(y)
    y_bound[:, :48] = 0.0  # gates: products with 1, exact
    want, bound = R.swiglu(y, y_bound)
    assert (np.abs(got - want) <= bound + R.HALF_BF16 * (np.abs(want) + bound) + 2.0 ** -133).all()


# -------------------------------------------------------- layer: every kernel

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
    # few tokens, 16 output columns a workgroup (d >= 4096), rows longer than the registers of a wave
    # (2048 columns) and of a workgroup (8192), codes made inside and by a launch of their own
    (3, 2, 4, 4, 0, 4096, 128), (3, 2, 4, 4, 0, 4112, 144), (12, 2, 4, 4, 0, 4096, 128), (1, 2, 2, 2, 0, 8320, 16),
    (3, 2, 4, 4, 0, 128, 2304), (10, 3, 4, 4, 0, 128, 2304), (2, 1, 1, 1, 0, 4096, 4096),
    # row-major weights, more than 64 pairs: streams, bands of 64 and of 128 rows
    (40, 2, 16, 16, 0, 272, 208), (100, 1, 4, 4, 0, 272, 144), (300, 1, 2, 2, 0, 144, 208),
    # tiled weights in bands of 64 rows; more than 512 tokens; more than 2048 pairs; a rank's share of them
    (100, 1, 4, 4, 0, 256, 128), (520, 1, 16, 16, 0, 256, 128), (1030, 2, 8, 8, 0, 256, 128),
    (1030, 2, 16, 8, 8, 272, 80), (520, 1, 90, 90, 0, 128, 128),
    # above 512 rows an expert: tiles (e4m3: for the down product)
    (1100, 1, 2, 2, 0, 384, 384)])
def test_layer_kernels(ops, experts_module, device, oracle, fmt, t, k, total, e, first, d, f):
    layer, packed = _layer(ops, experts_module, device, oracle, fmt, e, d, f, first)
    x = activations(t, d, seed=t + d, outlier_channels=2)
    ids, weights = _routed(t, k, total, t + k)
    got = layer(x.to(device), torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device))
    want, bound = R.ffn(oracle, fmt, x, ids, weights, *packed, first=first)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), np.max(err / bound)
    assert np.linalg.norm(err) <= 0.02 * np.linalg.norm(want)


def _cancelling(rows, k, gen, signs):
    """e4m3 values [rows, k] in 16 groups of 8 columns (the rest 0): one of 448 (its sign the
    group's) and seven of 2.5 to 3.5."""
    v = torch.zeros(rows, k)
    small = torch.tensor([2.5, 3.0, 3.5])
    for i, sign in enumerate(signs):
        g = 8 * (i * (k // 8) // len(signs))
        v[:, g] = 448.0 * sign
        v[:, g + 1:g + 8] = small[torch.randint(0, 3, (rows, 7), generator=gen)]
    return v


@pytest.mark.parametrize("t,k,e,d,f", [
    (3, 2, 4, 256, 128), (3, 2, 4, 272, 144), (12, 2, 4, 4096, 128), (12, 2, 4, 4112, 144),  # few tokens
    (40, 2, 16, 256, 128), (40, 2, 16, 272, 144),                                          # streams
    (100, 1, 4, 256, 128), (100, 1, 4, 272, 144),                                          # bands of 64 rows
    (300, 1, 2, 256, 128), (300, 1, 2, 272, 144)])                                         # bands of 128 rows
def test_e4m3_gate_and_up_are_exact_products(ops, experts_module, device, oracle, monkeypatch, t, k, e, d, f):
    """Gate and up of the e4m3 layer keep what the FP8 instruction drops.  Products of +-448^2 cancel
    over the groups and leave the small ones, all of them below 2^-13 of their group's largest.  Every
    partial sum in any order is a multiple of 1/4 below 2^22 (16 * 448^2 + 112 * 3.5^2): binary32 holds it,
    so the sums of the definition are exact and the bound has no term for them."""
    gen = torch.Generator().manual_seed(t + d)
    signs = [1, -1] * 8
    x = (_cancelling(t, d, gen, [1] * 16) * 2.0 ** -5).to(torch.bfloat16)
    w13 = (_cancelling(e * 2 * f, d, gen, signs) * 2.0 ** -5).to(torch.bfloat16).view(e, 2 * f, d)
    w2 = (torch.randn(e, d, f, generator=gen) * f ** -0.5).to(torch.bfloat16)
    layer = experts_module.QuantizedExperts.from_weights(w13.to(device), w2.to(device), ops.FMT_E4M3FN)
    packed = (*R.quantize_weights(w13, oracle, "e4m3"), *R.quantize_weights(w2, oracle, "e4m3"))
    ids, weights = _routed(t, k, e, t + k)

    def exact(O, fmt, qa, sa, qb, sb):
        a, b = O.e4m3_to_f32(qa).astype(np.float64), O.e4m3_to_f32(qb).astype(np.float64)
        sums = a @ b.T
        assert np.abs(a).max() == 448 and (np.abs(a) @ np.abs(b).T).max() < 2 ** 22 and (sums % 0.25 == 0).all()
        # the inputs tell the two apart: the instruction's model loses more than a quarter of every sum
        model, _ = O.gemm_e4m3_mfma(qa[:4], qb[:16])
        assert (np.abs(model - sums[:4, :16]) > 0.25 * np.abs(sums[:4, :16])).all()
        y = sums * (sa.astype(np.float64)[:, None] * sb.astype(np.float64)[None, :])
        return y, 2.5 * R.U32 * np.abs(y)

    monkeypatch.setattr(R, "scaled", exact)
    got = layer(x.to(device), torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device))
    want, bound = R.ffn(oracle, "e4m3", x, ids, weights, *packed)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), np.max(err / bound)
    assert np.linalg.norm(err) <= 0.02 * np.linalg.norm(want)
