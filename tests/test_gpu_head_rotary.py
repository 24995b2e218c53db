"""Rotary tables, rotation, head norms, the plan and the append to a paged cache on the GPU, against the plain
64-bit forms of _heads.py, at the sizes and layouts that take different kernels."""

from __future__ import annotations

import pytest
import torch

from _heads import assert_close, assert_codes, norm_rotate, plan

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tables(rows, pairs, device, seed=0):
    angle = torch.rand(rows, pairs, generator=_gen(seed), dtype=torch.float64) * 6.3
    return angle.cos().float().to(device), angle.sin().float().to(device)


def _rows(tokens, heads, d, dtype, device, seed=1, pad=0):
    """[tokens, heads, d], a view of wider packed rows with ``pad`` channels before it."""
    wide = torch.randn(tokens, heads * d + 2 * pad, generator=_gen(seed)).to(dtype).to(device)
    return wide[:, pad:pad + heads * d].unflatten(1, (heads, d))


# ---------------------------------------------------------------- tables

@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("pairs", [1, 3, 16, 64, 256])
def test_tables(ops, device, dtype, pairs):
    """|error| <= 12 * 2^-24 of the magnitude: half a turn's part rounded to binary32 moves the value by at most
    pi * 2^-24, sincospif by two steps of 2^-23, the product by 2^-24 twice; binary64 turns by less than 2^-24."""
    positions = torch.tensor([0, 1, 2, 4095, 65537, 1 << 20, 9_999_999, 7]).to(dtype)
    if dtype.is_floating_point:
        positions = torch.cat((positions, torch.tensor([0.25, -3.5]).to(dtype)))
    frequencies, _ = ops.rotary_frequencies(2 * pairs, device=device)
    for magnitude in (1.0, 1.2079):
        cos, sin = ops.rotary_tables(positions.to(device), frequencies, magnitude)
        angle = positions.double()[:, None] * frequencies.cpu()
        for got, want in ((cos, angle.cos()), (sin, angle.sin())):
            assert got.dtype == torch.float32 and got.shape == (len(positions), pairs)
            assert (got.cpu().double() - want * magnitude).abs().max() <= 12 * 2.0 ** -24 * magnitude


def test_tables_refuse_and_empty(ops, device):
    f = torch.ones(4, dtype=torch.float64, device=device)
    cos, sin = ops.rotary_tables(torch.empty(0, dtype=torch.int64, device=device), f)
    assert cos.shape == sin.shape == (0, 4)
    with pytest.raises(TypeError):
        ops.rotary_tables(torch.zeros(3, dtype=torch.int16, device=device), f)
    with pytest.raises(TypeError):
        ops.rotary_tables(torch.zeros(3, dtype=torch.int64, device=device), f.float())
    with pytest.raises(ValueError):
        ops.rotary_tables(torch.zeros(3, 1, dtype=torch.int64, device=device), f)


# -------------------------------------------------------------- rotation

SHAPES = [  # tokens, heads, head_dim, rot_dim
    (1, 1, 2, 2), (1, 32, 128, 128), (5, 3, 6, 2), (7, 5, 36, 36), (3, 2, 72, 24), (130, 28, 128, 64), (33, 7, 80, 32),
    (9, 9, 96, 96), (17, 4, 256, 256), (6, 2, 512, 512), (4, 3, 510, 254), (11, 65, 64, 32), (601, 28, 128, 128),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,heads,d,rot", SHAPES)
def test_rotary(ops, device, tokens, heads, d, rot, dtype, interleaved):
    x = _rows(tokens, heads, d, TYPES[dtype], device, seed=d + rot)
    cos, sin = _tables(50 + tokens, rot // 2, device)
    rows = torch.randint(0, 50 + tokens, (tokens,), generator=_gen(tokens))
    for inverse, positions in ((False, rows.to(device)), (True, rows.int().to(device)), (False, None)):
        got = ops.rotary(x, cos, sin, positions, interleaved=interleaved, inverse=inverse)
        want, size = norm_rotate(x, cos=cos, sin=sin, rows=None if positions is None else rows, interleaved=interleaved,
                                 inverse=inverse)
        assert got.shape == x.shape and got.dtype == x.dtype
        assert_close(got, want, size, d)
        assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("pad", [0, 1, 4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rotary_strided_misaligned_and_in_place(ops, device, dtype, pad):
    """Views that start at any element, of any head order; out = x."""
    cos, sin = _tables(19, 32, device)
    x = _rows(19, 6, 64, TYPES[dtype], device, pad=pad)
    want, size = norm_rotate(x, cos=cos, sin=sin)
    assert_close(ops.rotary(x, cos, sin), want, size, 64)
    flipped = x.transpose(0, 1).contiguous().transpose(0, 1)  # heads outside tokens
    out = torch.zeros(19, 6, 64 + pad, device=device, dtype=x.dtype)[..., pad:]
    assert ops.rotary(flipped, cos, sin, out=out).data_ptr() == out.data_ptr()
    assert_close(out, want, size, 64)
    packed = x._base if x._base is not None else x
    before = packed.clone()
    assert ops.rotary(x, cos, sin, out=x).data_ptr() == x.data_ptr()
    assert_close(x, want, size, 64)
    packed = packed.flatten(1)
    before = before.flatten(1)
    assert torch.equal(packed[:, :pad], before[:, :pad]) and torch.equal(packed[:, pad + 384:], before[:, pad + 384:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 64), (10, 4)])
def test_rotary_padding_far_positions_and_infinities(ops, device, d, rot, interleaved):
    x = _rows(6, 3, d, torch.bfloat16, device)
    x[4, 1, rot:] = torch.tensor([float("inf"), float("nan")], device=device).to(x.dtype).repeat((d - rot) // 2)
    x[5, 2, 0] = float("inf")
    cos, sin = _tables(8, rot // 2, device)
    cos[7, 0], sin[7, 0] = 0.0, 1.0
    rows = torch.tensor([3, -1, 8, -(1 << 40), 2, 7])
    out = torch.full((6, 3, d), 7.0, device=device, dtype=x.dtype)
    ops.rotary(x, cos, sin, rows.to(device), interleaved=interleaved, out=out)
    want, size = norm_rotate(x, cos=cos, sin=sin, rows=rows, interleaved=interleaved)
    for t in (0, 4):
        assert_close(out[t:t + 1], want[t:t + 1], size[t:t + 1], d)
    assert (out[1] == 7.0).all() and (out[3] == 7.0).all()  # padding
    assert torch.isnan(out[2, :, :rot]).all() and torch.equal(out[2, :, rot:], x[2, :, rot:])  # no such angle
    second = 1 if interleaved else rot // 2
    assert torch.isnan(out[5, 2, 0]) and torch.isinf(out[5, 2, second])  # inf * 0 and inf * 1
    rest = [i for i in range(d) if i not in (0, second)]
    assert torch.isfinite(out[5, 2, rest]).all()


def test_rotary_gradient(ops, device):
    """<g, R x> = <R^-1 g, x>, against a sum in 64 bits: inverse=True is the gradient."""
    x, g = (_rows(13, 4, 64, torch.float32, device, seed=s) for s in (1, 2))
    cos, sin = _tables(13, 24, device)
    turned, back = ops.rotary(x, cos, sin), ops.rotary(g, cos, sin, inverse=True)
    a, b = (turned.double() * g.double()).sum(), (back.double() * x.double()).sum()
    # both sides carry up to 3 roundings of 2^-24 a value of |x||g| <= 2 (|a c| + |b s|)
    bound = 8 * 2.0 ** -24 * float((x.double().abs().sum(2) * g.double().abs().sum(2)).sum())
    assert abs(float(a - b)) <= bound
    again = ops.rotary(turned, cos, sin, inverse=True)
    norm = (cos.double() ** 2 + sin.double() ** 2 - 1).abs().max()
    assert norm < 4 * 2.0 ** -24
    size = norm_rotate(turned, cos=cos, sin=sin, inverse=True)[1].to(device)
    size[..., :48] += x.double().abs().amax(2, keepdim=True)
    assert ((again.double() - x.double()).abs() <= 16 * 2.0 ** -24 * size).all()


def test_rotary_refuses(ops, device):
    x = _rows(4, 2, 16, torch.bfloat16, device)
    cos, sin = _tables(4, 8, device)
    with pytest.raises(TypeError):
        ops.rotary(x.double(), cos, sin)
    with pytest.raises(TypeError):
        ops.rotary(x, cos.double(), sin.double())
    with pytest.raises(ValueError):
        ops.rotary(x, cos[:3], sin[:3])  # a row for each token without positions
    with pytest.raises(ValueError):
        ops.rotary(x[0], cos, sin)
    with pytest.raises(ValueError):
        ops.rotary(x.transpose(1, 2), cos, sin)
    with pytest.raises(ValueError):
        ops.rotary(x[..., :14], cos, sin)  # 16 rotated of 14
    with pytest.raises(TypeError):
        ops.rotary(x, cos, sin, torch.zeros(4, device=device))
    with pytest.raises(ValueError):
        ops.rotary(x, cos, sin, torch.zeros(3, dtype=torch.int64, device=device))
    with pytest.raises(ValueError):
        ops.rotary(x, cos, sin, out=torch.empty(1, 2, 16, dtype=x.dtype, device=device).expand(4, 2, 16))
    with pytest.raises(TypeError):
        ops.rotary(x, cos, sin, out=torch.empty(4, 2, 16, device=device))
    with pytest.raises(RuntimeError):
        ops.rotary(x, cos.cpu(), sin)
    with pytest.raises(RuntimeError, match="even"):
        ops.rotary(_rows(4, 2, 17, torch.bfloat16, device), cos, sin)
    assert ops.rotary(x[:0], cos, sin).shape == (0, 2, 16)
    assert ops.rotary(x[:, :0], cos, sin).shape == (4, 0, 16)


# ------------------------------------------------------------- head norms

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [(1, 32, 8, 128, 128), (3, 1, 1, 2, 2), (37, 6, 2, 80, 32), (5, 4, 4, 36, 12),
                                                (130, 28, 28, 128, 64), (300, 33, 3, 96, 96), (2, 2, 1, 512, 128),
                                                (1200, 56, 8, 64, 64)])
def test_qk_norm_rotary(ops, device, tokens, hq, hk, d, rot, dtype, interleaved):
    kind = TYPES[dtype]
    qkv = _rows(tokens, hq + 2 * hk, d, kind, device, seed=tokens + d)
    q, k, _ = qkv.split((hq, hk, hk), dim=1)
    cos, sin = _tables(64, rot // 2, device)
    rows = torch.randint(0, 64, (tokens,), generator=_gen(d))
    w = lambda shape, seed: (1.0 + 0.3 * torch.randn(shape, generator=_gen(seed))).to(kind).to(device)
    weights = {"shared": (w((d,), 1), w((d,), 2)), "heads": (w((hq, d), 3), w((hk, d), 4)),
               "fp32": (w((d,), 5).float(), w((hk, d), 6).float()), "one": (w((d,), 7), None), "none": (None, None)}
    for name, (qw, kw) in weights.items():
        got = ops.qk_norm_rotary(q, k, qw, kw, cos, sin, rows.to(device), eps=1e-5, interleaved=interleaved)
        for x, weight, y in ((q, qw, got[0]), (k, kw, got[1])):
            few = slice(0, 40)  # the plain form goes row by row
            want, size = norm_rotate(x[few], weight, cos, sin, rows[few], eps=1e-5, interleaved=interleaved)
            assert_close(y[few], want, size, d, name)
            last = slice(max(0, tokens - 3), tokens)
            want, size = norm_rotate(x[last], weight, cos, sin, rows[last], eps=1e-5, interleaved=interleaved)
            assert_close(y[last], want, size, d, name)


def test_qk_norm_rotary_in_place_and_zero_rows(ops, device):
    qkv = _rows(50, 10, 128, torch.bfloat16, device)
    qkv[3] = 0.0  # a norm of nothing: x * 1 / sqrt(eps) = 0
    v = qkv[:, 8:].clone()
    cos, sin = _tables(50, 64, device)
    w = torch.ones(128, device=device, dtype=torch.bfloat16)
    want = ops.qk_norm_rotary(qkv[:, :6], qkv[:, 6:8], w, w, cos, sin)
    q, k = ops.qk_norm_rotary(qkv[:, :6], qkv[:, 6:8], w, w, cos, sin, q_out=qkv[:, :6], k_out=qkv[:, 6:8])
    assert torch.equal(qkv[:, :6], want[0]) and torch.equal(qkv[:, 6:8], want[1]) and torch.equal(qkv[:, 8:], v)
    assert (q[3] == 0).all() and (k[3] == 0).all()


def test_qk_norm_rotary_refuses(ops, device):
    q, k = _rows(4, 4, 16, torch.bfloat16, device), _rows(4, 2, 16, torch.bfloat16, device)
    cos, sin = _tables(4, 8, device)
    w = torch.ones(16, device=device, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        ops.qk_norm_rotary(q, k.half(), w, w, cos, sin)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, k[:3], w, w, cos, sin)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, k, w[:8], w, cos, sin)
    with pytest.raises(TypeError):
        ops.qk_norm_rotary(q, k, w.half(), w, cos, sin)
    with pytest.raises(TypeError):
        ops.qk_norm_rotary(q, k, w.float(), w, cos, sin)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, k, w, w.expand(3, 16), cos, sin)


# ------------------------------------------------------------------- plan

@pytest.mark.parametrize("seqs,page,pad,seed", [(1, 16, 0, 0), (7, 5, 3, 1), (300, 16, 1, 2), (40, 1, 0, 3), (3, 256, 9, 4)])
def test_plan_append(ops, device, seqs, page, pad, seed):
    gen = _gen(seed)
    new = torch.randint(0, 9, (seqs,), generator=gen)
    new[seqs // 2] = 0  # a sequence without tokens in this step
    lengths = torch.randint(0, 70, (seqs,), generator=gen).int()
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0))).int()
    tokens = int(cu[-1]) + pad
    columns = 78 // page  # the longest sequences outgrow it
    table = torch.randint(-1, 5000, (seqs, columns + 2), generator=gen).int().to(device)[:, :columns]
    got = ops.plan_append(table, lengths.to(device), cu.to(device), tokens, page)
    want = plan(table, lengths, cu, tokens, page)
    assert torch.equal(got.positions.cpu().long(), want[0]) and torch.equal(got.slots.cpu().long(), want[1])


@pytest.mark.parametrize("seqs", [255, 256, 1023, 1024, 1025, 3000])
def test_plan_append_of_many_sequences(ops, device, seqs):
    new = torch.randint(0, 3, (seqs,), generator=_gen(seqs))
    lengths = torch.randint(0, 60, (seqs,), generator=_gen(1)).int()
    cu = torch.cat((torch.tensor([2]), 2 + new.cumsum(0))).int()  # two tokens of no sequence before them
    tokens = int(cu[-1]) + 5
    table = torch.randperm(8 * seqs, generator=_gen(2)).int().view(seqs, 8)
    got = ops.plan_append(table.to(device), lengths.to(device), cu.to(device), tokens, 8)
    want = plan(table, lengths, cu, tokens, 8)
    assert torch.equal(got.positions.cpu().long(), want[0]) and torch.equal(got.slots.cpu().long(), want[1])


def test_plan_append_edges(ops, device):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    # slots of 2^31 and more, negative lengths, a first token that is padding
    got = ops.plan_append(i32(200_000_000, 3).view(2, 1), i32(0, -2), i32(1, 3, 5), 6, 16)
    assert got.positions.tolist() == [-1, 0, 1, -1, -1, -1] and got.slots.tolist() == [-1] * 6
    got = ops.plan_append(torch.empty(0, 4, dtype=torch.int32, device=device), i32(), i32(0), 3, 16)  # no sequences
    assert got.positions.tolist() == [-1] * 3 and got.slots.tolist() == [-1] * 3
    got = ops.plan_append(i32(5).view(1, 1), i32(2), i32(0, 0), 0, 16)
    assert got.positions.numel() == got.slots.numel() == 0
    with pytest.raises(TypeError):
        ops.plan_append(i32(5).view(1, 1).long(), i32(2), i32(0, 1), 1, 16)
    with pytest.raises(ValueError):
        ops.plan_append(i32(5).view(1, 1), i32(2, 3), i32(0, 1), 1, 16)
    with pytest.raises(ValueError):
        ops.plan_append(i32(5).view(1, 1), i32(2), i32(0, 1, 1), 1, 16)
    with pytest.raises(RuntimeError, match="page_size"):
        ops.plan_append(i32(5).view(1, 1), i32(2), i32(0, 1), 1, 0)
    with pytest.raises(ValueError):
        ops.plan_append(i32(5).view(1, 1), i32(2), i32(0, 1), -1, 16)


# ------------------------------------------------------------------ append

def _cache(pages, page, hk, d, dtype, layout, device, seed):
    shape = (pages, page, hk, d) if layout == "nhd" else (pages, hk, page, d)
    t = torch.randn(shape, generator=_gen(seed)).to(dtype).to(device)
    return t if layout == "nhd" else t.transpose(1, 2)


def _bits(t):
    return t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16 if t.element_size() == 2 else torch.int32)


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("kind", ["rows", "static", "one", "by_row"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,hq,hk,d,rot,page", [(1, 8, 2, 128, 128, 16), (45, 4, 4, 80, 32, 7), (33, 6, 1, 10, 4, 3),
                                                     (260, 28, 28, 128, 64, 64), (12, 3, 3, 64, 0, 16)])
def test_append_kv(ops, device, tokens, hq, hk, d, rot, page, dtype, kind, layout):
    kind_of = TYPES[dtype]
    qkv = _rows(tokens, hq + 2 * hk, d, kind_of, device, seed=tokens + d)
    q, k, v = qkv.split((hq, hk, hk), dim=1)
    pages = tokens // page + 3
    gen = _gen(tokens)
    slots = torch.randperm(pages * page, generator=gen)[:tokens].int()
    rows = torch.randint(0, 40, (tokens,), generator=gen)
    if tokens > 4:
        rows[tokens // 2], slots[tokens // 2] = -1, -1  # padding
        slots[3] = -1                                  # a token without a page: its q is made
        slots[4] = pages * page                        # and one past the cache
    cos, sin = _tables(40, rot // 2, device) if rot else (None, None)
    w = (1.0 + 0.3 * torch.randn(2, d, generator=gen)).to(kind_of).to(device)
    page_type = kind_of if kind == "rows" else torch.float8_e4m3fn
    caches = [_cache(pages, page, hk, d, page_type, layout, device, s) for s in (1, 2)]
    before = [c.clone() for c in caches]
    scales = [None, None]
    if kind in ("static", "one"):
        scales = [(torch.rand(hk if kind == "static" else 1, generator=gen) * 0.01 + 0.004).to(device) for _ in range(2)]
    elif kind == "by_row":
        scales = [torch.full((pages, page, hk), 7.0, device=device) for _ in range(2)]
    q_out = torch.full((tokens, hq, d), 3.0, device=device, dtype=kind_of)
    got = ops.append_kv(k, v, *caches, slots.to(device), k_scale=scales[0], v_scale=scales[1], k_weight=w[0], eps=1e-5,
                        cos=cos, sin=sin, positions=rows.to(device) if rot else None, q=q, q_weight=w[1], q_out=q_out)
    assert got.data_ptr() == q_out.data_ptr()
    live = (rows >= 0) if rot else torch.ones(tokens, dtype=torch.bool)
    want, size = norm_rotate(q, w[1], cos, sin, rows, eps=1e-5)
    assert_close(q_out[live.to(device)], want[live], size[live], d, "q")
    assert (q_out[~live.to(device)] == 3.0).all()
    stored = (slots >= 0) & (slots < pages * page) & live
    at = slots[stored].long()
    where = (at // page).to(device), (at % page).to(device)
    for i, (x, weight, turn) in enumerate(((k, w[0], cos), (v, None, None))):
        want, size = norm_rotate(x, weight, turn, None if turn is None else sin, rows, eps=1e-5)
        want, size = want[stored], size[stored]
        if kind == "rows":
            assert_close(caches[i][where], want, size, d, "kv"[i])
        else:
            by = scales[i].expand(len(at), hk) if kind != "by_row" else scales[i][where]
            if kind == "by_row":
                exact = want.abs().amax(2) / 448.0
                assert ((by.cpu().double() - exact).abs() <= ((32 + d / 8) * 2.0 ** -24) * size.amax(2) / 448.0 + 2e-24).all()
            assert_codes(caches[i][where], by.cpu()[:, :, None], want, size, d, "kv"[i])
        # everything else is as it was
        caches[i][where] = before[i][where]
        assert torch.equal(_bits(caches[i]), _bits(before[i]))
        if kind == "by_row":
            scales[i][where] = 7.0
            assert (scales[i] == 7.0).all()


def test_append_kv_values_alone_and_special_values(ops, device):
    """No norm, no rotation, no q: codes of rows with zeros, NaN, infinities and values past a static scale."""
    d = 64
    k = torch.zeros(6, 1, d, device=device, dtype=torch.bfloat16)
    k[1] = 1e-30
    k[2, 0, 5] = float("nan")
    k[3, 0, 5] = -float("inf")
    k[3, 0, 6] = 2.0
    k[4] = 1e30
    k[5, 0, :8] = torch.tensor([448.0, -448.0, 449.0, 464.0, 480.0, 1e4, -1e9, 0.0009765625], device=device).to(k.dtype)
    kp, vp = (torch.zeros(2, 4, 1, d, device=device, dtype=torch.float8_e4m3fn) for _ in range(2))
    ks, vs = torch.zeros(2, 4, 1, device=device), torch.ones(1, device=device)
    slots = torch.arange(6, device=device, dtype=torch.int32)
    assert ops.append_kv(k, k, kp, vp, slots, k_scale=ks, v_scale=vs) is None
    rows, flat, one = kp.float().view(8, d), ks.view(8), vp.float().view(8, d)
    assert (rows[0] == 0).all() and flat[0] == torch.tensor(1e-12)
    assert flat[1] == torch.tensor(1e-12) and (rows[1] == 0).all()
    assert torch.isnan(flat[2]) and torch.isnan(rows[2]).all()
    assert torch.isinf(flat[3]) and torch.isnan(rows[3, 5]) and (rows[3, [0, 6, 9]] == 0).all()
    assert (rows[4] == 448.0).all()
    assert one[5, :8].tolist() == [448.0, -448.0, 448.0, 448.0, 448.0, 448.0, -448.0, 0.0]  # 2^-10 is a tie to 0
    assert torch.isnan(one[2, 5]) and one[3, 5] == -448.0 and (one[4] == 448.0).all()
    assert (rows[6:] == 0).all() and (flat[6:] == 0).all()


def test_append_kv_past_32_bits(ops, device):
    """Slots whose elements lie past 2^32 of the cache."""
    page, hk, d = 64, 8, 128
    pages = (1 << 32) // (page * hk * d) + 40
    kp, vp = (torch.empty(pages, page, hk, d, device=device, dtype=torch.float8_e4m3fn) for _ in range(2))
    places = [0, 63, 64 * 32768 + 5, pages * page - 1, (pages - 3) * page]
    slots = torch.tensor(places, dtype=torch.int32, device=device)
    for cache in (kp, vp):
        flat = cache.view(torch.uint8).view(-1, hk, d)
        for s in places:
            flat[max(0, s - 1):s + 2] = 0x2A
    x = _rows(len(places), 2 * hk, d, torch.bfloat16, device)
    one = torch.ones(1, device=device) * 0.01
    ops.append_kv(x[:, :hk], x[:, hk:], kp, vp, slots, k_scale=one, v_scale=one)
    for cache, y in ((kp, x[:, :hk]), (vp, x[:, hk:])):
        flat = cache.view(-1, hk, d)
        for t, s in enumerate(places):
            assert_codes(flat[s][None], one[:, None, None], y[t:t + 1].double().cpu(), y[t:t + 1].abs().double().cpu(), d)
            for near in (s - 1, s + 1):
                if 0 <= near < pages * page and near not in places:
                    assert (flat[near].view(torch.uint8) == 0x2A).all()


def test_append_kv_refuses(ops, device):
    k = _rows(3, 2, 16, torch.bfloat16, device)
    kp, vp = (torch.zeros(2, 4, 2, 16, device=device, dtype=torch.bfloat16) for _ in range(2))
    e4 = kp.to(torch.float8_e4m3fn)
    slots = torch.arange(3, device=device, dtype=torch.int32)
    cos, sin = _tables(3, 4, device)
    with pytest.raises(TypeError):
        ops.append_kv(k, k, kp, vp, slots.long())
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp, slots[:2])
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp[:, :, :1], vp, slots)
    with pytest.raises(TypeError):
        ops.append_kv(k, k, kp.half(), vp, slots)
    with pytest.raises(TypeError):
        ops.append_kv(k, k, e4, vp, slots)  # codes without a scale
    with pytest.raises(ValueError):
        ops.append_kv(k, k, e4, vp, slots, k_scale=torch.ones(3, device=device))
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp, slots, k_scale=torch.ones(1, device=device))
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp[:1].expand(2, 4, 2, 16), vp, slots)  # pages that share memory
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp[:1], slots)  # not as many pages
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp.view(4, 2, 2, 16), slots)
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp, slots, cos=cos)
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp, slots, positions=slots)
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp, slots, q_out=k)
    with pytest.raises(ValueError):
        ops.append_kv(k, k[:, :1], kp, vp, slots)
    assert ops.append_kv(k[:0], k[:0], kp, vp, slots[:0]) is None
    empty = torch.zeros(0, 4, 2, 16, device=device, dtype=torch.bfloat16)
    assert ops.append_kv(k, k, empty, empty.clone(), slots) is None  # no pages: nothing is stored


def test_append_kv_refuses_shared_pages(ops, device):
    k = _rows(3, 2, 16, torch.bfloat16, device)
    pages = torch.zeros(2, 4, 2, 16, device=device, dtype=torch.bfloat16)
    slots = torch.arange(3, device=device, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.append_kv(k, k, pages, pages, slots)
    kp, vp = (torch.zeros(2, 4, 2, 16, device=device, dtype=torch.float8_e4m3fn) for _ in range(2))
    one, stored = torch.ones(2, device=device), torch.ones(2, 4, 2, device=device)
    with pytest.raises(ValueError):
        ops.append_kv(k, k, kp, vp, slots, k_scale=stored, v_scale=stored)
    ops.append_kv(k, k, kp, vp, slots, k_scale=one, v_scale=one)  # scales that are only read may be one tensor
    both = torch.zeros(2, 4, 4, 16, device=device, dtype=torch.bfloat16)
    ops.append_kv(k, 2 * k, both[:, :, :2], both[:, :, 2:], slots)  # and pages may be views of one
    assert torch.equal(both.flatten(0, 1)[:3], torch.cat((k, 2 * k), 1))


# ------------------------------------------- streams, graphs, the Python bodies

def _step(ops, device, seed=0):
    """Buffers of one decode step and a function that runs it."""
    hq, hk, d, page = 8, 2, 128, 16
    s = {"qkv": _rows(6, hq + 2 * hk, d, torch.bfloat16, device, seed=seed),
         "table": torch.randperm(40, generator=_gen(seed))[:20].int().view(5, 4).to(device),
         "lengths": torch.tensor([0, 15, 16, 40, 63], dtype=torch.int32, device=device),
         "cu": torch.arange(6, dtype=torch.int32, device=device),
         "kp": torch.zeros(40, page, hk, d, device=device, dtype=torch.float8_e4m3fn),
         "vp": torch.zeros(40, page, hk, d, device=device, dtype=torch.float8_e4m3fn),
         "ks": torch.zeros(40, page, hk, device=device), "vs": torch.zeros(40, page, hk, device=device),
         "w": torch.ones(d, device=device, dtype=torch.bfloat16),
         "q": torch.zeros(6, hq, d, device=device, dtype=torch.bfloat16)}
    s["cos"], s["sin"] = _tables(80, d // 2, device)

    def run(s=s):
        q, k, v = s["qkv"].split((hq, hk, hk), dim=1)
        plan = ops.plan_append(s["table"], s["lengths"], s["cu"], 6, page)
        ops.append_kv(k, v, s["kp"], s["vp"], plan.slots, k_scale=s["ks"], v_scale=s["vs"], k_weight=s["w"],
                      cos=s["cos"], sin=s["sin"], positions=plan.positions, q=q, q_weight=s["w"], q_out=s["q"])
        return s["q"]

    return s, run


_OUT = ("q", "kp", "vp", "ks", "vs")


def test_step_in_a_graph(ops, device):
    s, run = _step(ops, device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for replay in range(3):
        other, eager = _step(ops, device, seed=replay + 1)
        other["lengths"].add_(replay)
        for name in ("qkv", "table", "lengths"):
            s[name].copy_(other[name])
        for name in _OUT:
            s[name].zero_()
        eager()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in _OUT:
            assert torch.equal(s[name].float(), other[name].float()), name


def test_step_on_another_stream_equals_default(ops, device):
    s, run = _step(ops, device)
    other, again = _step(ops, device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    again()
    torch.cuda.synchronize()
    for name in _OUT:
        assert torch.equal(s[name].float(), other[name].float()), name


def test_python_bodies_equal_native(ops, device, monkeypatch):
    s, run = _step(ops, device)
    other, again = _step(ops, device)
    x = _rows(5, 3, 32, torch.float16, device)
    cos, sin = _tables(5, 8, device)
    positions = torch.arange(5, device=device)
    frequencies, _ = ops.rotary_frequencies(32, device=device)
    w = torch.ones(3, 32, device=device)
    calls = (lambda: ops.rotary(x, cos, sin, positions, interleaved=True, inverse=True),
             lambda: ops.qk_norm_rotary(x, x, w, None, cos, sin)[0], lambda: ops.rotary_tables(positions, frequencies)[1])
    run()
    native = [c() for c in calls]
    taken = []
    monkeypatch.setattr(ops, "_native_call", lambda name, *a: taken.append(name))
    again()
    for c, want in zip(calls, native):
        assert torch.equal(c(), want)
    assert set(taken) == {"plan_append", "append_kv", "rotary", "qk_norm_rotary", "rotary_tables"}
    for name in _OUT:
        assert torch.equal(s[name].float(), other[name].float()), name


# ------------------------------------- e4m3 pages: scales of rows, quotients

def _at(start, tokens, heads, d, dtype, device, seed):
    """[tokens, heads, d] whose first element lies ``start`` elements behind an aligned one."""
    wide = torch.empty(tokens * heads * d + start, device=device, dtype=dtype)
    rows = wide[start:].view(tokens, heads, d)
    return rows.copy_(torch.randn(tokens, heads, d, generator=_gen(seed)).to(dtype))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("start", [0, 1])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d,rot", [(80, 80), (96, 96), (192, 192), (10, 10), (36, 36), (510, 510), (128, 128), (192, 64)])
def test_append_kv_row_scales(ops, device, d, rot, dtype, start, interleaved):
    """Scales and codes of rows whose largest channel is one of the last pair's (or of a further pair), at an angle that
    makes it smaller; norms with a weight for each head.  Also the same keys in pages of their own type and with static
    scales, and the queries beside them."""
    tokens, hq, hk, page = 37, 3, 5, 8
    kind, half = TYPES[dtype], rot // 2
    q, k, v = (_at(start, tokens, h, d, kind, device, seed) for h, seed in ((hq, 1), (hk, 2), (hk, 3)))
    angle = torch.rand(50, half, generator=_gen(4), dtype=torch.float64) * 6.3
    rows = torch.randint(0, 50, (tokens,), generator=_gen(5))
    for t in range(tokens):
        pair = half - 1 if t % 3 else int(torch.randint(0, half, (1,), generator=_gen(t)))
        big, small = (2 * pair, 2 * pair + 1) if interleaved else (pair, half + pair)
        k[t, :, small], k[t, :, big] = 0.0, 30.0 if t % 2 else -30.0
        angle[rows[t], pair] = 0.7853981633974483  # the pair becomes (21, 21)
    cos, sin = angle.cos().float().to(device), angle.sin().float().to(device)
    weights = [(1.0 + 0.3 * torch.randn(h, d, generator=_gen(6))).to(kind).to(device) for h in (hq, hk)]
    pages = tokens // page + 2
    slots = torch.randperm(pages * page, generator=_gen(7))[:tokens]
    where = (slots // page).to(device), (slots % page).to(device)
    wanted = [norm_rotate(k, weights[1], cos, sin, rows, eps=1e-5, interleaved=interleaved), norm_rotate(v)]
    for form in ("by_row", "static", "rows"):
        caches = [_cache(pages, page, hk, d, kind if form == "rows" else torch.float8_e4m3fn, "nhd", device, s) for s in (8, 9)]
        scales = [None, None]
        if form == "static":
            scales = [torch.rand(hk, generator=_gen(10)).add(0.2).mul(0.05).to(device) for _ in range(2)]
        elif form == "by_row":
            scales = [torch.zeros(pages, page, hk, device=device) for _ in range(2)]
        got = ops.append_kv(k, v, *caches, slots.int().to(device), k_scale=scales[0], v_scale=scales[1], k_weight=weights[1],
                            eps=1e-5, cos=cos, sin=sin, positions=rows.to(device), interleaved=interleaved, q=q,
                            q_weight=weights[0])
        want, size = norm_rotate(q, weights[0], cos, sin, rows, eps=1e-5, interleaved=interleaved)
        assert_close(got, want, size, d, "q")
        for i, (want, size) in enumerate(wanted):
            if form == "rows":
                assert_close(caches[i][where], want, size, d, "kv"[i])
                continue
            by = scales[i][where] if form == "by_row" else scales[i].expand(tokens, hk)
            if form == "by_row":  # the product with RN(1 / 448): two roundings and the row's bound
                bound = ((32 + d / 8) * 2.0 ** -24) * size.amax(2) / 448.0 + 2e-24
                assert ((by.cpu().double() - want.abs().amax(2) / 448.0).abs() <= bound).all(), "kv"[i]
            assert_codes(caches[i][where], by.cpu()[:, :, None], want, size, d, "kv"[i])


@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_append_kv_codes_are_of_the_quotient(ops, device, dtype, by_row):
    """Codes are e4m3(clamp(RN(y / s))), as the other quantizers', bit for bit: rows without norm and rotation, many of
    their quotients halfway between two codes, where the product with RN(1 / s) is on either side."""
    kind, tokens, heads, d = TYPES[dtype], 64, 8, 128
    gen = _gen(11)
    odd = 2 * torch.randint(1, 16, (tokens if by_row else 1, heads, 1), generator=gen) + 1
    s = odd.float() * 2.0 ** -6
    # halfway between two codes: 17, 19 .. 31 sixteenths, times 2^0 .. 2^3, and (of few bits) 1, 3, 5, 7 times 2^-10;
    # a row's first channel is 448 s
    y = (2 * torch.randint(8, 16, (tokens, heads, d), generator=gen) + 1) / 16.0
    y = y * torch.exp2(torch.randint(0, 4, (tokens, heads, d), generator=gen).float())
    y[:, :, ::2] = (2 * torch.randint(0, 4, (tokens, heads, d // 2), generator=gen) + 1) * 2.0 ** -10
    y = y * s
    y = y * torch.where(torch.rand(tokens, heads, d, generator=gen) < 0.5, -1.0, 1.0)
    y[:, :, ::7] = 30.0 * torch.randn(y[:, :, ::7].shape, generator=gen) * s
    y[:, :, 1] = -0.0
    y[:, :, 0] = 448.0 * s[:, :, 0]
    rows = y.to(kind)
    value = rows.float()
    if by_row:
        s = (value.abs().amax(2, keepdim=True) * torch.tensor(1.0 / 448.0)).clamp(min=1e-12)
    quotient = (value / s).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    product = (value * (1.0 / s)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    assert (quotient.view(torch.uint8) != product.view(torch.uint8)).any()  # the inputs tell them apart
    caches = [torch.zeros(tokens // 16, 16, heads, d, device=device, dtype=torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(tokens // 16, 16, heads, device=device) if by_row else s.view(heads).to(device) for _ in range(2)]
    slots = torch.arange(tokens, dtype=torch.int32, device=device)
    x = rows.to(device)
    ops.append_kv(x, x, *caches, slots, k_scale=scales[0], v_scale=scales[1])
    for cache, scale in zip(caches, scales):
        if by_row:
            assert torch.equal(scale.view(tokens, heads, 1).cpu(), s)
        assert torch.equal(cache.view(tokens, heads, d).cpu().view(torch.uint8), quotient.view(torch.uint8))


def test_append_kv_static_scales_out_of_the_ordinary(ops, device):
    """Scales that have no binary32 reciprocal, 0, infinity and NaN: clamp(y / s) of IEEE division, NaN where that is."""
    s = torch.tensor([2.0 ** -140, 2.0 ** -149, 0.0, float("inf"), float("nan"), 2.0 ** 127, 1.0], dtype=torch.float32)
    heads, d = len(s), 16
    row = torch.tensor([0.0, -0.0, 1.0, -2.0, 2.0 ** -139, -(2.0 ** -140), 2.0 ** -133, 3e38, -1e38, float("inf"), -float("inf"),
                        float("nan"), 2.0 ** -149, 448.0, -449.0, 1e-12])
    x = row.expand(2, heads, d)
    want = (x / s[:, None]).clamp(-448.0, 448.0)
    caches = [torch.zeros(1, 2, heads, d, device=device, dtype=torch.float8_e4m3fn) for _ in range(2)]
    x, by = x.to(device), s.to(device)
    ops.append_kv(x, x, *caches, torch.arange(2, dtype=torch.int32, device=device), k_scale=by, v_scale=by)
    for cache in caches:
        got = cache[0].float().cpu()
        want_codes = want.to(torch.float8_e4m3fn).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7.0), want_codes.nan_to_num(7.0))


def test_outputs_that_are_another_rows_are_refused(ops, device):
    """An output may be its own input; one that starts where another output or the other input does is a race."""
    q, k = _rows(4, 2, 16, torch.bfloat16, device), _rows(4, 2, 16, torch.bfloat16, device, seed=2)
    cos, sin = _tables(4, 8, device)
    out = torch.zeros_like(q)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, k, None, None, cos, sin, q_out=out, k_out=out)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, k, None, None, cos, sin, q_out=k)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, k, None, None, cos, sin, k_out=q)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(q, k, None, None, cos, sin, q_out=k, k_out=q)
    pages = [torch.zeros(1, 4, 2, 16, device=device, dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.arange(4, device=device, dtype=torch.int32)
    for other in (k, out):
        with pytest.raises(ValueError):
            ops.append_kv(k, out, *pages, slots, cos=cos, sin=sin, q=q, q_out=other)
    want = ops.qk_norm_rotary(q, q, None, None, cos, sin)  # one input as both is read only
    assert torch.equal(want[0], want[1])
    got = ops.qk_norm_rotary(q.clone(), k, None, None, cos, sin, q_out=q)
    assert torch.equal(got[0], want[0]) and got[0].data_ptr() == q.data_ptr()


def test_out_as_x_in_other_strides_is_refused(ops, device):
    x = _rows(4, 4, 16, torch.bfloat16, device)
    cos, sin = _tables(4, 8, device)
    want = ops.rotary(x, cos, sin)
    with pytest.raises(RuntimeError, match="strides"):
        ops.rotary(x, cos, sin, out=x.transpose(0, 1))
    with pytest.raises(RuntimeError, match="strides"):
        ops.qk_norm_rotary(x, x.clone(), None, None, cos, sin, q_out=x.transpose(0, 1))
    assert torch.equal(ops.rotary(x, cos, sin, out=x), want)
    one, again = x[:1].clone(), ops.rotary(x[:1], cos, sin)
    assert torch.equal(ops.rotary(one, cos, sin, out=one.as_strided((1, 4, 16), (99, 16, 1))), again)


def test_more_tokens_than_a_grids_second_extent(ops, device):
    """65535 blocks of 32 tokens and some: the rest lies in the grid's third extent."""
    tokens, d = 65535 * 32 + 77, 8
    x = torch.randn(tokens, 2, d, generator=torch.Generator(device=device).manual_seed(1), device=device).to(torch.bfloat16)
    cos, sin = _tables(100, d // 2, device)
    rows = torch.arange(tokens, device=device) % 100
    rows[65535 * 32 + 5] = -1
    out = torch.zeros_like(x)
    ops.rotary(x, cos, sin, rows, out=out)
    pages = [torch.zeros(tokens // 16 + 1, 16, 2, d, device=device, dtype=x.dtype) for _ in range(2)]
    slots = torch.arange(tokens, dtype=torch.int32, device=device).flip(0).contiguous()
    ops.append_kv(x, x, *pages, slots, cos=cos, sin=sin, positions=rows)
    for part in (slice(0, 50), slice(65535 * 32 - 40, 65535 * 32 + 4), slice(65535 * 32 + 6, tokens)):
        want = ops.rotary(x[part], cos, sin, rows[part])
        assert torch.equal(out[part], want)
        at = slots[part].long()
        assert torch.equal(pages[0].flatten(0, 1)[at], want) and torch.equal(pages[1].flatten(0, 1)[at], x[part])
    assert (out[65535 * 32 + 5] == 0).all()
