"""Products with 4-bit weights on the GPU against the plain 64-bit form of _w4.py: every kernel, row count around its
tiles, group size, type, ragged widths, strides, splits, graphs."""

from __future__ import annotations

import pytest
import torch

from _util import activations
from _w4 import assert_product, packed_codes, packed_groups, product, quantize

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _weights(n, k, group, zeros, dtype, device, seed=0):
    """Codes over their whole range, scales of either sign, zero points: rows on the host and the packed form."""
    gen = torch.Generator().manual_seed(seed + n + k)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    scales = (torch.randn(n, groups, generator=gen) * k ** -0.5 * 0.25).to(dtype)
    points = torch.randint(0, 16, (n, groups), generator=gen, dtype=torch.uint8) if zeros else None
    return codes, scales, points


def _pack(ops, device, codes, scales, points, group):
    up = lambda t: None if t is None else t.to(device)
    return ops.pack_w4(up(codes), up(scales), up(points), group=group)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("m", [1, 13, 16, 17, 32, 33, 64, 65, 130, 200])
@pytest.mark.parametrize("n,k", [(48, 64), (201, 528), (1000, 1040)])
def test_w4_mm(ops, device, m, n, k, group, dtype, zeros):
    kind = TYPES[dtype]
    rows = _weights(n, k, group, zeros, kind, device)
    w = _pack(ops, device, *rows, group)
    x = activations(m, k, seed=m, outlier_channels=3).to(kind).to(device)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(kind).to(device) if m % 2 else None
    got = ops.w4_mm(x, w, bias=bias)
    assert got.shape == (m, n) and got.dtype == kind
    assert_product(got, *product(x, *rows, group, bias))


@pytest.mark.parametrize("m,n,k,group", [(1, 5376, 7168, 128), (5, 16, 14336, 128), (48, 256, 14336, 64),
                                         (100, 5376, 7168, 32), (700, 2048, 2048, 128), (2500, 1000, 512, 128),
                                         (1111, 5376, 1040, 64), (1, 1, 16, 32), (64, 1, 16, 32), (300, 17, 16, 128),
                                         (2048, 4096, 256, 32),
                                         # x of few rows in several chunks of LDS; two and four column blocks a workgroup
                                         (4, 40, 14336, 64), (1, 33, 23056, 128), (3, 4100, 9200, 32), (2, 12400, 256, 32),
                                         (12, 4112, 400, 32), (12, 8300, 400, 64), (31, 4112, 400, 32),
                                         (31, 8300, 400, 64), (31, 8300, 400, 32)])
def test_w4_mm_sizes(ops, device, m, n, k, group):
    rows = _weights(n, k, group, True, torch.bfloat16, device)
    w = _pack(ops, device, *rows, group)
    x = activations(m, k, seed=m).to(device)
    got = ops.w4_mm(x, w)
    assert_product(got, *product(x, *rows, group))
    again = ops.w4_mm(x, w)
    assert torch.equal(got, again)  # sums in a fixed order


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k,group", [(40, 8300, 1040, 32), (64, 9217, 144, 128), (70, 8300, 528, 128),
                                         (130, 12300, 400, 64), (33, 16500, 1040, 256), (129, 2070, 2320, 32),
                                         (600, 4096, 4096, 128), (17, 5000, 1040, 128), (18, 9000, 1040, 64),
                                         (32, 16500, 1040, 32), (25, 300, 9008, 128)])
def test_w4_mm_dozens_of_rows(ops, device, m, n, k, group, dtype, zeros):
    """Where a workgroup's waves split k: one to three column tiles of 32, ragged in rows, columns and k."""
    kind = TYPES[dtype]
    rows = _weights(n, k, group, zeros, kind, device)
    w = _pack(ops, device, *rows, group)
    x = activations(m, k, seed=m).to(kind).to(device)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(kind).to(device)
    got = ops.w4_mm(x, w, bias=bias)
    assert_product(got, *product(x, *rows, group, bias))
    assert torch.equal(ops.w4_mm(x, w, bias=bias), got)


@pytest.mark.parametrize("group", [32, 128, 384])
@pytest.mark.parametrize("m", [1, 20, 100, 1000])
def test_w4_mm_single_columns(ops, device, m, group):
    """x picks one column a row: every product is s (u - z), exact in both types."""
    n, k = 333, 464
    rows = _weights(n, k, group, True, torch.bfloat16, device)
    scales = torch.exp2(torch.randint(-8, 3, rows[1].shape, generator=torch.Generator().manual_seed(1)).float())
    rows = rows[0], scales.to(torch.bfloat16), rows[2]
    w = _pack(ops, device, *rows, group)
    x = torch.zeros(m, k, dtype=torch.bfloat16)
    at = torch.randperm(k, generator=torch.Generator().manual_seed(2)).repeat(3)[:m]
    x[torch.arange(m), at] = 1.0
    want, _ = product(x, *rows, group)
    assert torch.equal(ops.w4_mm(x.to(device), w).cpu().double(), want)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(20, 99, 272), (40, 8300, 1040), (33, 16500, 1040), (64, 64, 9232), (2048, 4096, 144)])
def test_w4_mm_scales_of_the_other_type(ops, device, m, n, k, dtype, zeros):
    kind = TYPES[dtype]
    rows = _weights(n, k, 32, zeros, torch.float16 if kind == torch.bfloat16 else torch.bfloat16, device)
    x = activations(m, k, seed=m).to(kind).to(device)
    assert_product(ops.w4_mm(x, _pack(ops, device, *rows, 32)), *product(x, *rows, 32))


@pytest.mark.parametrize("m", [7, 40, 900])
def test_w4_mm_strides_and_scale_types(ops, device, m):
    """Rows of wider x and out, an unaligned out and bias, scales of the other type; the rest of out is left."""
    n, k, group = 99, 272, 64
    rows = _weights(n, k, group, True, torch.float16, device)
    w = _pack(ops, device, *rows, group)
    wide = activations(m, k + 24, seed=m).to(device)
    x = wide[:, 8:8 + k]
    bias = torch.randn(n + 1, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(device)[1:]
    whole = torch.full((m + 1, n + 7), 5.0, device=device, dtype=torch.bfloat16)
    out = whole[:m, 3:3 + n]
    assert ops.w4_mm(x, w, bias=bias, out=out).data_ptr() == out.data_ptr()
    assert_product(out, *product(x, *rows, group, bias))
    assert (whole[:, :3] == 5.0).all() and (whole[:, 3 + n:] == 5.0).all() and (whole[m] == 5.0).all()


@pytest.mark.parametrize("m", [3, 150])
def test_w4_mm_other_rows_of_x_do_not_reach_a_row(ops, device, m):
    """Infinities and NaN in one row of x, and in the columns behind k of a wider x, stay there."""
    n, k, group = 64, 208, 32
    rows = _weights(n, k, group, False, torch.bfloat16, device)
    w = _pack(ops, device, *rows, group)
    wide = activations(m, k + 16, seed=m).to(device)
    clean = ops.w4_mm(wide[:, :k], w)
    wide[:, k:] = float("nan")
    wide[1, 5], wide[1, 100] = float("inf"), float("nan")
    got = ops.w4_mm(wide[:, :k], w)
    others = [i for i in range(m) if i != 1]
    assert torch.equal(got[others], clean[others]) and not torch.isfinite(got[1]).any()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", [(1, 16, 32), (37, 208, 32), (16, 1024, 128), (70, 400, 256), (5, 96, 64)])
def test_pack_and_quantize(ops, device, n, k, group, zeros):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        w = torch.randn(n, k, generator=torch.Generator().manual_seed(n + k)).to(dtype)
        w[n // 2, :16] = 0.0
        want = quantize(w, group, zeros)
        got = ops.quantize_w4(w.to(device), group, zeros=zeros)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1]) and got[1].dtype == want[1].dtype
        assert (got[2] is None) == (not zeros) and (not zeros or torch.equal(got[2].cpu(), want[2]))
        packed = ops.pack_w4(*got, group=group)
        assert torch.equal(packed.codes.cpu(), packed_codes(want[0]))
        assert torch.equal(packed.scales.cpu(), packed_groups(want[1]))
        assert (packed.zeros is None) == (not zeros)
        assert not zeros or torch.equal(packed.zeros.cpu(), packed_groups(want[2]))


def test_quantize_and_pack_of_strided_rows(ops, device):
    w = torch.randn(20, 200, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(device)
    want = ops.quantize_w4(w[:, 3:163].contiguous(), 32, zeros=True)
    got = ops.quantize_w4(w[:, 3:163], 32, zeros=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    wide = [torch.cat((t, t), dim=1) for t in want]
    sliced = [t[:, :t.shape[1] // 2] for t in wide]
    for a, b in zip(ops.pack_w4(*sliced, group=32)[:3], ops.pack_w4(*want, group=32)[:3]):
        assert torch.equal(a, b)


def test_w4_refuses(ops, device):
    rows = _weights(32, 256, 32, True, torch.bfloat16, device)
    w = _pack(ops, device, *rows, 32)
    x = activations(4, 256).to(device)
    with pytest.raises(TypeError):
        ops.w4_mm(x.float(), w)
    with pytest.raises(ValueError):
        ops.w4_mm(x[:, :48], w)
    with pytest.raises(ValueError):
        ops.w4_mm(x[0], w)
    with pytest.raises(RuntimeError, match="ldx"):
        ops.w4_mm(torch.zeros(4, 260, device=device, dtype=x.dtype)[:, :256], w)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.w4_mm(torch.zeros(4, 264, device=device, dtype=x.dtype)[:, 4:260], w)
    with pytest.raises(TypeError):
        ops.w4_mm(x, w, bias=torch.zeros(32, device=device))
    with pytest.raises(ValueError):
        ops.w4_mm(x, w, bias=torch.zeros(31, device=device, dtype=x.dtype))
    with pytest.raises(ValueError):
        ops.w4_mm(x, w, out=torch.zeros(4, 31, device=device, dtype=x.dtype))
    with pytest.raises(ValueError):
        ops.w4_mm(x, w, out=torch.zeros(1, 32, device=device, dtype=x.dtype).expand(4, 32))
    with pytest.raises(ValueError):
        ops.w4_mm(x, w._replace(group=64))
    with pytest.raises(ValueError):
        ops.w4_mm(x, w._replace(n=33))
    with pytest.raises(TypeError):
        ops.w4_mm(x, w._replace(scales=w.scales.float()))
    with pytest.raises(RuntimeError):
        ops.w4_mm(x, w._replace(codes=w.codes.cpu()))
    codes, scales, points = (t.to(device) for t in rows)
    with pytest.raises(ValueError):
        ops.pack_w4(codes, scales, points, group=64)
    with pytest.raises(ValueError):
        ops.pack_w4(codes, scales, points, group=48)
    with pytest.raises(TypeError):
        ops.pack_w4(codes, scales.float(), points, group=32)
    with pytest.raises(TypeError):
        ops.pack_w4(codes.int(), scales, points, group=32)
    with pytest.raises(ValueError):
        ops.quantize_w4(x[:, :40])
    with pytest.raises(TypeError):
        ops.quantize_w4(x.double())
    assert ops.w4_mm(x[:0], w).shape == (0, 32)


def test_w4_mm_in_a_graph_and_on_a_stream(ops, device):
    """Captured once over the three kinds of call (their workspaces are the graph's own), replayed with new
    inputs and eager work between; and eager on another stream."""
    rows = _weights(1000, 1040, 64, True, torch.bfloat16, device)
    w = _pack(ops, device, *rows, 64)
    xs = [activations(m, 1040, seed=m).to(device) for m in (3, 90, 1500)]
    outs = [torch.empty(x.shape[0], 1000, device=device, dtype=x.dtype) for x in xs]

    def run():
        for x, out in zip(xs, outs):
            ops.w4_mm(x, w, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, out in zip(xs, outs):
        assert torch.equal(out, ops.w4_mm(x, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for replay in range(3):
        for x in xs:
            x.copy_(activations(x.shape[0], 1040, seed=50 + replay).to(device))
        want = [ops.w4_mm(x, w) for x in xs]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for out, y in zip(outs, want):
            assert torch.equal(out, y)


def test_w4_python_body_equals_native(ops, device, monkeypatch):
    rows = _weights(200, 528, 32, True, torch.float16, device)
    w = _pack(ops, device, *rows, 32)
    xs = [activations(m, 528, seed=m).half().to(device) for m in (1, 70)]
    bias = torch.ones(200, device=device, dtype=torch.float16)
    want = [ops.w4_mm(x, w, bias=bias) for x in xs]
    taken = []
    monkeypatch.setattr(ops, "_native_call", lambda name, *a: taken.append(name))
    for x, y in zip(xs, want):
        assert torch.equal(ops.w4_mm(x, w, bias=bias), y)
    assert taken == ["w4_mm", "w4_mm"]


def test_w4_split_sums_of_two_graphs(ops, device):
    """Long rows and few tiles: k in parts, whose sums lie in a workspace of each captured call's own."""
    n, k = 256, 14336
    rows = _weights(n, k, 128, True, torch.bfloat16, device)
    w = _pack(ops, device, *rows, 128)
    xs = [activations(m, k, seed=m).to(device) for m in (48, 100)]
    outs = [torch.empty(x.shape[0], n, device=device, dtype=x.dtype) for x in xs]
    graphs = []
    for x, out in zip(xs, outs):
        assert_product(ops.w4_mm(x, w), *product(x, *rows, 128))
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.w4_mm(x, w, out=out)
    side = torch.cuda.Stream()
    for replay in range(3):
        for x in xs:
            x.copy_(activations(x.shape[0], k, seed=70 + replay).to(device))
        want = [ops.w4_mm(x, w) for x in xs]
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for out, y in zip(outs, want):
            assert torch.equal(out, y)


def _picked(n, k, group, cols, x, device, seed=3):
    """Weights with exact values and an x whose row r holds 2^-3 in column cols[r % len(cols)], and the result: the weights
    there (exact in both kinds of kernel)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, device=device, dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-6, 3, (n, groups), generator=gen, device=device).float()).to(torch.bfloat16)
    points = torch.randint(0, 16, (n, groups), generator=gen, device=device, dtype=torch.uint8)
    at = torch.tensor(cols, device=device)[torch.arange(x.shape[0], device=device) % len(cols)]
    x[torch.arange(x.shape[0], device=device), at] = 0.125
    u = codes[:, at // 2].int() >> (4 * (at % 2)) & 15
    g = at // group
    return (codes, scales, points), ((u - points[:, g].int()).float() * scales[:, g].float() * 0.125).t().to(torch.bfloat16)


@pytest.mark.parametrize("group", [32, 1 << 18])
def test_w4_mm_longest_rows(ops, device, group):
    n, k = 19, 1 << 22
    for m in (1, 5, 20, 40):
        x = torch.zeros(m, k, device=device, dtype=torch.bfloat16)
        cols = [k - 1, 0, k // 2 + 77, 3 * 128 + 31, k - 4097] if m > 1 else [k - 1]
        rows, want = _picked(n, k, group, cols, x, device)
        assert torch.equal(ops.w4_mm(x, ops.pack_w4(*rows, group=group)), want)


@pytest.mark.parametrize("m,ldx,n,k", [(130, (1 << 23) - 8, 48, 208), (3, (1 << 23) - 8, 48, 208), (33, (1 << 23) - 8, 48, 208),
                                       (140001, 16400, 17, 80), (40, 4096, (1 << 20) + 5, 144), (2, 4096, (1 << 20) + 5, 144),
                                       (70001, 64, 32771, 48)])
def test_w4_mm_far_rows_and_columns(ops, device, m, ldx, n, k):
    """The widest row stride, and x and out past 4 GiB."""
    x = torch.zeros(m, ldx, device=device, dtype=torch.bfloat16)[:, :k]
    rows, want = _picked(n, k, 32, [k - 1, 5, k // 2], x, device)
    assert torch.equal(ops.w4_mm(x, ops.pack_w4(*rows, group=32)), want)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_keeps_nan_and_infinities(ops, device, dtype, zeros):
    """A NaN weight makes its group's scale NaN, an infinity one that is not finite: such a group's products are not
    finite either, and every other group is what it was."""
    n, k, group = 21, 208, 32
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(1)).to(dtype)
    clean = quantize(w, group, zeros)
    for place, value in (((0, 0), float("nan")), ((5, 63), float("nan")), ((20, 207), float("nan")), ((7, 100), float("inf")),
                         ((8, 100), -float("inf"))):
        w[place] = value
    got = [None if t is None else t.cpu() for t in ops.quantize_w4(w.to(device), group, zeros=zeros)]
    odd = torch.zeros(n, 7, dtype=torch.bool)
    for r, g in ((0, 0), (5, 1), (20, 6), (7, 3), (8, 3)):
        odd[r, g] = True
    assert torch.equal(~torch.isfinite(got[1]), odd)
    assert torch.isnan(got[1][0, 0]) and torch.isnan(got[1][5, 1]) and torch.isnan(got[1][20, 6])
    columns = ~odd.repeat_interleave(group // 2, dim=1)[:, :k // 2]
    assert torch.equal(got[0][columns], clean[0][columns]) and torch.equal(got[1][~odd], clean[1][~odd])
    assert not zeros or torch.equal(got[2][~odd], clean[2][~odd])
    packed = ops.pack_w4(*(None if t is None else t.to(device) for t in got), group=group)
    for m in (1, 9, 30, 300):
        x = activations(m, k, seed=m).to(torch.float16 if dtype == torch.float16 else torch.bfloat16).to(device)
        finite = torch.isfinite(ops.w4_mm(x, packed).cpu())
        assert torch.equal(finite, (~odd.any(1)).expand(m, n))


def test_quantize_more_groups_than_a_launch_has_threads(ops, device):
    """2^28 and some groups, 16 lanes each: past 2^32 threads."""
    n, k, group = (1 << 16) + 1, 1 << 17, 32
    w = torch.zeros(n, k, device=device, dtype=torch.bfloat16)
    at = [0, 1, 777, n // 2, n - 2, n - 1]
    w[at] = torch.randn(len(at), k, generator=torch.Generator(device=device).manual_seed(1), device=device).to(w.dtype)
    codes, scales, _ = ops.quantize_w4(w, group)
    want = quantize(w[at].cpu(), group, False)
    assert torch.equal(codes[at].cpu(), want[0]) and torch.equal(scales[at].cpu(), want[1])
    assert (codes[2:700] == 0x88).all() and (scales[n - 1000:n - 2] == 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m", [1, 3, 4, 16])
def test_w4_mm_of_few_rows_takes_weights_as_they_are(ops, device, m, dtype):
    """x has +1 in one column and -1 in one of another group: s (u - z) - s' (u' - z') of weights that cancel to a few of
    their last bits.  Every step of the kernel is exact for them (u, z and 8-bit or 11-bit scales: products below 2^24
    steps), so the result is the exact difference, rounded once; weights rounded first miss it by whole steps."""
    kind = TYPES[dtype]
    n, k, group = 40, 128, 32
    gen = torch.Generator().manual_seed(7)
    bits = 8 if dtype == "bf16" else 11
    codes = torch.randint(0, 16, (n, k), generator=gen)
    points = torch.randint(0, 4, (n, 4), generator=gen)
    codes[:, 5], codes[:, 37] = points[:, 0] + 11, points[:, 1] + 12
    # 11 s near 12 s'
    s = torch.randint(1 << (bits - 1), 1 << bits, (n, 4), generator=gen).float()
    s[:, 0] = torch.randint(round(0.75 * 2 ** bits), 1 << bits, (n,), generator=gen).float()
    s[:, 1] = (s[:, 0] * 11 / 12).round()
    scales = (s * 2.0 ** -12).to(kind)
    assert torch.equal(scales.float(), s * 2.0 ** -12)
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8), scales, points.to(torch.uint8)
    x = torch.zeros(m, k)
    x[:, 5], x[:, 37] = 1.0, -1.0
    got = ops.w4_mm(x.to(kind).to(device), _pack(ops, device, *packed, group)).cpu()
    want = (11 * s[:, 0] - 12 * s[:, 1]) * 2.0 ** -12
    rounded = (11 * s[:, 0] * 2.0 ** -12).to(kind).float() - (12 * s[:, 1] * 2.0 ** -12).to(kind).float()
    assert (want.to(kind) != rounded.to(kind)).any()  # the inputs tell them apart
    assert torch.equal(got, want.to(kind).expand(m, n))


@pytest.mark.parametrize("scale_type", list(TYPES))
@pytest.mark.parametrize("m", [2, 16, 17, 40, 300, 2048])
def test_w4_mm_binary16_weights_below_its_normal_range(ops, device, m, scale_type):
    """Above 16 rows weights are rounded to binary16, below 2^-14 to its subnormal steps and not to zero; up to 16 rows
    bf16 scales stay as they are."""
    n, k, group = 272, 208, 32
    rows = _weights(n, k, group, True, TYPES[scale_type], device)
    scales = (rows[1].float() * 2.0 ** -10).to(TYPES[scale_type])
    x = (activations(m, k, seed=m).float() * 64.0).half().to(device)
    got = ops.w4_mm(x, _pack(ops, device, rows[0], scales, rows[2], group))
    assert_product(got, *product(x, rows[0], scales, rows[2], group))
    assert (got != 0).float().mean() > 0.9
