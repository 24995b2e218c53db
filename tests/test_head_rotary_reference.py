"""CPU tests of the rotary operators: the plain forms that the GPU tests compare with, the frequencies, and
what the entry points refuse before any launch."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from _heads import assert_close, norm_rotate, plan


def _tables(rows: int, pairs: int, seed: int = 0):
    angle = torch.rand(rows, pairs, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 6.0
    return angle.cos().float(), angle.sin().float(), angle


@pytest.mark.parametrize("interleaved", [False, True])
def test_plain_rotation_is_a_complex_product(interleaved):
    x = torch.randn(5, 3, 12, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    cos, sin, _ = _tables(9, 4)
    rows = [8, 0, 3, 3, 7]
    got, size = norm_rotate(x, cos=cos, sin=sin, rows=rows, interleaved=interleaved)
    a, b = (x[..., 0:8:2], x[..., 1:8:2]) if interleaved else (x[..., :4], x[..., 4:8])
    z = torch.complex(a, b) * torch.complex(cos[rows].double(), sin[rows].double())[:, None]
    ga, gb = (got[..., 0:8:2], got[..., 1:8:2]) if interleaved else (got[..., :4], got[..., 4:8])
    assert torch.allclose(torch.complex(ga, gb), z, rtol=1e-14, atol=1e-14)
    assert torch.equal(got[..., 8:], x[..., 8:]) and (size >= got.abs() - 1e-12).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_rotation_is_the_gradient(interleaved):
    """d(sum g . R x) / dx is the rotation of g by the negative angle: against autograd's of the formula and
    against differences (the map is linear: a difference of any step is exact to rounding)."""
    x = torch.randn(4, 2, 8, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    g = torch.randn(4, 2, 8, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    cos, sin, _ = _tables(4, 3, seed=4)
    want, _ = norm_rotate(g, cos=cos, sin=sin, interleaved=interleaved, inverse=True)
    leaf = x.clone().requires_grad_()
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (leaf[..., 0:6:2], leaf[..., 1:6:2]) if interleaved else (leaf[..., :3], leaf[..., 3:6])
    ga, gb = (g[..., 0:6:2], g[..., 1:6:2]) if interleaved else (g[..., :3], g[..., 3:6])
    ((a * c - b * s) * ga + (a * s + b * c) * gb).sum().add((leaf[..., 6:] * g[..., 6:]).sum()).backward()
    assert torch.allclose(leaf.grad, want, rtol=1e-13, atol=1e-13)
    value = lambda at: (norm_rotate(at, cos=cos, sin=sin, interleaved=interleaved)[0] * g).sum()
    for i in (0, 5, 7):
        step = torch.zeros_like(x)
        step[2, 1, i] = 0.5
        assert math.isclose(float(value(x + step) - value(x - step)), float(want[2, 1, i]), rel_tol=1e-11, abs_tol=1e-11)


def test_plain_plan():
    table = torch.tensor([[4, 2, -1], [0, 1, 3]])
    positions, slots = plan(table, torch.tensor([3, 0]), torch.tensor([0, 3, 4]), 6, 4)
    assert positions.tolist() == [3, 4, 5, 0, -1, -1]
    assert slots.tolist() == [4 * 4 + 3, 2 * 4, 2 * 4 + 1, 0, -1, -1]


def test_assert_close_notices_a_step():
    x = torch.randn(2, 2, 8, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    good = x.to(torch.bfloat16)
    assert_close(good, x, x.abs(), 8)
    with pytest.raises(AssertionError):
        assert_close(good * 1.02, x, x.abs(), 8)


# ------------------------------------------------------------- frequencies

def test_frequencies_without_scaling(ops):
    f, magnitude = ops.rotary_frequencies(8, 100.0, device="cpu")
    assert magnitude == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], dtype=torch.float64), rtol=1e-15)


def test_frequencies_scaled(ops):
    plain, _ = ops.rotary_frequencies(64, device="cpu")
    linear, m = ops.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert m == 1.0 and torch.equal(linear, plain / 4.0)
    base, m = ops.rotary_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert m == 1.0 and base[0] == 1.0 and math.isclose(base[-1], plain[-1] / 4.0, rel_tol=1e-12)
    assert (base[1:-1] < plain[1:-1]).all() and (base[1:-1] > linear[1:-1]).all()
    yarn, m = ops.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    assert math.isclose(m, 0.1 * math.log(8.0) + 1.0)
    turns = 4096 * plain / (2.0 * math.pi)
    assert torch.equal(yarn[turns > 48.0], plain[turns > 48.0])
    assert torch.allclose(yarn[turns < 0.7], plain[turns < 0.7] / 8.0, rtol=1e-14)
    assert (yarn.diff() < 0).all()
    bands, m = ops.rotary_frequencies(64, 500000.0, scaling="bands", factor=8.0, original_length=8192, device="cpu")
    plain, _ = ops.rotary_frequencies(64, 500000.0, device="cpu")
    length = 2.0 * math.pi / plain
    assert m == 1.0 and torch.equal(bands[length < 8192 / 4.0], plain[length < 8192 / 4.0])
    assert torch.equal(bands[length > 8192.0], plain[length > 8192.0] / 8.0)
    assert (bands <= plain).all() and (bands >= plain / 8.0).all()


@pytest.mark.parametrize("kwargs", [dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=514), dict(rot_dim=8, base=-1.0),
                                    dict(rot_dim=8, scaling="yarn", factor=2.0), dict(rot_dim=8, scaling="other"),
                                    dict(rot_dim=2, scaling="base", factor=2.0), dict(rot_dim=8, factor=0.0),
                                    dict(rot_dim=8, scaling="bands", original_length=64, low=4.0, high=4.0)])
def test_frequencies_refuse(ops, kwargs):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(device="cpu", **kwargs)


# ---------------------------------------------------------------- refusals

def test_wrappers_refuse_cpu_tensors(ops):
    x = torch.zeros(2, 2, 8, dtype=torch.bfloat16)
    cos = sin = torch.zeros(2, 4)
    ids = torch.zeros(2, dtype=torch.int32)
    pages = torch.zeros(2, 4, 2, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.rotary(x, cos, sin), lambda: ops.qk_norm_rotary(x, x, None, None, cos, sin),
                 lambda: ops.rotary_tables(ids, torch.ones(4, dtype=torch.float64)),
                 lambda: ops.plan_append(ids.view(2, 1), ids, torch.zeros(3, dtype=torch.int32), 2, 4),
                 lambda: ops.append_kv(x, x, pages, pages.clone(), ids)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


@pytest.fixture(scope="module")
def lib():
    from taomate_h3_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    return _lib


def _rows(lib, heads=2, weight=None):
    return lib.Heads(256, 16, 8, heads, weight, 0, 256, 16, 8)


def _turn(lib, rows=4, rot=8, positions=256):
    return lib.Rotation(256, 256, rows, rot, positions, 0, 0, 0)


def _pages(lib, **kw):
    fields = dict(pages=256, n_pages=4, page_size=16, page_stride=256, slot_stride=16, head_stride=8, kind=0, scale=None)
    return lib.Pages(**{**fields, **kw})


def test_c_entry_points_refuse(lib):
    """On the host, before any launch (there is no GPU here)."""
    handle = lib.lib()
    error = lambda: handle.h3q_last_error().decode()
    p = ctypes.c_void_p(256)
    x, turn = _rows(lib), _turn(lib)
    assert handle.h3q_rotary(3, x, 4, 8, turn, None) == 1 and "unknown dtype" in error()
    assert handle.h3q_rotary(0, x, 4, 9, turn, None) == 2 and "even" in error()
    assert handle.h3q_rotary(0, x, 4, 514, turn, None) == 2 and "512" in error()
    assert handle.h3q_rotary(0, x, 4, 6, turn, None) == 1 and "rotated channels" in error()
    assert handle.h3q_rotary(0, x, 4, 8, _turn(lib, rot=7), None) == 1 and "rotated channels" in error()
    assert handle.h3q_rotary(0, x, 5, 8, _turn(lib, positions=None), None) == 1 and "without positions" in error()
    assert handle.h3q_rotary(0, x, 5, 8, _turn(lib, rows=0), None) == 1 and "without rows" in error()
    assert handle.h3q_rotary(0, _rows(lib, weight=256), 4, 8, turn, None) == 1 and "without a norm" in error()
    assert handle.h3q_rotary(0, _rows(lib, heads=16385), 4, 8, turn, None) == 1 and "heads" in error()
    assert handle.h3q_rotary(2, lib.Heads(258, 16, 8, 2, None, 0, 256, 16, 8), 4, 8, turn, None) == 1 and "aligned" in error()
    assert handle.h3q_rotary(0, x, 1 << 31, 8, turn, None) == 1 and "tokens" in error()
    assert handle.h3q_rotary(0, None, 4, 8, turn, None) == 1 and "null" in error()
    assert handle.h3q_rotary(0, x, 0, 8, turn, None) == 0
    f = ctypes.c_float(1e-6)
    assert handle.h3q_qk_norm_rotary(0, 1, x, x, 4, 8, f, turn, None) == 1 and "weights" in error()
    assert handle.h3q_qk_norm_rotary(0, 2, x, lib.Heads(), 4, 8, f, None, None) == 1 and "null" in error()
    assert handle.h3q_qk_norm_rotary(0, 2, lib.Heads(), lib.Heads(), 4, 8, f, turn, None) == 0  # no heads
    assert handle.h3q_rotary_tables(p, 4, 4, p, 8, 1.0, p, p, None) == 1 and "type of positions" in error()
    assert handle.h3q_rotary_tables(p, 0, 1 << 24, p, 128, 1.0, p, p, None) == 2 and "2^31" in error()
    assert handle.h3q_rotary_tables(p, 0, 4, p, 257, 1.0, p, p, None) == 1
    assert handle.h3q_rotary_tables(None, 0, 4, p, 8, 1.0, p, p, None) == 1 and "null" in error()
    assert handle.h3q_rotary_tables(p, 0, 0, p, 8, 1.0, p, p, None) == 0
    assert handle.h3q_plan_append(p, 3, 2, 4, p, p, 4, 16, p, p, None) == 1 and "between rows" in error()
    assert handle.h3q_plan_append(p, 4, 2, 4, p, p, 4, 0, p, p, None) == 1 and "page_size" in error()
    assert handle.h3q_plan_append(p, 4, 2, 4, None, p, 4, 16, p, p, None) == 1 and "null" in error()
    assert handle.h3q_plan_append(p, 4, 2, 4, p, p, 0, 16, p, p, None) == 0

    def append(q=None, k=x, v=x, kp=None, vp=None, slots=p, tokens=4, d=8, turn=turn, wt=0):
        return handle.h3q_append_kv(0, wt, q, k, v, kp or _pages(lib), vp or _pages(lib), slots, tokens, d, f, turn, None)

    assert append(kp=_pages(lib, kind=3)) == 1 and "kind" in error()
    assert append(kp=_pages(lib, kind=1)) == 1 and "need scales" in error()
    assert append(vp=_pages(lib, n_pages=1 << 27)) == 2 and "2^31" in error()
    assert append(vp=_pages(lib, page_size=0)) == 2
    assert append(vp=_pages(lib, n_pages=5)) == 1 and "v pages" in error()
    assert append(v=_rows(lib, heads=3)) == 1 and "v heads" in error()
    assert append(v=_rows(lib, weight=256)) == 1 and "no norm" in error()
    assert append(slots=None) == 1 and "slots" in error()
    assert append(turn=_turn(lib, rot=10)) == 1 and "rotated" in error()
    assert append(q=lib.Heads(256, 16, 8, 2, None, 0, None, 0, 0)) == 1 and "null q" in error()
    assert append(tokens=0) == 0


def test_c_entry_points_refuse_outputs_in_other_rows(lib):
    handle = lib.lib()
    error = lambda: handle.h3q_last_error().decode()
    rows = lambda x, out, heads=2: lib.Heads(x, 16, 8, heads, None, 0, out, 16, 8)
    p, f = ctypes.c_void_p(256), ctypes.c_float(1e-6)
    norm = lambda q, k, tokens=4: handle.h3q_qk_norm_rotary(0, 0, q, k, tokens, 8, f, _turn(lib), None)
    for q, k in ((rows(256, 1024), rows(512, 1024)), (rows(256, 512), rows(512, 1024)), (rows(256, 1024), rows(512, 256)),
                 (rows(256, 512), rows(512, 256))):
        assert norm(q, k) == 1 and "other rows" in error()
        assert norm(q, k, 0) == 0  # no rows
    append = lambda q, k, v: handle.h3q_append_kv(0, 0, q, k, v, _pages(lib), _pages(lib, pages=4096), p, 4, 8, f, None, None)
    for out in (512, 1024):
        assert append(rows(256, out), rows(512, None), rows(1024, None)) == 1 and "k or v" in error()


def test_c_entry_points_refuse_out_as_x_in_other_strides(lib):
    """Rows that lie where others are still read; strides of one token or head do not count."""
    handle = lib.lib()
    p, f = ctypes.c_void_p(256), ctypes.c_float(1e-6)
    rows = lambda token, head, out_token, out_head, heads=2: lib.Heads(256, token, head, heads, None, 0, 256, out_token, out_head)
    good = lib.Heads(1024, 16, 8, 2, None, 0, 2048, 16, 8)
    for bad in (rows(16, 8, 8, 32), rows(16, 8, 16, 32), rows(16, 8, 32, 8), rows(16, 8, 32, 8, heads=1)):
        assert handle.h3q_rotary(0, bad, 4, 8, _turn(lib), None) == 1
        assert "strides" in handle.h3q_last_error().decode()
        for q, k in ((bad, good), (good, bad)):
            assert handle.h3q_qk_norm_rotary(0, 0, q, k, 4, 8, f, _turn(lib), None) == 1
        assert handle.h3q_append_kv(0, 0, bad, good, lib.Heads(4096, 16, 8, 2), _pages(lib), _pages(lib), p, 4, 8, f, None, None) == 1
    # one token, or one head: refused further on, for another reason (a weight without a norm)
    for fine, tokens in ((rows(16, 8, 32, 8), 1), (rows(16, 8, 16, 32, heads=1), 4), (rows(16, 8, 16, 8), 4)):
        fine.weight = 256
        assert handle.h3q_rotary(0, fine, tokens, 8, _turn(lib), None) == 1
        assert "without a norm" in handle.h3q_last_error().decode()


def test_gather_refuses_a_length_past_its_pages(ops):
    from taomate_h3_amd.inference.paged_cache import PagedKVCache

    cache = PagedKVCache(4, 16, 2, 8, device="cpu")
    k, v = cache.gather(torch.tensor([2, 0]), 32)
    assert k.shape == v.shape == (32, 2, 8) and cache.gather(torch.tensor([2, 0]), 0)[0].shape == (0, 2, 8)
    with pytest.raises(ValueError):
        cache.gather(torch.tensor([2, 0]), 33)
    with pytest.raises(ValueError):
        cache.gather(torch.tensor([2, 0]), -1)
