"""CPU tests of the 4-bit products: the plain forms that the GPU tests compare with, and refusals before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from _w4 import assert_product, dequantized, packed_codes, product, quantize, unpack_rows


def test_plain_forms_agree_with_a_hand_made_example():
    codes = torch.tensor([[0x10, 0xF8] * 8], dtype=torch.uint8)  # 0 1 8 15, four times a group of ... 32 columns
    codes = torch.cat((codes, codes), dim=1)
    assert unpack_rows(codes)[0, :4].tolist() == [0, 1, 8, 15]
    scales, zeros = torch.tensor([[0.5, 2.0]]), torch.tensor([[8, 1]], dtype=torch.uint8)
    w, _ = dequantized(codes, scales, zeros, 32)
    assert w[0, :4].tolist() == [-4.0, -3.5, 0.0, 3.5] and w[0, 32:36].tolist() == [-2.0, 0.0, 14.0, 28.0]
    x = torch.ones(1, 64, dtype=torch.bfloat16)
    y, bound = product(x, codes, scales, zeros, 32)
    assert float(y) == 8 * (-4.0 + 40.0) and float(bound) < 0.5
    with pytest.raises(AssertionError):
        assert_product((y * 1.02).to(torch.bfloat16), y, bound)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantizer_is_within_half_a_step(dtype, zeros):
    w = torch.randn(9, 208, generator=torch.Generator().manual_seed(1)).to(dtype)
    w[3, 64:96] = 0.0
    codes, scales, points = quantize(w, 32, zeros)
    back, s = dequantized(codes, scales, points, 32)
    # half a step of s, and what its own rounding (half a step of its type) takes from the ends of the range
    eps = torch.finfo(scales.dtype).eps / 2
    assert ((back - w.double()).abs() <= s * (0.5 + 15 * eps + 0.5 * zeros) + 1e-12).all()
    assert (back[3, 64:96] == 0).all()


def test_packed_layout_by_hand():
    codes = torch.zeros(3, 72, dtype=torch.uint8)  # k = 144: a second block of 16 columns
    codes[2, 65] = 0x90  # column 131: code 9 of row 2: block 1, word 0, lane 2, element 3: the low nibble of byte 3
    codes[1, 6] = 0x05   # column 12: row 1, word 0, lane 16 + 1, element 4: the high nibble of byte 0
    packed = packed_codes(codes).view(torch.int32).view(1, 2, 64, 4)
    assert packed[0, 1, 2, 0] == 9 << 24 and packed[0, 0, 17, 0] == 5 << 4
    assert int((packed != 0).sum()) == 2


def test_wrappers_refuse_cpu_tensors(ops):
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    w = ops.W4Weight(torch.zeros(1, 1, 1024, dtype=torch.uint8), torch.zeros(1, 1, 16, 4, dtype=torch.bfloat16), None, 16, 32, 32)
    for call in (lambda: ops.quantize_w4(x), lambda: ops.pack_w4(torch.zeros(2, 16, dtype=torch.uint8), x[:, :1]),
                 lambda: ops.w4_mm(x, w)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_c_entry_points_refuse():
    from taomate_h3_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.lib()
    error = lambda: lib.h3q_last_error().decode()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)

    def mm(dtype=0, x=p, ldx=64, sd=0, group=32, out=p, ldo=48, m=4, n=48, k=64, ws=None, size=0, codes=p):
        return lib.h3q_w4_mm(dtype, x, ldx, codes, p, sd, None, group, None, out, ldo, m, n, k, ws, size, None)

    assert mm(dtype=2) == 1 and "binary16" in error()
    assert mm(sd=2) == 1 and "binary16" in error()
    assert mm(k=72, ldx=72) == 1 and "multiple of 16" in error()
    assert mm(k=0, ldx=0) == 1 and mm(k=(1 << 22) + 16, ldx=1 << 23) == 1
    assert mm(group=48) == 1 and "group" in error()
    assert mm(group=96) == 1 and mm(group=0) == 1 and mm(group=-128) == 1
    assert mm(ldx=60) == 1 and "ldx" in error()
    assert mm(ldx=68) == 1 and "ldx" in error()
    assert mm(ldx=1 << 23) == 1 and "ldx" in error()
    assert mm(ldo=47) == 1 and "ldo" in error()
    assert mm(m=-1) == 1 and mm(n=-1) == 1
    assert mm(x=odd) == 1 and "aligned" in error()
    assert mm(codes=None) == 1 and "null" in error()
    assert mm(m=0) == 0 and mm(n=0) == 0
    need = lib.h3q_w4_mm_workspace_bytes(300, 48, 16384, 32)  # few tiles, long rows: a split sum
    assert need > 0 and lib.h3q_w4_mm_workspace_bytes(4, 48, 4096, 32) == 0
    assert mm(m=300, k=16384, ldx=16384) == 1 and "workspace" in error()
    assert mm(m=300, k=16384, ldx=16384, ws=p, size=need - 1) == 1 and "needed" in error()
    assert mm(m=(1 << 31) - 1, n=1 << 20, ldo=1 << 20) == 2 and "too many" in error()
    assert lib.h3q_w4_code_bytes(17, 144) == 2 * 2 * 1024 and lib.h3q_w4_code_bytes(0, 144) == 0
    pack = lambda ldc=32, lds=2, z=None, ldz=0, n=4, k=64, zo=None, out=p: lib.h3q_w4_pack(
        p, ldc, p, lds, z, ldz, n, k, 32, out, p, zo, None)
    assert pack(ldc=31) == 1 and "row strides" in error()
    assert pack(lds=1) == 1 and pack(z=p, ldz=1, zo=p) == 1
    assert pack(z=p, ldz=2) == 1 and "one side" in error()
    assert pack(out=odd) == 1 and "aligned" in error()
    assert pack(n=0) == 0
    assert lib.h3q_w4_quantize(p, 3, 64, 4, 64, 32, p, p, None, None) == 1
    assert lib.h3q_w4_quantize(p, 0, 63, 4, 64, 32, p, p, None, None) == 1 and "stride" in error()
    assert lib.h3q_w4_quantize(None, 0, 64, 4, 64, 32, p, p, None, None) == 1 and "null" in error()
    assert lib.h3q_w4_quantize(p, 0, 64, 0, 64, 32, p, p, None, None) == 0


def test_c_entry_points_refuse_grids_past_32_bits():
    """A launch of 2^32 threads or more is cut off without an error: products that would need one are refused."""
    from taomate_h3_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.lib()
    p = ctypes.c_void_p(256)
    mm = lambda m, n: lib.h3q_w4_mm(0, p, 64, p, p, 0, None, 32, None, p, n, m, n, 64, None, 0, None)
    for m, n in ((1, 1 << 28), (16, 1 << 30), (1 << 20, 1 << 20)):
        assert mm(m, n) == 2 and "too many" in lib.h3q_last_error().decode()


def test_scales_keep_their_dtype(ops):
    """Conversions of a model convert neither a W4Linear's scales nor those beside a module of another class."""
    import torch
    from taomate_h3_amd.inference import w4

    scales = torch.tensor([1.0009765625, 3e-6] * 32).to(torch.float16).view(1, 1, 16, 4)
    weight = ops.W4Weight(torch.zeros(1, 1, 1024, dtype=torch.uint8), scales, None, 16, 64, 32)
    linear, other = w4.W4Linear(weight, torch.zeros(16)), torch.nn.Linear(64, 16)
    w4.set_module_w4_weight_(other, weight)
    model = torch.nn.Sequential(linear, other).to(torch.bfloat16).float().half().bfloat16()
    assert linear.bias.dtype == torch.bfloat16 and other.bias.dtype == torch.bfloat16
    for held in (linear.weight, w4.module_w4_weight(other)):
        assert held.scales.dtype == torch.float16 and torch.equal(held.scales, scales) and held.zeros is None
        assert held.codes.dtype == torch.uint8
    model.to("meta")
    assert linear.scales.device.type == "meta" and linear.scales.dtype == torch.float16
