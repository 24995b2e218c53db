"""The CPU restatements of the routed-expert operators (tests/_experts.py) against
second forms of the same definitions, and the operators' refusals that need no GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import _experts as R


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_restatement_against_sort(scoring, renorm):
    gen = torch.Generator().manual_seed(1)
    logits = torch.randn(50, 12, generator=gen).to(torch.bfloat16).float()
    logits[3] = -torch.inf
    logits[4, :10] = -torch.inf
    logits[5, 2] = torch.nan
    ids, weights = R.route(logits, 4, scoring, renorm)
    clean = torch.nan_to_num(logits.double(), nan=-torch.inf, neginf=-torch.inf, posinf=torch.inf)
    values, order = torch.sort(clean, dim=1, descending=True, stable=True)
    want = torch.where(values[:, :4] > -torch.inf, order[:, :4], -1)
    assert (ids == want.numpy()).all()
    if scoring == "softmax":
        p = torch.softmax(values[:, :4] if renorm else clean, dim=1)
        p = p if renorm else torch.gather(p, 1, order[:, :4])
    else:
        p = torch.sigmoid(values[:, :4])
        p = p / p.sum(1, keepdim=True) if renorm else p
    np.testing.assert_allclose(weights, np.where(ids >= 0, p.numpy(), 0.0), rtol=1e-12)


def test_plan_restatement():
    ids = np.array([[2, 0], [-1, 2], [1, 5], [2, 0]], np.int32)
    order, offsets, slots = R.plan(ids, 3)
    assert order.tolist() == [1, 7, 4, 0, 3, 6, -1, -1]
    assert offsets.tolist() == [0, 2, 3, 6]
    assert slots.tolist() == [[3, 0], [-1, 4], [2, -1], [5, 1]]
    order, offsets, _ = R.plan(ids, 2, first=2)
    assert order.tolist()[:3] == [0, 3, 6] and offsets.tolist() == [0, 3, 3]


def test_bf16_rounding_restatement():
    v = np.array([1.0 + 2.0 ** -8, 1.0 + 2.0 ** -8 + 2.0 ** -40, 1.0 + 3 * 2.0 ** -8, -1.0 - 2.0 ** -8 - 2.0 ** -40, 0.0,
                  3.0e-39])
    want = torch.tensor([1.0, 1.0 + 2.0 ** -7, 1.0 + 2.0 ** -6, -1.0 - 2.0 ** -7, 0.0, 3.0e-39], dtype=torch.float64)
    want[5] = torch.tensor(3.0e-39).to(torch.bfloat16).double()
    assert (R.to_bf16(v) == want.numpy()).all()


def test_native_refusals_without_gpu():
    """Arguments that are refused on the host before any launch (no pointer is followed)."""
    from taomate_h3_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.lib()
    p = ctypes.c_void_p(256)

    def refused(code, text, name, *args):
        assert getattr(lib, name)(*args) == code, name
        assert text in lib.h3q_last_error(), lib.h3q_last_error()

    route = lambda **k: [p, k.get("dtype", 2), k.get("ldl", 8), k.get("t", 4), k.get("e", 8), k.get("k", 2),  # noqa: E731
                         k.get("scoring", 0), 1, 1.0, p, p, None]
    refused(1, b"top_k", "h3q_route_topk", *route(k=0))
    refused(1, b"top_k", "h3q_route_topk", *route(k=9))
    refused(1, b"experts", "h3q_route_topk", *route(e=1025, ldl=1025))
    refused(1, b"dtype", "h3q_route_topk", *route(dtype=3))
    refused(1, b"scoring", "h3q_route_topk", *route(scoring=2))
    refused(1, b"leading dimension", "h3q_route_topk", *route(ldl=7))
    refused(1, b"negative", "h3q_route_topk", *route(t=-1))
    refused(2, b"31 bits", "h3q_route_topk", *route(t=2 ** 31))
    refused(1, b"null", "h3q_route_topk", None, *route()[1:])
    assert lib.h3q_route_topk(*route(t=0)) == 0

    refused(1, b"first", "h3q_plan_experts", p, 4, 2, -1, 8, p, p, p, None, 0, None)
    refused(1, b"null", "h3q_plan_experts", p, 4, 2, 0, 8, p, None, p, None, 0, None)
    many = lib.h3q_plan_experts_workspace_bytes(1 << 15, 8, 64)
    assert many > 0 and lib.h3q_plan_experts_workspace_bytes(100, 8, 64) == 0
    refused(1, b"workspace", "h3q_plan_experts", p, 1 << 15, 8, 0, 64, p, p, p, None, 0, None)
    refused(1, b"workspace", "h3q_plan_experts", p, 1 << 15, 8, 0, 64, p, p, p, p, many - 1, None)

    def grouped(**k):
        return [k.get("fmt", 1), p, k.get("lda", 128), k.get("a_rows", 8), p, k.get("order"), k.get("top_k", 1), k.get("b", p),
                k.get("layout", 0), p, p, k.get("e", 4), k.get("rows", 8), k.get("n", 64), k.get("k", 128),
                k.get("swiglu", 0), k.get("f32", 0), k.get("out", p), k.get("ldo", 64), None]

    refused(1, b"unknown format", "h3q_grouped_mm", *grouped(fmt=2))
    refused(1, b"unknown layout", "h3q_grouped_mm", *grouped(layout=2))
    refused(1, b"multiple of 128", "h3q_grouped_mm", *grouped(layout=1, k=144, lda=144))
    refused(1, b"multiple of 16", "h3q_grouped_mm", *grouped(k=120))
    refused(1, b"n=48", "h3q_grouped_mm", *grouped(n=48, swiglu=1))
    refused(2, b"bf16", "h3q_grouped_mm", *grouped(swiglu=1, f32=1))
    refused(1, b"lda", "h3q_grouped_mm", *grouped(lda=112))
    refused(1, b"ldo", "h3q_grouped_mm", *grouped(ldo=60))
    refused(1, b"8 rows, 9", "h3q_grouped_mm", *grouped(rows=9))
    refused(2, b"2 GiB", "h3q_grouped_mm", *grouped(n=1 << 20, k=2048, lda=2048, ldo=1 << 20))
    refused(2, b"gathered", "h3q_grouped_mm", *grouped(order=p, a_rows=1 << 24))
    refused(2, b"32 bits", "h3q_grouped_mm", *grouped(k=1 << 18, lda=1 << 18))
    refused(1, b"top_k", "h3q_grouped_mm", *grouped(order=p, top_k=1 << 32))
    refused(1, b"null", "h3q_grouped_mm", *grouped(b=None))
    refused(1, b"aligned", "h3q_grouped_mm", *grouped(out=ctypes.c_void_p(264)))
    assert lib.h3q_grouped_mm(*grouped(rows=0)) == 0

    refused(1, b"columns", "h3q_combine_experts", p, 0, 8, 4, p, p, 2, 2, 12, p, 16, None)
    refused(1, b"strides", "h3q_combine_experts", p, 0, 8, 4, p, p, 2, 2, 16, p, 16, None)

    def ffn(**k):
        return [k.get("fmt", 0), p, k.get("ldx", 128), k.get("t", 4), k.get("d", 128), k.get("f", 128), p, p, 2,
                k.get("first", 0), k.get("e", 8), p, k.get("l13", 0), p, p, k.get("l2", 0), p, p, 128, k.get("ws", p),
                k.get("bytes", 1 << 30), None]

    refused(1, b"multiples of 16", "h3q_expert_ffn", *ffn(f=120))
    refused(1, b"multiple of 128", "h3q_expert_ffn", *ffn(f=144, l2=1))
    refused(1, b"workspace", "h3q_expert_ffn", *ffn(bytes=64))
    refused(1, b"workspace", "h3q_expert_ffn", *ffn(ws=None))
    refused(1, b"strides", "h3q_expert_ffn", *ffn(ldx=120))
    refused(1, b"first", "h3q_expert_ffn", *ffn(first=-1))
    refused(2, b"2 GiB", "h3q_expert_ffn", *ffn(t=1 << 24))
    assert lib.h3q_expert_ffn(*ffn(t=0)) == 0


def test_wrappers_refuse_cpu_tensors(ops):
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    ids, w = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    codes = torch.zeros(4, 128, dtype=torch.int8)
    stack = torch.zeros(2, 128, 128, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.route_experts(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.plan_experts(ids, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.grouped_scaled_mm(codes, stack, torch.zeros(4), torch.zeros(2, 128), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.combine_experts(x, ids, w)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.expert_ffn(x, ids, w, stack.expand(2, 128, 128), torch.zeros(2, 128), stack[:, :, :64].contiguous(),
                       torch.zeros(2, 128))


def test_expert_module_checks_shapes():
    import importlib

    experts = importlib.import_module("taomate_h3_amd.inference.experts")
    with pytest.raises(TypeError, match="bf16"):
        experts.quantize_expert_weights(torch.zeros(2, 16, 16), 1)
    with pytest.raises(ValueError, match="multiples of 16"):
        experts.quantize_expert_weights(torch.zeros(2, 24, 16, dtype=torch.bfloat16), 1)
    with pytest.raises(ValueError, match="expert weights"):
        experts.QuantizedExperts(torch.zeros(2, 64, 32), torch.zeros(2, 64), torch.zeros(2, 32, 16), torch.zeros(2, 32),
                                 w13_tiled=False, w2_tiled=False)


def test_int8_sums_stay_below_32_bits():
    """128 * 128 * k of codes that are all -128 reaches 2^31 at k = 131072: refused, the k below it taken."""
    from taomate_h3_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.lib()
    p = ctypes.c_void_p(256)

    def grouped(fmt, k):  # no rows: checked, nothing launched
        return lib.h3q_grouped_mm(fmt, p, k, 8, p, None, 1, p, 0, p, p, 4, 0, 16, k, 0, 0, p, 16, None)

    def ffn(fmt, d, f):
        return lib.h3q_expert_ffn(fmt, p, d, 0, d, f, p, p, 2, 0, 4, p, 0, p, p, 0, p, p, d, p, 1 << 30, None)

    assert 128 * 128 * 131056 < 2 ** 31 <= 128 * 128 * 131072
    for call in (lambda fmt, k: grouped(fmt, k), lambda fmt, k: ffn(fmt, k, 16), lambda fmt, k: ffn(fmt, 16, k)):
        assert call(1, 131056) == 0
        assert call(1, 131072) == 2 and b"32 bits" in lib.h3q_last_error()
        assert call(0, 131072) == 0  # e4m3 sums are binary32


def test_router_refuses_more_tokens_than_a_launch_takes():
    """16 lanes a token (64 above 256 experts or 16 slots) and a grid of fewer than 2^32 threads."""
    from taomate_h3_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.lib()
    p = ctypes.c_void_p(256)
    for tokens, experts, top_k in ((1 << 28, 256, 1), (1 << 26, 257, 1), (1 << 26, 64, 17)):
        assert lib.h3q_route_topk(p, 2, experts, tokens, experts, top_k, 0, 1, 1.0, p, p, None) == 2
        assert b"workgroups" in lib.h3q_last_error()
