"""4-bit linears, head norms with rotation and the paged cache together, as a decoder block uses them: prompts and
then single tokens of several sequences; and the module forms against the operators."""

from __future__ import annotations

import copy

import pytest
import torch

from _heads import assert_close, assert_codes, norm_rotate
from _toy_layers import ToyColumnLinear
from _util import activations
from _w4 import assert_product, product
from taomate_h3_amd.distributed.linear import _module_linear
from taomate_h3_amd.inference import lora, w4
from taomate_h3_amd.inference.fused_kernels import QuantizedActivations
from taomate_h3_amd.inference.paged_cache import PagedKVCache, QKNormRotary

pytestmark = pytest.mark.gpu

HQ, HK, D, WIDTH, PAGE = 8, 2, 64, 320, 16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _block(ops, device, zeros):
    """The linears (with the rows they were packed from) and the rotation of a block."""
    layers = []
    for n, k, seed in (((HQ + 2 * HK) * D, WIDTH, 1), (WIDTH, HQ * D, 2)):
        full = (torch.randn(n, k, generator=_gen(seed)) * k ** -0.5).to(torch.bfloat16).to(device)
        rows = ops.quantize_w4(full, 64, zeros=zeros)
        layers.append((w4.W4Linear.from_rows(*rows, group=64), [None if r is None else r.cpu() for r in rows]))
    weights = (1.0 + 0.2 * torch.randn(2, D, generator=_gen(3))).to(torch.bfloat16).to(device)
    norm = QKNormRotary(HQ, HK, D, positions=256, q_weight=weights[0], k_weight=weights[1], rot_dim=32, base=1000.0,
                        scaling="linear", factor=2.0, device=device)
    return layers, norm


def _attend(q, k, v):
    """Causal attention of the last rows, float64: q [new, HQ, D], k and v [length, HK, D]."""
    k, v = (t.double().repeat_interleave(HQ // HK, dim=1) for t in (k, v))
    scores = torch.einsum("qhd,khd->hqk", q.double(), k) * D ** -0.5
    past = len(k) - len(q)
    hidden = torch.arange(len(k), device=q.device)[None] > past + torch.arange(len(q), device=q.device)[:, None]
    return torch.einsum("hqk,khd->qhd", scores.masked_fill(hidden, -torch.inf).softmax(-1), v)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scales", [None, "static", "rows"])
def test_prompt_and_decode_steps(ops, device, scales, zeros):
    """Every stage is checked on the actual output of the one before it: qkv and out products, q, the cached rows
    (a prompt's and single tokens'), and what gather gives the attention."""
    (qkv, qkv_rows), (out, out_rows) = _block(ops, device, zeros)[0]
    norm = _block(ops, device, zeros)[1]
    static = torch.tensor([0.02, 0.03], device=device)
    fixed = dict(k_scale=static, v_scale=static) if scales == "static" else {}
    cache = PagedKVCache(24, PAGE, HK, D, scales=scales, device=device, **fixed)
    table = torch.randperm(24, generator=_gen(4))[:18].int().view(3, 6).to(device)
    lengths = torch.zeros(3, dtype=torch.int32, device=device)
    held = [[torch.zeros(0, HK, D, dtype=torch.float64)] * 2 for _ in range(3)]
    sizes = [[torch.zeros(0, HK, D, dtype=torch.float64)] * 2 for _ in range(3)]
    for step, new in enumerate(([37, 0, 16], [1, 15, 1], [1, 1, 1], [1, 33, 1])):
        tokens, pad = sum(new), 3
        cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=device)
        x = activations(tokens + pad, WIDTH, seed=step).to(device)
        rows = qkv(x)
        assert_product(rows, *product(x, *qkv_rows, 64), f"qkv {step}")
        plan = cache.plan(table, lengths, cu, tokens + pad)
        q_out = torch.full((tokens + pad, HQ, D), 9.0, device=device, dtype=x.dtype)
        q = norm.append(rows, cache, plan, q_out)
        positions = plan.positions.cpu()
        want, size = norm_rotate(norm.split(rows)[0], norm.q_weight, norm.cos, norm.sin, positions)
        assert_close(q[:tokens], want[:tokens], size[:tokens], D, f"q {step}")
        assert (q[tokens:] == 9.0).all()  # padding
        k, v = norm.split(rows)[1:]
        wanted = [norm_rotate(k, norm.k_weight, norm.cos, norm.sin, positions), norm_rotate(v)]
        lengths += torch.tensor(new, dtype=torch.int32, device=device)
        attended = torch.zeros(tokens, HQ, D, dtype=torch.float64, device=device)
        for s in range(3):
            mine = slice(int(cu[s]), int(cu[s + 1]))
            for i in range(2):
                held[s][i] = torch.cat((held[s][i], wanted[i][0][mine]))
                sizes[s][i] = torch.cat((sizes[s][i], wanted[i][1][mine]))
            length = int(lengths[s])
            got = cache.gather(table[s], length)
            for i in range(2):
                if scales is None:
                    assert_close(got[i], held[s][i], sizes[s][i], D, f"cache {step}")
                    continue
                at = torch.arange(length, device=device)
                where = table[s][at // PAGE].long(), at % PAGE
                codes = (cache.k, cache.v)[i].view(torch.uint8)[where].view(torch.float8_e4m3fn)
                by = (cache.k_scale, cache.v_scale)[i]
                by = by[where][:, :, None] if scales == "rows" else by[None, :, None].expand(length, HK, 1)
                assert_codes(codes, by.cpu(), held[s][i], sizes[s][i], D, f"codes {step}")
                assert torch.equal(got[i], (codes.float() * by).to(torch.bfloat16))
            if new[s]:
                attended[mine] = _attend(q[mine], *got)
        y = out(attended.flatten(1).to(torch.bfloat16))
        assert_product(y, *product(attended.flatten(1).to(torch.bfloat16), *out_rows, 64), f"out {step}")


@pytest.mark.parametrize("scales", [None, "rows"])
def test_tokens_appended_in_pieces_are_the_prompts_rows(ops, device, scales):
    """The same qkv rows appended at once and token by token give the same pages, bit for bit."""
    norm = _block(ops, device, False)[1]
    rows = activations(50, (HQ + 2 * HK) * D, seed=9).to(device)
    table = torch.tensor([[3, 0, 2, 1]], dtype=torch.int32, device=device)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    whole, pieces = (PagedKVCache(4, PAGE, HK, D, scales=scales, device=device) for _ in range(2))
    q = norm.append(rows, whole, whole.plan(table, i32(0), i32(0, 50), 50))
    at = 0
    for count in (1, 15, 1, 1, 30, 1, 1):
        part = norm.append(rows[at:at + count], pieces, pieces.plan(table, i32(at), i32(0, count), count))
        assert torch.equal(part, q[at:at + count])
        at += count
    assert at == 50
    for a, b in ((whole.k, pieces.k), (whole.v, pieces.v)):
        assert torch.equal(a.float(), b.float())
    if scales:
        assert torch.equal(whole.k_scale, pieces.k_scale) and torch.equal(whole.v_scale, pieces.v_scale)
    q2, k2, v2 = norm(rows, torch.arange(50, device=device))
    assert torch.equal(q2, q)
    if scales is None:
        k, v = whole.gather(table[0], 50)
        assert torch.equal(k, k2) and torch.equal(v, v2)


@pytest.mark.parametrize("scales", [None, "rows"])
def test_decode_step_in_a_graph(ops, device, scales):
    """A step of three sequences captured once (a product, plan, append, a product) and replayed as they grow, with
    eager work between; every replay gives the eager step's bits, in the pages too."""
    (qkv, _), (out, _) = _block(ops, device, False)[0]
    norm = _block(ops, device, False)[1]
    cache, eager = (PagedKVCache(12, PAGE, HK, D, scales=scales, device=device) for _ in range(2))
    table = torch.randperm(12, generator=_gen(4)).int().view(3, 4).to(device)
    lengths = torch.tensor([14, 0, 47], dtype=torch.int32, device=device)
    cu = torch.arange(4, dtype=torch.int32, device=device)
    x = activations(4, WIDTH, seed=0).to(device)  # the last row is padding

    def step(cache):
        rows = qkv(x)
        return out(norm.append(rows, cache, cache.plan(table, lengths, cu, 4)).flatten(1))

    q = step(cache)  # also what the graph's own first call would otherwise load
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = step(cache)
    assert torch.equal(step(eager)[:3], step(cache)[:3])
    for replay in range(4):
        x.copy_(activations(4, WIDTH, seed=10 + replay).to(device))
        want = step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q[:3], want[:3])
        assert torch.equal(cache.k.float(), eager.k.float()) and torch.equal(cache.v.float(), eager.v.float())
        if scales:
            assert torch.equal(cache.k_scale, eager.k_scale) and torch.equal(cache.v_scale, eager.v_scale)
        lengths += 1


@pytest.mark.parametrize("bias", [False, True])
def test_module_dispatch(ops, device, bias):
    """A parallel linear with 4-bit weights through _module_linear, its deep copy, and any leading dimensions."""
    layer = ToyColumnLinear(208, 100, bias=bias, dtype=torch.bfloat16, device=device)
    with torch.no_grad():
        layer.weight.copy_(torch.randn(100, 208, generator=_gen(1)) * 0.07)
        if bias:
            layer.bias.copy_(torch.randn(100, generator=_gen(2)))
    rows = ops.quantize_w4(layer.weight.detach(), 32, zeros=True)
    w4.set_module_w4_weight_(layer, ops.pack_w4(*rows, group=32))
    for shape in ((208,), (3, 5, 208), (2, 40, 208)):
        x = activations(max(1, torch.Size(shape[:-1]).numel()), 208, seed=3).to(device).view(shape)
        got = layer(x)
        assert got.shape == (*shape[:-1], 100)
        want, bound = product(x.reshape(-1, 208), *(r.cpu() for r in rows), 32, layer.bias)
        assert_product(got.reshape(-1, 100), want, bound)
        assert torch.equal(copy.deepcopy(layer)(x), got)
    assert _module_linear(layer, x[:0], layer.bias).shape == (0, 40, 100)
    unaligned = torch.zeros(4, 216, device=device, dtype=torch.bfloat16)[:, 3:211]
    assert layer(unaligned).shape == (4, 100)
    values = activations(4, 216, seed=4).to(device)
    for view in (values[:, 3:211], values[0, 3:211], values[:1, 8:].expand(6, 208), values.t()[:208, :1].t()):
        want, bound = product(view.reshape(-1, 208), *(r.cpu() for r in rows), 32, layer.bias)
        assert_product(layer(view).reshape(-1, 100), want, bound)
    with pytest.raises(TypeError):  # codes of another format have no bf16 rows
        codes, s = ops.quant_rows(x.reshape(-1, 208), ops.FMT_INT8)
        layer(QuantizedActivations(codes, s, tuple(x.shape), ops.FMT_INT8))


def test_lora_on_a_4_bit_base(ops, device):
    """The wrapper adds its branch to such a base by the two-product formula; folding it in is refused."""
    layer = ToyColumnLinear(128, 96, bias=False, dtype=torch.bfloat16, device=device)
    rows = ops.quantize_w4((torch.randn(96, 128, generator=_gen(1)) * 0.1).to(torch.bfloat16).to(device), 64)
    w4.set_module_w4_weight_(layer, ops.pack_w4(*rows, group=64))
    a, b = ((torch.randn(shape, generator=_gen(seed)) * 0.1).to(torch.bfloat16).to(device)
            for shape, seed in (((8, 128), 2), ((96, 8), 3)))
    wrapped = lora.H3InferenceParallelLinearLoRA(layer, kind="column", a=a, b=b, scale=0.5)
    x = activations(7, 128, seed=4).to(device)
    branch = torch.nn.functional.linear(torch.nn.functional.linear(x, a), b)
    assert torch.equal(wrapped(x), layer(x) + branch * 0.5)
    model = torch.nn.Module()
    model.layer = torch.nn.Module()  # an installed wrapper, to be swapped
    model.layer.base, model.layer.kind, model.layer.scale = layer, "column", 0.5
    model.layer.lora_a, model.layer.lora_b, model.layer._taomate_h3_inference_lora = a, b, True
    assert lora.fuse_h3_lora_wrappers_(model)["replaced_count"] == 1
    assert torch.equal(model.layer(x), wrapped(x))
    with pytest.raises(lora.H3LoRACheckpointError):
        lora.merge_h3_lora_weights_(model)


def test_block_policy(ops, device):
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            make = lambda k, n: ToyColumnLinear(k, n, bias=False, dtype=torch.bfloat16, device=device)
            self.attn, self.mlp = torch.nn.Module(), torch.nn.Module()
            self.attn.qkv_proj, self.attn.out_proj = make(128, 384), make(128, 128)
            self.mlp.fc1, self.mlp.fc2 = make(128, 256), make(128, 128)

    model = torch.nn.Module()
    model.blocks = torch.nn.ModuleList(Block() for _ in range(7))
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(torch.randn(p.shape, generator=_gen(5)) * 0.1)
    whole = {n: m.weight.detach().clone() for n, m in model.named_modules() if hasattr(m, "input_size")}
    receipt = w4.quantize_h3_block_linears_w4_(model, policy="quality_first_residual_v1", group=64)
    assert receipt["quantized_linear_names"] == [f"blocks.{b}.{p}" for b in (2, 3) for p in ("attn.qkv_proj", "mlp.fc1")]
    assert receipt["source_weight_bytes"] == 2 * (384 + 256) * 128 * 2
    assert receipt["quantized_weight_bytes"] == 2 * ((384 + 256) * 64 + (384 + 256) * 4 * 2)
    x = activations(9, 128, seed=6).to(device)
    for name, module in model.named_modules():
        if not hasattr(module, "input_size"):
            continue
        if name in receipt["quantized_linear_names"]:
            rows = [r.cpu() if r is not None else None for r in ops.quantize_w4(whole[name], 64)]
            assert_product(module(x), *product(x, *rows, 64), name)
        else:
            assert torch.equal(module.weight, whole[name])
    with pytest.raises(RuntimeError):
        w4.quantize_h3_block_linears_w4_(torch.nn.Module())


def test_cache_refuses():
    with pytest.raises(ValueError):
        PagedKVCache(2, 16, 1, 64, scales="other", device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(2, 16, 1, 64, scales="static", device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(2, 16, 1, 64, k_scale=torch.ones(1), v_scale=torch.ones(1), device="cpu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_4_bit_linears_keep_their_scales(ops, device, dtype):
    """``Module.to(dtype)`` of a model does not convert the group scales, which the codes were made for: results stay bit
    for bit; and so they do after a move to the host and back, in a deep copy and from a state dict."""
    (qkv, _), _ = _block(ops, device, True)[0]
    half = w4.W4Linear(w4.quantize_w4_weight((torch.randn(96, WIDTH, generator=_gen(1)) * 1e-3).half().to(device), group=32))
    layer = ToyColumnLinear(WIDTH, 100, bias=False, dtype=torch.float16, device=device)
    with torch.no_grad():
        layer.weight.copy_(torch.randn(100, WIDTH, generator=_gen(2)) * 0.02)
    w4.set_module_w4_weight_(layer, w4.quantize_w4_weight(layer.weight, group=32, zeros=True))
    model = torch.nn.ModuleList([qkv, half, layer])
    x = activations(20, WIDTH, seed=1).to(device)
    run = lambda m: [m[0](x), m[1](x.half()), m[2](x.half())]
    want = run(model)
    model.to(dtype)
    for a, b in zip(run(model), want):
        assert torch.equal(a, b)
    again = copy.deepcopy(model.cpu()).to(device)
    model.to(device)
    other = copy.deepcopy(model)
    for t in other.state_dict().values():
        t.zero_()
    other.load_state_dict(model.state_dict())
    for m in (model, again, other):
        for a, b in zip(run(m), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_angle_tables_keep_their_type(ops, device, dtype):
    """``Module.to(dtype)`` of a model leaves cos and sin in fp32, also on the way to the host and back."""
    norm = QKNormRotary(HQ, HK, D, positions=64, device=device)
    rows = activations(20, (HQ + 2 * HK) * D, seed=1).to(device)
    want = norm(rows)
    model = torch.nn.ModuleList([norm]).to(dtype)
    for m in (model, copy.deepcopy(model.to("cpu")).to(device), model.to(device)):
        for a, b in zip(m[0](rows), want):
            assert torch.equal(a, b)
