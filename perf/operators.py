"""Performance cases of the routed-expert operators, plain and through the package's public entry points.

Operators (``op``):

``route``    the router of an expert layer: top-k of the logits with their weights, and the
             plan that sorts the (token, slot) pairs by expert.
``grouped``  one 8-bit product with scales for each token and channel over rows grouped by
             expert, the rows gathered from the tokens or already sorted (``gather``), the
             gate and up columns optionally joined by SwiGLU (``swiglu``).
``ffn``      the whole expert layer on routed tokens: activation codes, gate and up
             products, SwiGLU, codes again, down product, weighted sum over the experts.

Widths are the H3 block's (5376, 7168) and generic ones; token counts run from one decoded
token to a prefill of many thousand, odd ones among them.
"""

from __future__ import annotations

import importlib

import numpy as np
import torch

from __graft_entry__ import load_package

own = False

DEVICE = "cuda"
_LIMIT = {"int8": 127.0, "e4m3": 448.0}
_MOST_FLOPS = 2 * 16384 * 14336 * 5376


def listed() -> list[dict]:
    return [
        # One decoded token through the router: launches and latency.
        {"name": "route_t1", "op": "route", "t": 1, "e": 64, "k": 8, "dtype": "f32", "scoring": "softmax",
         "renorm": True, "total": 64, "first": 0},
        # A prefill over many experts, bf16 logits (ties), sigmoid scores, one expert-parallel rank's share.
        {"name": "route_t4093_rank", "op": "route", "t": 4093, "e": 64, "k": 8, "dtype": "bf16", "scoring": "sigmoid",
         "renorm": True, "total": 256, "first": 64},
        # The largest routing call: a packed batch of chunks.
        {"name": "route_t32768", "op": "route", "t": 32768, "e": 128, "k": 4, "dtype": "f32", "scoring": "softmax",
         "renorm": False, "total": 128, "first": 0},
        # One decoded token: eight of 64 fine-grained experts, the weight stream and the launches.
        {"name": "ffn_int8_t1", "op": "ffn", "fmt": "int8", "t": 1, "e": 64, "k": 8, "d": 2048, "f": 1024,
         "total": 64, "first": 0},
        # A few audio tokens over eight wide experts of the H3 widths: nearly every expert is read.
        {"name": "ffn_e4m3_t7", "op": "ffn", "fmt": "e4m3", "t": 7, "e": 8, "k": 2, "d": 5376, "f": 7168,
         "total": 8, "first": 0},
        # A decode batch over 128 small experts: a handful of tokens each, some with none.
        {"name": "ffn_int8_t40", "op": "ffn", "fmt": "int8", "t": 40, "e": 128, "k": 8, "d": 2048, "f": 768,
         "total": 128, "first": 0},
        # Odd widths (row-major weights) on one expert-parallel rank: half of the pairs belong to others.
        {"name": "ffn_e4m3_t53_odd", "op": "ffn", "fmt": "e4m3", "t": 53, "e": 20, "k": 4, "d": 1424, "f": 592,
         "total": 40, "first": 20},
        # A prefill chunk through the whole layer.
        {"name": "ffn_int8_t2048", "op": "ffn", "fmt": "int8", "t": 2048, "e": 64, "k": 6, "d": 2048, "f": 1408,
         "total": 64, "first": 0},
        # The down product of a mid-sized step, skewed groups, sorted rows.
        {"name": "grouped_e4m3_p601", "op": "grouped", "fmt": "e4m3", "t": 601, "e": 16, "k": 1, "d": 2048, "n": 4096,
         "gather": False, "swiglu": False, "total": 16, "first": 0},
        # Gate and up of a prefill chunk, rows gathered, groups of a few hundred rows.
        {"name": "grouped_e4m3_t4096_swiglu", "op": "grouped", "fmt": "e4m3", "t": 4096, "e": 64, "k": 8, "d": 2048,
         "n": 2816, "gather": True, "swiglu": True, "total": 64, "first": 0},
        # The largest product: gate and up of eight H3-wide experts over a whole 480p chunk.
        {"name": "grouped_int8_t8192_swiglu", "op": "grouped", "fmt": "int8", "t": 8192, "e": 8, "k": 2, "d": 5376,
         "n": 14336, "gather": True, "swiglu": True, "total": 8, "first": 0},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng) -> dict:
    op = rng.choice(("route", "ffn", "ffn", "ffn", "grouped", "grouped"))
    fmt = rng.choice(("int8", "e4m3"))
    e = rng.choice((4, 8, 20, 64, 128))
    ranks = rng.choice((1, 1, 1, 2, 4))
    total = e * ranks
    first = e * rng.randrange(ranks)
    if op == "route":
        return {"op": op, "t": _log_int(rng, 1, 32768), "e": e, "k": rng.randint(1, min(8, total)),
                "dtype": rng.choice(("f32", "bf16", "f16")), "scoring": rng.choice(("softmax", "sigmoid")),
                "renorm": rng.random() < 0.5, "total": total, "first": first}
    # Widths in 16s, and in 128s half of the time (the tiled layout).
    unit = rng.choice((16, 128))
    width = 8 if e <= 8 else 2
    d = unit * _log_int(rng, 256 // unit, 1024 * width // unit)
    f = unit * _log_int(rng, 256 // unit, 768 * width // unit)
    k = rng.randint(1, min(8, total))
    if op == "ffn":
        return {"op": op, "fmt": fmt, "t": min(_log_int(rng, 1, 2048), _MOST_FLOPS // (6 * k * d * f)), "e": e, "k": k,
                "d": d, "f": f, "total": total, "first": first}
    swiglu, gather = rng.random() < 0.5, rng.random() < 0.5
    k, n = k if gather else 1, 2 * f if swiglu else f
    return {"op": op, "fmt": fmt, "t": min(_log_int(rng, 1, 4096), _MOST_FLOPS // (2 * k * d * n)), "e": e, "k": k,
            "d": d, "n": n, "gather": gather, "swiglu": swiglu, "total": total, "first": first}


# ------------------------------------------------------------------ inputs

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _logits(gen, t: int, total: int, dtype=torch.float32) -> torch.Tensor:
    """Router logits: some experts are favoured, 1 token of 64 is padding (no expert at all) and
    one logit of 50 is masked."""
    l = torch.randn((t, total), generator=gen, device=DEVICE) * 1.5
    l += torch.randn((1, total), generator=gen, device=DEVICE) * 0.7
    l[torch.rand((t, total), generator=gen, device=DEVICE) < 0.02] = -torch.inf
    l[torch.rand((t, 1), generator=gen, device=DEVICE).expand(t, total) < 1 / 64] = -torch.inf
    return l.to(dtype)


def _activations(gen, t: int, d: int) -> torch.Tensor:
    """N(0, 1) with 1% of the channels 15 times larger."""
    x = torch.randn((t, d), generator=gen, device=DEVICE)
    x[:, torch.randperm(d, generator=gen, device=DEVICE)[:max(1, d // 100)]] *= 15.0
    return x.to(torch.bfloat16)


def _weights(gen, e: int, n: int, d: int) -> torch.Tensor:
    w = torch.empty((e, n, d), device=DEVICE, dtype=torch.bfloat16)
    for i in range(e):
        w[i] = torch.randn((n, d), generator=gen, device=DEVICE) * d ** -0.5
    return w


def _inputs(case: dict, seed: int) -> dict:
    gen, op = _gen(seed), case["op"]
    if op == "route":
        dtype = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[case["dtype"]]
        return {"logits": _logits(gen, case["t"], case["total"], dtype)}
    experts, weights = _route(_logits(gen, case["t"], case["total"]), case["k"], "softmax", True)
    t = {"experts": experts, "weights": weights, "x": _activations(gen, case["t"], case["d"])}
    if op == "ffn":
        t["w13"] = _weights(gen, case["e"], 2 * case["f"], case["d"])
        t["w2"] = _weights(gen, case["e"], case["d"], case["f"])
    else:
        t["w"] = _weights(gen, case["e"], case["n"], case["d"])
    return t


def prepare(case: dict, seed: int):
    t, op = _inputs(case, seed), case["op"]
    if own:
        load_package()
        ops = t["ops"] = importlib.import_module("taomate_h3_amd.ops")
    if op == "route":
        return {**case, **t}
    if own:
        experts = importlib.import_module("taomate_h3_amd.inference.experts")
        fmt = ops.FMT_INT8 if case["fmt"] == "int8" else ops.FMT_E4M3FN
        if op == "ffn":
            layer = experts.QuantizedExperts.from_weights(t.pop("w13"), t.pop("w2"), fmt, first_expert=case["first"])
            return {**case, **t, "layer": layer}
        w, w_scale, tiled = experts.quantize_expert_weights(t.pop("w"), fmt)
        t.update(w=w, w_scale=w_scale, tiled=tiled)
    else:
        for name in ("w13", "w2") if op == "ffn" else ("w",):
            w = t.pop(name)
            codes, scales = zip(*(_quantize(w[i].float(), case["fmt"], True) for i in range(case["e"])))
            t[name] = torch.stack([c.view(torch.uint8) for c in codes]).view(codes[0].dtype)
            t[name + "_scale"] = torch.stack(scales).squeeze(2)
            del w, codes, scales
    if op == "grouped":
        # The program has the activation codes (of the tokens, or of the sorted rows), the plan and an output buffer.
        order, offsets, _ = _plan(t.pop("experts"), case["e"], case["first"])
        t.pop("weights")
        t["a"], t["a_scale"] = _quantize(t.pop("x").float(), case["fmt"], False)
        t["order"], t["offsets"] = order, offsets
        cols = case["n"] // 2 if case["swiglu"] else case["n"]
        t["out"] = torch.zeros((case["t"] * case["k"], cols), device=DEVICE, dtype=torch.bfloat16)
    return {**case, **t}


# ------------------------------------------------------------- plain forms

def _route(logits: torch.Tensor, k: int, scoring: str, renorm: bool):
    l = logits.float()
    l = torch.where(torch.isnan(l), -torch.inf, l)
    values, experts = torch.sort(l, dim=1, descending=True, stable=True)
    values, experts = values[:, :k], experts[:, :k].to(torch.int32)
    taken = values > -torch.inf
    if scoring == "sigmoid":
        weights = torch.where(taken, 1.0 / (1.0 + torch.exp(-values)), 0.0)
        if renorm:
            weights = weights / weights.sum(dim=1, keepdim=True)
    else:
        top = values[:, :1]
        weights = torch.where(taken, torch.exp(values - top), 0.0)
        whole = weights if renorm else torch.where(l > -torch.inf, torch.exp(l - top), 0.0)
        weights = weights / whole.sum(dim=1, keepdim=True)
    return torch.where(taken, experts, -1), torch.where(taken, weights, 0.0)


def _plan(experts: torch.Tensor, e: int, first: int):
    """Pairs (token * k + slot) sorted by expert, in their own order within one: the pair behind each
    sorted row (-1 past the last), the groups' bounds, and the row of each pair (-1: no expert here)."""
    flat = experts.flatten().long() - first
    flat = torch.where((experts.flatten() >= 0) & (flat >= 0) & (flat < e), flat, e)
    group, order = torch.sort(flat, stable=True)
    counts = (flat[:, None] == torch.arange(e, device=flat.device)).sum(dim=0)
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
    slots = torch.empty_like(order)
    slots[order] = torch.where(group < e, torch.arange(order.numel(), device=order.device), -1)
    order = torch.where(group < e, order, -1)
    return order.to(torch.int32), offsets, slots.to(torch.int32).view(experts.shape)


def _quantize(x: torch.Tensor, fmt: str, weight: bool):
    """Codes and scale of each row: of the largest magnitude over 448 or 127 (int8 activations:
    the reciprocal form)."""
    amax = x.abs().amax(dim=1, keepdim=True)
    if fmt == "e4m3":
        scale = torch.clamp(amax * (1.0 / 448.0), min=1e-12)
        return torch.clamp(x / scale, -448.0, 448.0).to(torch.float8_e4m3fn), scale
    if weight:
        scale = torch.clamp(amax * (1.0 / 127.0), min=1e-12)
        return torch.clamp(torch.round(x / scale), -127.0, 127.0).to(torch.int8), scale
    # tensors on both sides: torch divides by a number, and a number by a tensor, through a rounded reciprocal
    limit = torch.full_like(amax, 127.0)
    inverse = torch.where(amax > 0, limit / amax, 0.0)
    return torch.clamp(torch.round(x * inverse), -128.0, 127.0).to(torch.int8), amax / limit


def _product(a, a_scale, w, w_scale, swiglu: bool):
    y = a_scale * (w_scale * (a.float() @ w.float().T))
    if not swiglu:
        return y
    gate, up = y.chunk(2, dim=1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_grouped(s) -> torch.Tensor:
    bounds = s["offsets"].tolist()
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if hi > lo:
            rows = s["order"][lo:hi] // s["k"] if s["gather"] else slice(lo, hi)
            a = s["a"].view(torch.uint8)[rows].view(s["a"].dtype)
            s["out"][lo:hi] = _product(a, s["a_scale"][rows], s["w"][e], s["w_scale"][e], s["swiglu"])
    return s["out"]


def _plain_ffn(s) -> torch.Tensor:
    order, offsets, _ = _plan(s["experts"], s["e"], s["first"])
    q, q_scale = _quantize(s["x"].float(), s["fmt"], False)
    pairs = torch.zeros((s["t"] * s["k"], s["d"]), device=DEVICE)
    bounds = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if hi == lo:
            continue
        pair = order[lo:hi].long()
        rows = pair // s["k"]
        # what the second quantizer takes is bf16, as every activation that is quantized
        a = q.view(torch.uint8)[rows].view(q.dtype)
        h = _product(a, q_scale[rows], s["w13"][e], s["w13_scale"][e], True).to(torch.bfloat16)
        h, h_scale = _quantize(h.float(), s["fmt"], False)
        pairs[pair] = _product(h, h_scale, s["w2"][e], s["w2_scale"][e], False)
    weighted = pairs.view(s["t"], s["k"], s["d"]) * s["weights"][:, :, None]
    return weighted.sum(dim=1).to(torch.bfloat16)


def run(state):
    s, op = state, state["op"]
    if own:
        ops = s["ops"]
        if op == "ffn":
            return s["layer"](s["x"], s["experts"], s["weights"])
        if op == "grouped":
            return ops.grouped_scaled_mm(s["a"], s["w"], s["a_scale"], s["w_scale"], s["offsets"],
                                         order=s["order"] if s["gather"] else None, top_k=s["k"], swiglu=s["swiglu"],
                                         b_tiled=s["tiled"], out=s["out"])
        experts, weights = ops.route_experts(s["logits"], s["k"], scoring=s["scoring"], renormalize=s["renorm"])
        plan = ops.plan_experts(experts, s["e"], first_expert=s["first"])
        return {"experts": experts, "weights": weights, "order": plan.order, "offsets": plan.offsets,
                "slots": plan.slots}
    if op == "ffn":
        return _plain_ffn(s)
    if op == "grouped":
        return _plain_grouped(s)
    experts, weights = _route(s["logits"], s["k"], s["scoring"], s["renorm"])
    order, offsets, slots = _plan(experts, s["e"], s["first"])
    return {"experts": experts, "weights": weights, "order": order, "offsets": offsets, "slots": slots}


# -------------------------------------------------------------------- work

def work(case: dict) -> dict:
    """What a pass cannot do without: each input read once, each output written once.  The experts
    read are those that the expected share of the pairs falls on."""
    op, t, k, e = case["op"], case["t"], case["k"], case["e"]
    if op == "route":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": size * t * case["total"] + t * k * (8 + 8) + 4 * e, "flops": t * case["total"] * 6}
    here = e / case["total"]
    pairs = t * k * here
    active = e * (1.0 - (1.0 - k / case["total"]) ** t)
    if op == "ffn":
        d, f = case["d"], case["f"]
        weights = active * (3 * f * d + 4 * (2 * f + d))
        return {"bytes": int(weights + 4 * t * d + 8 * t * k), "flops": int(6 * pairs * f * d)}
    d, n = case["d"], case["n"]
    rows = min(t, pairs) if case["gather"] else pairs
    cols = n // 2 if case["swiglu"] else n
    return {"bytes": int(active * (n * d + 4 * n) + rows * (d + 4) + 2 * pairs * cols),
            "flops": int(2 * pairs * n * d)}


# ------------------------------------------- the definition, in 64 bits

def _exact_route(case, logits):
    l = logits.double().cpu()
    l[torch.isnan(l)] = -torch.inf
    experts = torch.full((case["t"], case["k"]), -1, dtype=torch.int32)
    weights = torch.zeros((case["t"], case["k"]), dtype=torch.float64)
    left = l.clone()
    rows = torch.arange(case["t"])
    for j in range(case["k"]):  # the largest left, the lowest index among equals
        best = left.amax(dim=1)
        index = (left == best[:, None]).to(torch.int8).argmax(dim=1)
        ok = best > -torch.inf
        experts[ok, j] = index[ok].to(torch.int32)
        weights[:, j] = torch.where(ok, best, -torch.inf)
        left[rows, index] = -torch.inf
    if case["scoring"] == "sigmoid":
        weights = torch.sigmoid(weights)
        if case["renorm"]:
            weights = weights / weights.sum(dim=1, keepdim=True)
    else:
        weights = torch.softmax(weights, dim=1) if case["renorm"] else torch.exp(
            weights - torch.logsumexp(l, dim=1, keepdim=True))
    return experts, torch.where(experts >= 0, weights, 0.0)


def _exact_plan(case, experts):
    e, first = case["e"], case["first"]
    flat = experts.flatten().cpu().numpy()
    mine = np.flatnonzero((flat >= first) & (flat < first + e) & (flat >= 0))
    mine = mine[np.argsort(flat[mine], kind="stable")]
    order = np.full(flat.size, -1, np.int32)
    order[:mine.size] = mine
    slots = np.full(flat.size, -1, np.int32)
    slots[mine] = np.arange(mine.size)
    offsets = np.searchsorted(flat[mine], np.arange(first, first + e + 1)).astype(np.int32)
    return torch.from_numpy(order), torch.from_numpy(offsets), torch.from_numpy(slots).view(experts.shape)


def _exact_codes(x: torch.Tensor, fmt: str, weight: bool):
    """Codes (as binary64 values) and scales: the codes are a definition in binary32, all that
    follows is arithmetic on exact values."""
    x = x.float()
    amax = x.abs().max(dim=1, keepdim=True).values
    if fmt == "int8" and not weight:
        inverse = torch.div(torch.full_like(amax, 127.0), amax)  # one IEEE division, as the codes' definition has it
        codes = torch.round(x * torch.nan_to_num(inverse, posinf=0.0)).clamp(-128, 127)
        return codes.double(), amax.double() / 127.0
    scale = torch.clamp(amax * (1.0 / _LIMIT[fmt]), min=1e-12)
    if fmt == "e4m3":
        return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double(), scale.double()
    return torch.round(x / scale).clamp(-127, 127).double(), scale.double()


def exact(case: dict, seed: int):
    t, op = _inputs(case, seed), case["op"]
    if op == "route":
        experts, weights = _exact_route(case, t["logits"])
        order, offsets, slots = _exact_plan(case, experts)
        return {"experts": experts, "weights": weights, "order": order, "offsets": offsets, "slots": slots}
    order, offsets, _ = _exact_plan(case, t["experts"])
    bounds, order = offsets.tolist(), order.to(DEVICE).long()
    x, x_scale = _exact_codes(t["x"], case["fmt"], False)

    def product(a, a_scale, w):
        q, s = _exact_codes(w, case["fmt"], True)
        return (a @ q.T) * a_scale * s.T

    def silu_mul(y):
        gate, up = y[:, :y.shape[1] // 2], y[:, y.shape[1] // 2:]
        return gate * torch.sigmoid(gate) * up

    if op == "grouped":
        cols = case["n"] // 2 if case["swiglu"] else case["n"]
        out = torch.zeros((case["t"] * case["k"], cols), device=DEVICE, dtype=torch.float64)
        for e in range(case["e"]):
            lo, hi = bounds[e], bounds[e + 1]
            if lo == hi:
                continue
            rows = order[lo:hi] // case["k"] if case["gather"] else torch.arange(lo, hi, device=DEVICE)
            y = product(x[rows], x_scale[rows], t["w"][e])
            out[lo:hi] = silu_mul(y) if case["swiglu"] else y
        return out
    out = torch.zeros((case["t"], case["d"]), device=DEVICE, dtype=torch.float64)
    share = t["weights"].double().flatten()
    for e in range(case["e"]):
        pair = order[bounds[e]:bounds[e + 1]]
        if pair.numel() == 0:
            continue
        rows = pair // case["k"]
        h = silu_mul(product(x[rows], x_scale[rows], t["w13"][e]))
        q, s = _exact_codes(h.to(torch.bfloat16), case["fmt"], False)
        out.index_add_(0, rows, product(q, s, t["w2"][e]) * share[pair, None])
    return out
