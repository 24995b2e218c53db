// The tensor wrappers of ops.py in native code: the same checks, the same
// output allocations and the same C entry points, without the interpreter
// between them.  Each function takes torch tensors and the raw stream of the
// first one's device, and returns None for anything out of the ordinary (a
// wrong type, shape, stride or device, an empty tensor, a call that the library
// refuses): ops.py then runs its own checks on the same arguments and raises
// what it always raised.  Nothing is kept between calls.  The interpreter lock is
// released from the checks to the last launch, as ctypes releases it: a launch
// queue that is full, or the first SwiGLU call's wait for its table, holds up no
// other thread of the program.
//
// What it saves is the host's time per call, which bounds every call of a few
// dozen rows (measured on an MI355X host, Python wrapper -> this: quantizer 11.1
// -> 5.7 us, scaled GEMM 13.7 -> 5.5 us, of which the launch itself is about 3).
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>

#include "../../include/taomate_h3_amd.h"

using at::Tensor;
using Opt = std::optional<Tensor>;
using OptInt = std::optional<int64_t>;
using Pair = std::tuple<Tensor, Tensor>;
using Three = std::tuple<Tensor, Tensor, Tensor>;
using Triple = std::tuple<Opt, Opt, Opt>;

namespace {

bool on(const Tensor& t, const Tensor& first) { return t.is_cuda() && t.device() == first.device(); }

// A 2-D tensor of the given type with unit stride along its rows.
bool rows_2d(const Tensor& t, at::ScalarType type) {
    return t.scalar_type() == type && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1);
}

at::ScalarType code_type(int64_t fmt) { return fmt == H3Q_FMT_INT8 ? at::kChar : at::kFloat8_e4m3fn; }

bool valid_fmt(int64_t fmt) { return fmt == H3Q_FMT_INT8 || fmt == H3Q_FMT_E4M3FN; }

Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
    return at::empty(shape, like.options().dtype(type));
}

bool scales_ok(const Tensor& s, const Tensor& first, int64_t count) {
    return on(s, first) && s.scalar_type() == at::kFloat && s.numel() == count && s.is_contiguous();
}

void* stream_of(int64_t raw) { return reinterpret_cast<void*>(raw); }

float* floats(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }

const void* ptr(const Opt& t) { return t ? t->data_ptr() : nullptr; }

std::optional<Pair> quant_rows(const Tensor& x, int64_t fmt, int64_t rounding, Opt codes, Opt scales, int64_t stream) {
    if (!x.is_cuda() || !rows_2d(x, at::kBFloat16) || !valid_fmt(fmt) || x.size(0) == 0) return std::nullopt;
    const int64_t rows = x.size(0), cols = x.size(1);
    if (codes && !(on(*codes, x) && rows_2d(*codes, code_type(fmt)) && codes->size(0) == rows && codes->size(1) == cols))
        return std::nullopt;
    if (scales && !scales_ok(*scales, x, rows)) return std::nullopt;
    if (!codes) codes = empty(x, {rows, cols}, code_type(fmt));
    if (!scales) scales = empty(x, {rows, 1}, at::kFloat);
    if (h3q_quant_rows(x.data_ptr(), rows, cols, x.stride(0), (int)fmt, (int)rounding, codes->data_ptr(),
                       codes->stride(0), floats(*scales), stream_of(stream)))
        return std::nullopt;
    return Pair(*codes, *scales);
}

std::optional<Pair> quant_rows_tiled(const Tensor& x, int64_t fmt, int64_t rounding, Opt codes, int64_t row0,
                                     Opt scales, int64_t stream) {
    if (!x.is_cuda() || !rows_2d(x, at::kBFloat16) || !valid_fmt(fmt) || x.size(0) == 0) return std::nullopt;
    const int64_t rows = x.size(0), cols = x.size(1);
    if (cols % 128 || row0 < 0 || (!codes && row0)) return std::nullopt;
    if (codes && !(on(*codes, x) && codes->scalar_type() == code_type(fmt) && codes->dim() == 2 &&
                   codes->size(1) == cols && codes->is_contiguous() && codes->size(0) % 16 == 0 &&
                   row0 + rows <= codes->size(0)))
        return std::nullopt;
    if (scales && !scales_ok(*scales, x, rows)) return std::nullopt;
    if (!codes) codes = empty(x, {(rows + 15) / 16 * 16, cols}, code_type(fmt));
    if (!scales) scales = empty(x, {rows, 1}, at::kFloat);
    if (h3q_quant_rows_tiled(x.data_ptr(), rows, cols, x.stride(0), (int)fmt, (int)rounding, row0, codes->data_ptr(),
                             floats(*scales), stream_of(stream)))
        return std::nullopt;
    return Pair(*codes, *scales);
}

// Per row, per tensor, or -1 for neither.
int scale_kind(const Tensor& s, const Tensor& first, int64_t count) {
    if (!on(s, first) || s.scalar_type() != at::kFloat || !s.is_contiguous()) return -1;
    if (s.numel() == 1 && count != 1) return H3Q_SCALE_PER_TENSOR;
    return s.numel() == count ? H3Q_SCALE_PER_ROW : -1;
}

// rows_a, rows_b: the logical row counts where they are not those of a and b.
Opt scaled_mm(const Tensor& a, const Tensor& b, const Tensor& a_scale, const Tensor& b_scale, const Opt& bias,
              const Opt& lora_t, const Opt& lora_b, double lora_scale, Opt out, bool a_tiled, bool b_tiled, OptInt rows_a,
              OptInt rows_b, bool f16, int64_t stream) {
    const at::ScalarType type = a.scalar_type();
    if (!a.is_cuda() || (type != at::kChar && type != at::kFloat8_e4m3fn) || !on(b, a)) return std::nullopt;
    if (!rows_2d(a, type) || !rows_2d(b, type) || b.size(1) != a.size(1)) return std::nullopt;
    const int64_t k = a.size(1), m = rows_a.value_or(a.size(0)), n = rows_b.value_or(b.size(0));
    if (m <= 0 || n <= 0) return std::nullopt;
    const auto held = [](const Tensor& t, int64_t rows, bool tiled) {
        return t.size(0) >= (tiled ? (rows + 15) / 16 * 16 : rows) && (!tiled || t.is_contiguous());
    };
    if (!held(a, m, a_tiled) || !held(b, n, b_tiled)) return std::nullopt;
    const int ak = scale_kind(a_scale, a, m), bk = scale_kind(b_scale, a, n);
    if (ak < 0 || bk < 0) return std::nullopt;
    const at::ScalarType out_type = f16 ? at::kHalf : at::kBFloat16;
    if (bias && !(on(*bias, a) && bias->scalar_type() == out_type && bias->numel() == n && bias->is_contiguous()))
        return std::nullopt;
    if (lora_t.has_value() != lora_b.has_value()) return std::nullopt;
    int64_t rank = 0;
    if (lora_t) {
        if (!on(*lora_t, a) || !on(*lora_b, a) || !rows_2d(*lora_t, at::kBFloat16) || !rows_2d(*lora_b, at::kBFloat16))
            return std::nullopt;
        rank = lora_t->size(1);
        if (lora_t->size(0) != m || lora_b->size(0) != n || lora_b->size(1) != rank) return std::nullopt;
    }
    if (out && !(on(*out, a) && rows_2d(*out, out_type) && out->size(0) == m && out->size(1) == n)) return std::nullopt;
    if (!out) out = empty(a, {m, n}, out_type);
    const int fmt = (type == at::kChar ? H3Q_FMT_INT8 : H3Q_FMT_E4M3FN) | (f16 ? H3Q_OUT_F16 : 0);
    if (h3q_scaled_mm(fmt, a.data_ptr(), a.stride(0), a_tiled ? H3Q_LAYOUT_TILED : H3Q_LAYOUT_ROWS, floats(a_scale), ak,
                      b.data_ptr(), b.stride(0), b_tiled ? H3Q_LAYOUT_TILED : H3Q_LAYOUT_ROWS, floats(b_scale), bk,
                      ptr(bias), ptr(lora_t), lora_t ? lora_t->stride(0) : 0, ptr(lora_b),
                      lora_b ? lora_b->stride(0) : 0, rank, (float)lora_scale, out->data_ptr(), out->stride(0), m, n, k,
                      stream_of(stream)))
        return std::nullopt;
    return out;
}

Opt lora_down(const Tensor& x, const Tensor& lora_a, Opt out, int64_t stream) {
    if (!x.is_cuda() || !on(lora_a, x) || !rows_2d(x, at::kBFloat16) || !rows_2d(lora_a, at::kBFloat16)) return std::nullopt;
    const int64_t m = x.size(0), k = x.size(1), rank = lora_a.size(0);
    if (m == 0 || lora_a.size(1) != k) return std::nullopt;
    if (out && !(on(*out, x) && rows_2d(*out, at::kBFloat16) && out->size(0) >= m && out->size(1) >= rank))
        return std::nullopt;
    if (!out) out = empty(x, {m, rank}, at::kBFloat16);
    const int64_t bytes = h3q_lora_down_workspace_bytes(m, k, rank);
    int rc;
    if (bytes == 0) {
        rc = h3q_lora_down(x.data_ptr(), x.stride(0), lora_a.data_ptr(), lora_a.stride(0), out->data_ptr(),
                           out->stride(0), m, k, rank, stream_of(stream));
    } else {  // from torch's allocator: reused in stream order, kept by a graph capture
        const Tensor ws = empty(x, {bytes}, at::kByte);
        rc = h3q_lora_down_ws(x.data_ptr(), x.stride(0), lora_a.data_ptr(), lora_a.stride(0), out->data_ptr(),
                              out->stride(0), m, k, rank, ws.data_ptr(), bytes, stream_of(stream));
    }
    if (rc) return std::nullopt;
    return out;
}

// A [T, cols] bf16 modulation table; its row stride, or -1.
int64_t table_stride(const Tensor& t, const Tensor& first, int64_t cols) {
    if (!on(t, first) || !rows_2d(t, at::kBFloat16) || t.size(1) != cols) return -1;
    const int64_t stride = t.size(0) > 1 ? t.stride(0) : cols;
    return stride % 8 ? -1 : stride;
}

// No fmt: no codes.  Returns (out, codes, scales), None for those not wanted.  gated:
// (branch, gate, hidden).
std::optional<Triple> norm_modulate_quant(const Tensor& value, const Tensor& weight, const Tensor& scale,
                                          const Tensor& shift, const Tensor& indices, double eps, OptInt fmt,
                                          int64_t rounding, bool want_out, const std::optional<Three>& gated,
                                          int64_t stream) {
    if (!value.is_cuda() || !rows_2d(value, at::kBFloat16) || value.size(0) == 0) return std::nullopt;
    const int64_t rows = value.size(0), cols = value.size(1);
    if (!on(weight, value) || weight.scalar_type() != at::kBFloat16 || weight.numel() != cols || !weight.is_contiguous())
        return std::nullopt;
    const int64_t stride = table_stride(scale, value, cols);
    if (stride < 0 || table_stride(shift, value, cols) != stride) return std::nullopt;
    if (!on(indices, value) || indices.scalar_type() != at::kLong || indices.numel() != rows || !indices.is_contiguous())
        return std::nullopt;
    if (fmt ? !valid_fmt(*fmt) : !want_out) return std::nullopt;
    const auto matrix = [&](const Tensor& t) {
        return on(t, value) && rows_2d(t, at::kBFloat16) && t.size(0) == rows && t.size(1) == cols;
    };
    const Tensor none;
    const auto& [branch, gate, hidden] = gated ? *gated : Three(none, none, none);
    if (gated && !(matrix(branch) && matrix(hidden) && table_stride(gate, value, cols) == stride)) return std::nullopt;
    Opt out, codes, scales;
    if (want_out) out = empty(value, {rows, cols}, at::kBFloat16);
    if (fmt) {
        codes = empty(value, {rows, cols}, code_type(*fmt));
        scales = empty(value, {rows, 1}, at::kFloat);
    }
    const auto ld = [&](const Tensor& t) { return rows > 1 ? t.stride(0) : cols; };
    const int f = (int)fmt.value_or(H3Q_FMT_INT8);
    void* const out_p = out ? out->data_ptr() : nullptr;
    void* const codes_p = codes ? codes->data_ptr() : nullptr;
    float* const scales_p = scales ? floats(*scales) : nullptr;
    const int64_t* const idx = static_cast<const int64_t*>(indices.data_ptr());
    const int rc =
        gated ? h3q_residual_gate_rms_norm_modulate_quant(
                    value.data_ptr(), ld(value), branch.data_ptr(), ld(branch), gate.data_ptr(), weight.data_ptr(),
                    scale.data_ptr(), shift.data_ptr(), stride, idx, rows, cols, (float)eps, hidden.data_ptr(),
                    ld(hidden), out_p, cols, f, (int)rounding, codes_p, cols, scales_p, stream_of(stream))
              : h3q_rms_norm_modulate_quant(value.data_ptr(), ld(value), weight.data_ptr(), scale.data_ptr(),
                                            shift.data_ptr(), stride, idx, rows, cols, (float)eps, out_p, cols, f,
                                            (int)rounding, codes_p, cols, scales_p, stream_of(stream));
    if (rc) return std::nullopt;
    return Triple(out, codes, scales);
}

std::optional<Triple> swiglu_quant(const Tensor& x, OptInt fmt, int64_t rounding, bool want_out, int64_t stream) {
    if (!x.is_cuda() || !rows_2d(x, at::kBFloat16) || x.size(0) == 0 || x.size(1) % 2) return std::nullopt;
    if (fmt ? !valid_fmt(*fmt) : !want_out) return std::nullopt;
    const int64_t rows = x.size(0), half = x.size(1) / 2;
    Opt out, codes, scales;
    if (want_out) out = empty(x, {rows, half}, at::kBFloat16);
    if (fmt) {
        codes = empty(x, {rows, half}, code_type(*fmt));
        scales = empty(x, {rows, 1}, at::kFloat);
    }
    if (h3q_swiglu_quant(x.data_ptr(), rows > 1 ? x.stride(0) : 2 * half, rows, half, out ? out->data_ptr() : nullptr,
                         half, (int)fmt.value_or(H3Q_FMT_INT8), (int)rounding, codes ? codes->data_ptr() : nullptr,
                         half, scales ? floats(*scales) : nullptr, stream_of(stream)))
        return std::nullopt;
    return Triple(out, codes, scales);
}

std::optional<Pair> quant_per_head(const Tensor& x, int64_t stream) {
    if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || x.dim() != 4 || !x.is_contiguous() || x.numel() == 0)
        return std::nullopt;
    const int64_t b = x.size(0), s = x.size(1), h = x.size(2), d = x.size(3);
    const Tensor codes = empty(x, x.sizes(), at::kFloat8_e4m3fn), scales = empty(x, {b, h}, at::kFloat);
    const Tensor ws = empty(x, {h3q_quant_per_head_workspace_floats(b, s, h, d)}, at::kFloat);
    if (h3q_quant_per_head_e4m3(x.data_ptr(), b, s, h, d, floats(ws), codes.data_ptr(), floats(scales),
                                stream_of(stream)))
        return std::nullopt;
    return Pair(codes, scales);
}

std::optional<Pair> quant_tensor(const Tensor& x, const Opt& static_scale, bool eager, int64_t stream) {
    const at::ScalarType type = x.scalar_type();
    if (!x.is_cuda() || x.numel() == 0 || x.dim() < 1 || !x.is_contiguous()) return std::nullopt;
    const int dtype = type == at::kBFloat16 ? H3Q_DTYPE_BF16 : type == at::kHalf ? H3Q_DTYPE_F16
                      : type == at::kFloat ? H3Q_DTYPE_F32 : -1;
    if (dtype < 0) return std::nullopt;
    if (static_scale && !scales_ok(*static_scale, x, 1)) return std::nullopt;
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    const Tensor codes = empty(x, x.sizes(), at::kFloat8_e4m3fn), scale = empty(x, {}, at::kFloat);
    Opt ws;
    if (!static_scale) ws = empty(x, {h3q_quant_tensor_workspace_floats(rows, cols)}, at::kFloat);
    if (h3q_quant_tensor_e4m3_typed(x.data_ptr(), dtype, eager ? H3Q_QUOTIENT_EAGER : H3Q_QUOTIENT_TRITON, rows, cols,
                                    cols, static_scale ? floats(*static_scale) : nullptr, ws ? floats(*ws) : nullptr,
                                    codes.data_ptr(), cols, floats(scale), stream_of(stream)))
        return std::nullopt;
    return Pair(codes, scale);
}

// Elements between rows; a single row has the width's, rounded up to 16.
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 16 * 16; }

// A contiguous tensor of the given type beside `first`.
bool dense(const Tensor& t, const Tensor& first, at::ScalarType type) {
    return on(t, first) && t.scalar_type() == type && t.is_contiguous();
}

int logit_type(at::ScalarType type) {
    return type == at::kBFloat16 ? H3Q_DTYPE_BF16 : type == at::kHalf ? H3Q_DTYPE_F16 : type == at::kFloat ? H3Q_DTYPE_F32 : -1;
}

int32_t* ints(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

std::optional<Pair> route_experts(const Tensor& logits, int64_t top_k, int64_t scoring, bool renormalize, double scale,
                                  int64_t stream) {
    const int dtype = logit_type(logits.scalar_type());
    if (!logits.is_cuda() || dtype < 0 || !rows_2d(logits, logits.scalar_type()) || logits.size(0) == 0) return std::nullopt;
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    if (top_k < 1 || top_k > experts) return std::nullopt;
    const c10::DeviceGuard guard(logits.device());
    const Tensor ids = empty(logits, {tokens, top_k}, at::kInt), weights = empty(logits, {tokens, top_k}, at::kFloat);
    if (h3q_route_topk(logits.data_ptr(), dtype, tokens > 1 ? logits.stride(0) : experts, tokens, experts, top_k,
                       (int)scoring, renormalize, (float)scale, ints(ids), floats(weights), stream_of(stream)))
        return std::nullopt;
    return Pair(ids, weights);
}

std::optional<Three> plan_experts(const Tensor& experts, int64_t n_experts, int64_t first, int64_t stream) {
    if (!experts.is_cuda() || !dense(experts, experts, at::kInt) || experts.dim() != 2 || experts.numel() == 0 ||
        n_experts < 1 || n_experts > 1024)
        return std::nullopt;
    const int64_t tokens = experts.size(0), top_k = experts.size(1);
    const c10::DeviceGuard guard(experts.device());
    const Tensor order = empty(experts, {tokens * top_k}, at::kInt), offsets = empty(experts, {n_experts + 1}, at::kInt);
    const Tensor slots = empty(experts, {tokens, top_k}, at::kInt);
    const int64_t bytes = h3q_plan_experts_workspace_bytes(tokens, top_k, n_experts);
    Opt ws;
    if (bytes > 0) ws = empty(experts, {bytes}, at::kByte);
    if (h3q_plan_experts(ints(experts), tokens, top_k, first, n_experts, ints(order), ints(offsets), ints(slots),
                         ws ? ws->data_ptr() : nullptr, bytes, stream_of(stream)))
        return std::nullopt;
    return Three(order, offsets, slots);
}

Opt grouped_scaled_mm(const Tensor& a, const Tensor& b, const Tensor& a_scale, const Tensor& b_scale,
                      const Tensor& offsets, const Opt& order, int64_t top_k, bool swiglu, bool b_tiled, Opt out, bool f32,
                      int64_t stream) {
    const at::ScalarType type = a.scalar_type();
    if (!a.is_cuda() || (type != at::kChar && type != at::kFloat8_e4m3fn) || !rows_2d(a, type)) return std::nullopt;
    if (!dense(b, a, type) || b.dim() != 3 || b.size(2) != a.size(1)) return std::nullopt;
    const int64_t experts = b.size(0), n = b.size(1), k = b.size(2);
    if (!scales_ok(a_scale, a, a.size(0)) || !scales_ok(b_scale, a, experts * n)) return std::nullopt;
    if (!dense(offsets, a, at::kInt) || offsets.dim() != 1 || offsets.size(0) != experts + 1) return std::nullopt;
    if (order && (!dense(*order, a, at::kInt) || order->dim() != 1)) return std::nullopt;
    if (swiglu && f32) return std::nullopt;
    const int64_t rows = order ? order->size(0) : a.size(0), cols = swiglu ? n / 2 : n;
    const at::ScalarType out_type = f32 ? at::kFloat : at::kBFloat16;
    if (out && !(on(*out, a) && rows_2d(*out, out_type) && out->size(0) == rows && out->size(1) == cols))
        return std::nullopt;
    const c10::DeviceGuard guard(a.device());
    if (!out) out = empty(a, {rows, cols}, out_type);
    if (h3q_grouped_mm(type == at::kChar ? H3Q_FMT_INT8 : H3Q_FMT_E4M3FN, a.data_ptr(), row_stride(a), a.size(0),
                       floats(a_scale), order ? ints(*order) : nullptr, top_k, b.data_ptr(),
                       b_tiled ? H3Q_LAYOUT_TILED : H3Q_LAYOUT_ROWS, floats(b_scale), ints(offsets), experts, rows, n, k,
                       swiglu, f32, out->data_ptr(), row_stride(*out), stream_of(stream)))
        return std::nullopt;
    return out;
}

Opt combine_experts(const Tensor& y, const Tensor& slots, const Tensor& weights, Opt out, int64_t stream) {
    const at::ScalarType type = y.scalar_type();
    if (!y.is_cuda() || (type != at::kBFloat16 && type != at::kFloat) || !rows_2d(y, type)) return std::nullopt;
    if (!dense(slots, y, at::kInt) || slots.dim() != 2 || !dense(weights, y, at::kFloat) ||
        weights.sizes() != slots.sizes())
        return std::nullopt;
    const int64_t tokens = slots.size(0), top_k = slots.size(1), cols = y.size(1);
    if (out && !(on(*out, y) && rows_2d(*out, at::kBFloat16) && out->size(0) == tokens && out->size(1) == cols))
        return std::nullopt;
    const c10::DeviceGuard guard(y.device());
    if (!out) out = empty(y, {tokens, cols}, at::kBFloat16);
    if (h3q_combine_experts(y.data_ptr(), type == at::kFloat, row_stride(y), y.size(0), ints(slots), floats(weights),
                            tokens, top_k, cols, out->data_ptr(), row_stride(*out), stream_of(stream)))
        return std::nullopt;
    return out;
}

Opt expert_ffn(const Tensor& x, const Tensor& experts, const Tensor& weights, const Tensor& w13, const Tensor& w13_scale,
               const Tensor& w2, const Tensor& w2_scale, int64_t first, bool w13_tiled, bool w2_tiled, Opt out,
               int64_t stream) {
    if (!x.is_cuda() || !rows_2d(x, at::kBFloat16) || x.size(0) == 0) return std::nullopt;
    const int64_t tokens = x.size(0), d = x.size(1);
    if (!dense(experts, x, at::kInt) || experts.dim() != 2 || experts.size(0) != tokens ||
        !dense(weights, x, at::kFloat) || weights.sizes() != experts.sizes())
        return std::nullopt;
    const at::ScalarType type = w13.scalar_type();
    if ((type != at::kChar && type != at::kFloat8_e4m3fn) || !dense(w13, x, type) || !dense(w2, x, type))
        return std::nullopt;
    if (w13.dim() != 3 || w13.size(1) % 2 || w13.size(2) != d || w2.dim() != 3) return std::nullopt;
    const int64_t count = w13.size(0), f = w13.size(1) / 2, top_k = experts.size(1);
    if (w2.size(0) != count || w2.size(1) != d || w2.size(2) != f) return std::nullopt;
    if (!scales_ok(w13_scale, x, count * 2 * f) || !scales_ok(w2_scale, x, count * d)) return std::nullopt;
    if (out && !(on(*out, x) && rows_2d(*out, at::kBFloat16) && out->size(0) == tokens && out->size(1) == d))
        return std::nullopt;
    const c10::DeviceGuard guard(x.device());
    if (!out) out = empty(x, {tokens, d}, at::kBFloat16);
    const int64_t bytes = h3q_expert_ffn_workspace_bytes(tokens, top_k, count, d, f);
    const Tensor ws = empty(x, {bytes}, at::kByte);  // from torch's allocator, as in lora_down
    if (h3q_expert_ffn(type == at::kChar ? H3Q_FMT_INT8 : H3Q_FMT_E4M3FN, x.data_ptr(), row_stride(x), tokens, d, f,
                       ints(experts), floats(weights), top_k, first, count, w13.data_ptr(),
                       w13_tiled ? H3Q_LAYOUT_TILED : H3Q_LAYOUT_ROWS, floats(w13_scale), w2.data_ptr(),
                       w2_tiled ? H3Q_LAYOUT_TILED : H3Q_LAYOUT_ROWS, floats(w2_scale), out->data_ptr(),
                       row_stride(*out), ws.data_ptr(), bytes, stream_of(stream)))
        return std::nullopt;
    return out;
}

// ---- rotary positions, head norms, paged cache

bool head_rows(const Tensor& t, const Tensor& first, at::ScalarType type) {
    return on(t, first) && t.scalar_type() == type && t.dim() == 3 && (t.size(2) <= 1 || t.stride(2) == 1);
}

// Whether no two elements share memory.
bool apart(const Tensor& t) {
    int64_t stride[4], size[4], n = 0;
    if (t.dim() > 4) return false;
    for (int64_t i = 0; i < t.dim(); ++i) {
        if (t.size(i) <= 1) continue;
        int64_t at = n++;
        for (; at > 0 && stride[at - 1] > t.stride(i); --at) stride[at] = stride[at - 1], size[at] = size[at - 1];
        stride[at] = t.stride(i), size[at] = t.size(i);
    }
    int64_t reach = 0;
    for (int64_t i = 0; i < n; ++i) {
        if (stride[i] <= reach) return false;
        reach += stride[i] * (size[i] - 1);
    }
    return true;
}

// The rows, their norm's weights and where they go; false: something is out of the ordinary.
bool heads_of(h3q_heads& h, const Tensor& x, const Opt& weight, const Tensor* out, int& weight_dtype) {
    const int64_t heads = x.size(1), d = x.size(2);
    h = {};
    h.x = x.data_ptr();
    h.token_stride = x.stride(0);
    h.head_stride = x.stride(1);
    h.heads = heads;
    if (weight) {
        const at::ScalarType type = weight->scalar_type();
        if (!on(*weight, x) || (type != x.scalar_type() && type != at::kFloat)) return false;
        const int kind = logit_type(type);
        if (weight_dtype >= 0 && weight_dtype != kind) return false;
        weight_dtype = kind;
        const bool each = weight->dim() == 2 && weight->size(0) == heads && weight->size(1) == d;
        if (!each && !(weight->dim() == 1 && weight->size(0) == d)) return false;
        if (d > 1 && weight->stride(-1) != 1) return false;
        h.weight = weight->data_ptr();
        h.weight_stride = each ? weight->stride(0) : 0;
    }
    if (out) {
        h.out = out->data_ptr();
        h.out_token_stride = out->stride(0);
        h.out_head_stride = out->stride(1);
    }
    return true;
}

bool rotation_of(h3q_rotation& r, const Tensor& x, const Tensor& cos, const Tensor& sin, const Opt& positions,
                 bool interleaved, bool inverse) {
    if (!dense(cos, x, at::kFloat) || !dense(sin, x, at::kFloat) || cos.dim() != 2 || sin.sizes() != cos.sizes())
        return false;
    r = {};
    r.cos = floats(cos);
    r.sin = floats(sin);
    r.rows = cos.size(0);
    r.rot_dim = 2 * cos.size(1);
    r.interleaved = interleaved;
    r.inverse = inverse;
    if (positions) {
        const at::ScalarType type = positions->scalar_type();
        if ((type != at::kInt && type != at::kLong) || !dense(*positions, x, type) || positions->dim() != 1 ||
            positions->size(0) != x.size(0))
            return false;
        r.positions = positions->data_ptr();
        r.positions_i64 = type == at::kLong;
    }
    return true;
}

// out as given, or a new tensor; false: it does not fit.
bool rows_like(const Tensor& x, Opt& out) {
    if (!out) {
        out = empty(x, x.sizes(), x.scalar_type());
        return true;
    }
    return head_rows(*out, x, x.scalar_type()) && out->sizes() == x.sizes() && apart(*out);
}

std::optional<Pair> rotary_tables(const Tensor& positions, const Tensor& frequencies, double magnitude, int64_t stream) {
    const at::ScalarType type = positions.scalar_type();
    const int kind = type == at::kInt     ? H3Q_POSITIONS_I32
                     : type == at::kLong  ? H3Q_POSITIONS_I64
                     : type == at::kFloat ? H3Q_POSITIONS_F32
                     : type == at::kDouble ? H3Q_POSITIONS_F64
                                           : -1;
    if (!positions.is_cuda() || kind < 0 || !positions.is_contiguous() || positions.dim() != 1 ||
        !dense(frequencies, positions, at::kDouble) || frequencies.dim() != 1 || positions.size(0) == 0)
        return std::nullopt;
    const int64_t n = positions.size(0), half = frequencies.size(0);
    if (half < 1 || half > 256 || n >= (int64_t(1) << 31) / half) return std::nullopt;
    const c10::DeviceGuard guard(positions.device());
    const Tensor cos = empty(positions, {n, half}, at::kFloat), sin = empty(positions, {n, half}, at::kFloat);
    if (h3q_rotary_tables(positions.data_ptr(), kind, n, static_cast<const double*>(frequencies.data_ptr()), half,
                          magnitude, floats(cos), floats(sin), stream_of(stream)))
        return std::nullopt;
    return Pair(cos, sin);
}

Opt rotary(const Tensor& x, const Tensor& cos, const Tensor& sin, const Opt& positions, bool interleaved, bool inverse,
           Opt out, int64_t stream) {
    const int dtype = logit_type(x.scalar_type());
    if (!x.is_cuda() || dtype < 0 || !head_rows(x, x, x.scalar_type()) || x.numel() == 0) return std::nullopt;
    h3q_rotation r;
    h3q_heads h;
    int weight_dtype = -1;
    if (!rotation_of(r, x, cos, sin, positions, interleaved, inverse)) return std::nullopt;
    const c10::DeviceGuard guard(x.device());
    if (!rows_like(x, out) || !heads_of(h, x, std::nullopt, &*out, weight_dtype)) return std::nullopt;
    if (h3q_rotary(dtype, &h, x.size(0), x.size(2), &r, stream_of(stream))) return std::nullopt;
    return out;
}

std::optional<Pair> qk_norm_rotary(const Tensor& q, const Tensor& k, const Opt& q_weight, const Opt& k_weight,
                                   const Tensor& cos, const Tensor& sin, const Opt& positions, double eps,
                                   bool interleaved, Opt q_out, Opt k_out, int64_t stream) {
    const int dtype = logit_type(q.scalar_type());
    if (!q.is_cuda() || dtype < 0 || !head_rows(q, q, q.scalar_type()) || q.numel() == 0 ||
        !head_rows(k, q, q.scalar_type()) || k.size(0) != q.size(0) || k.size(2) != q.size(2))
        return std::nullopt;
    h3q_rotation r;
    h3q_heads qh, kh;
    int weight_dtype = -1;
    if (!rotation_of(r, q, cos, sin, positions, interleaved, false)) return std::nullopt;
    const c10::DeviceGuard guard(q.device());
    if (!rows_like(q, q_out) || !rows_like(k, k_out) || !heads_of(qh, q, q_weight, &*q_out, weight_dtype) ||
        !heads_of(kh, k, k_weight, &*k_out, weight_dtype))
        return std::nullopt;
    if (h3q_qk_norm_rotary(dtype, weight_dtype < 0 ? dtype : weight_dtype, &qh, &kh, q.size(0), q.size(2), (float)eps, &r,
                           stream_of(stream)))
        return std::nullopt;
    return Pair(*q_out, *k_out);
}

std::optional<Pair> plan_append(const Tensor& table, const Tensor& lengths, const Tensor& cu, int64_t tokens,
                                int64_t page_size, int64_t stream) {
    if (!table.is_cuda() || !rows_2d(table, at::kInt) || !dense(lengths, table, at::kInt) || !dense(cu, table, at::kInt))
        return std::nullopt;
    const int64_t seqs = table.size(0), columns = table.size(1);
    if (lengths.dim() != 1 || lengths.size(0) != seqs || cu.dim() != 1 || cu.size(0) != seqs + 1 || tokens < 1 ||
        tokens >= (int64_t(1) << 31))
        return std::nullopt;
    const c10::DeviceGuard guard(table.device());
    const Tensor positions = empty(table, {tokens}, at::kInt), slots = empty(table, {tokens}, at::kInt);
    if (h3q_plan_append(ints(table), seqs > 1 ? table.stride(0) : columns, seqs, columns, ints(lengths), ints(cu), tokens,
                        page_size, ints(positions), ints(slots), stream_of(stream)))
        return std::nullopt;
    return Pair(positions, slots);
}

bool pages_of(h3q_pages& p, const Tensor& x, const Tensor& pages, const Opt& scale) {
    const int64_t heads = x.size(1), d = x.size(2);
    const at::ScalarType type = pages.scalar_type();
    if (!on(pages, x) || (type != x.scalar_type() && type != at::kFloat8_e4m3fn) || pages.dim() != 4 ||
        pages.size(2) != heads || pages.size(3) != d || pages.stride(3) != 1 || !apart(pages))
        return false;
    p = {};
    p.pages = pages.data_ptr();
    p.n_pages = pages.size(0);
    p.page_size = pages.size(1);
    p.page_stride = pages.stride(0);
    p.slot_stride = pages.stride(1);
    p.head_stride = pages.stride(2);
    p.kind = H3Q_PAGES_ROWS;
    if ((type == at::kFloat8_e4m3fn) != scale.has_value()) return false;
    if (!scale) return true;
    if (!on(*scale, x) || scale->scalar_type() != at::kFloat) return false;
    p.scale = floats(*scale);
    if (scale->dim() == 1 && (scale->size(0) == 1 || scale->size(0) == heads)) {
        p.kind = H3Q_PAGES_STATIC;
        p.scale_head_stride = scale->size(0) > 1 ? scale->stride(0) : 0;
        return true;
    }
    if (scale->dim() != 3 || scale->size(0) != p.n_pages || scale->size(1) != p.page_size || scale->size(2) != heads ||
        !apart(*scale))
        return false;
    p.kind = H3Q_PAGES_BY_ROW;
    p.scale_page_stride = scale->stride(0);
    p.scale_slot_stride = scale->stride(1);
    p.scale_head_stride = scale->stride(2);
    return true;
}

// q's output (k where there is no q), or nothing.
Opt append_kv(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& slots,
              const Opt& k_scale, const Opt& v_scale, const Opt& k_weight, double eps, const Opt& cos, const Opt& sin,
              const Opt& positions, bool interleaved, const Opt& q, const Opt& q_weight, Opt q_out, int64_t stream) {
    const at::ScalarType type = k.scalar_type();
    const int dtype = logit_type(type);
    if (!k.is_cuda() || dtype < 0 || !head_rows(k, k, type) || k.numel() == 0 || !head_rows(v, k, type) ||
        v.sizes() != k.sizes() || !dense(slots, k, at::kInt) || slots.dim() != 1 || slots.size(0) != k.size(0))
        return std::nullopt;
    if (cos.has_value() != sin.has_value() || (positions && !cos) || (!q && (q_weight || q_out))) return std::nullopt;
    const auto same = [](const Tensor& a, const Tensor& b) { return a.numel() > 0 && a.data_ptr() == b.data_ptr(); };
    if (same(k_pages, v_pages) || (k_scale && v_scale && k_scale->dim() == 3 && same(*k_scale, *v_scale)))
        return std::nullopt;
    h3q_rotation r;
    if (cos && !rotation_of(r, k, *cos, *sin, positions, interleaved, false)) return std::nullopt;
    h3q_heads qh, kh, vh;
    h3q_pages kp, vp;
    int weight_dtype = -1;
    const c10::DeviceGuard guard(k.device());
    if (q) {
        if (!head_rows(*q, k, type) || q->size(0) != k.size(0) || q->size(2) != k.size(2) || !rows_like(*q, q_out) ||
            !heads_of(qh, *q, q_weight, &*q_out, weight_dtype))
            return std::nullopt;
    }
    if (!heads_of(kh, k, k_weight, nullptr, weight_dtype) || !heads_of(vh, v, std::nullopt, nullptr, weight_dtype) ||
        !pages_of(kp, k, k_pages, k_scale) || !pages_of(vp, v, v_pages, v_scale))
        return std::nullopt;
    if (h3q_append_kv(dtype, weight_dtype < 0 ? dtype : weight_dtype, q ? &qh : nullptr, &kh, &vh, &kp, &vp, ints(slots),
                      k.size(0), k.size(2), (float)eps, cos ? &r : nullptr, stream_of(stream)))
        return std::nullopt;
    return q ? q_out : Opt(k);
}

Opt w4_mm(const Tensor& x, const Tensor& codes, const Tensor& scales, const Opt& zeros, int64_t n, int64_t k,
          int64_t group, const Opt& bias, Opt out, int64_t stream) {
    const at::ScalarType type = x.scalar_type(), scale_type = scales.scalar_type();
    if (!x.is_cuda() || (type != at::kBFloat16 && type != at::kHalf) || !rows_2d(x, type) || x.size(1) != k ||
        x.size(0) == 0 || n < 1 || k < 16 || group < 32)
        return std::nullopt;
    const int64_t m = x.size(0), blocks = (n + 15) / 16, quads = ((k + group - 1) / group + 3) / 4;
    const auto packed = [&](const Tensor& t, at::ScalarType of) {
        return dense(t, x, of) && t.dim() == 4 && t.size(0) == blocks && t.size(1) == quads && t.size(2) == 16 &&
               t.size(3) == 4;
    };
    if ((scale_type != at::kBFloat16 && scale_type != at::kHalf) || !dense(codes, x, at::kByte) || codes.dim() != 3 ||
        codes.size(0) != blocks || codes.size(1) != (k + 127) / 128 || codes.size(2) != 1024 ||
        !packed(scales, scale_type) || (zeros && !packed(*zeros, at::kByte)))
        return std::nullopt;
    if (bias && !(dense(*bias, x, type) && bias->dim() == 1 && bias->size(0) == n)) return std::nullopt;
    if (out && !(on(*out, x) && rows_2d(*out, type) && out->size(0) == m && out->size(1) == n && apart(*out)))
        return std::nullopt;
    const c10::DeviceGuard guard(x.device());
    if (!out) out = empty(x, {m, n}, type);
    const int64_t bytes = h3q_w4_mm_workspace_bytes(m, n, k, group);
    Opt ws;
    if (bytes > 0) ws = empty(x, {bytes}, at::kByte);
    if (h3q_w4_mm(logit_type(type), x.data_ptr(), m > 1 ? x.stride(0) : (k + 7) / 8 * 8, codes.data_ptr(),
                  scales.data_ptr(), logit_type(scale_type), ptr(zeros), group, ptr(bias), out->data_ptr(),
                  m > 1 ? out->stride(0) : n, m, n, k, ws ? ws->data_ptr() : nullptr, bytes, stream_of(stream)))
        return std::nullopt;
    return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("quant_rows", torch::wrap_pybind_function_no_gil(&quant_rows));
    m.def("quant_rows_tiled", torch::wrap_pybind_function_no_gil(&quant_rows_tiled));
    m.def("scaled_mm", torch::wrap_pybind_function_no_gil(&scaled_mm));
    m.def("lora_down", torch::wrap_pybind_function_no_gil(&lora_down));
    m.def("norm_modulate_quant", torch::wrap_pybind_function_no_gil(&norm_modulate_quant));
    m.def("swiglu_quant", torch::wrap_pybind_function_no_gil(&swiglu_quant));
    m.def("quant_per_head", torch::wrap_pybind_function_no_gil(&quant_per_head));
    m.def("quant_tensor", torch::wrap_pybind_function_no_gil(&quant_tensor));
    m.def("route_experts", torch::wrap_pybind_function_no_gil(&route_experts));
    m.def("plan_experts", torch::wrap_pybind_function_no_gil(&plan_experts));
    m.def("grouped_scaled_mm", torch::wrap_pybind_function_no_gil(&grouped_scaled_mm));
    m.def("combine_experts", torch::wrap_pybind_function_no_gil(&combine_experts));
    m.def("rotary_tables", torch::wrap_pybind_function_no_gil(&rotary_tables));
    m.def("rotary", torch::wrap_pybind_function_no_gil(&rotary));
    m.def("qk_norm_rotary", torch::wrap_pybind_function_no_gil(&qk_norm_rotary));
    m.def("plan_append", torch::wrap_pybind_function_no_gil(&plan_append));
    m.def("append_kv", torch::wrap_pybind_function_no_gil(&append_kv));
    m.def("w4_mm", torch::wrap_pybind_function_no_gil(&w4_mm));
    m.def("expert_ffn", torch::wrap_pybind_function_no_gil(&expert_ffn));
}
