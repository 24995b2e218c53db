// Routing of a mixture-of-experts layer, gfx950: the top-k of the router's logits, the
// plan that sorts the (token, slot) pairs by expert, and the weighted sum that brings
// the experts' rows back to their tokens.
#include "h3q_common.hpp"
#include "h3q_kernels.hpp"

namespace h3q {

namespace {

// Order of logits as unsigned integers: a larger value has a larger key, +0 and -0 the
// same one, and NaN and -inf have 0 (never taken).  Keys of finite values and +inf are
// above 0x007FFFFF.
__device__ __forceinline__ uint32_t logit_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 + 0 = +0
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return v > -__builtin_inff() ? k : 0u;  // false for NaN too
}

__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Rotation by N lanes inside each row of 16 lanes.
template <int N>
__device__ __forceinline__ uint32_t row_ror(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xF, 0xF, true);
}

// Reductions over the LPT lanes (16 or 64) of a token; every lane gets the result.
template <int LPT, class F>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, F f) {
    v = f(v, row_ror<8>(v));
    v = f(v, row_ror<4>(v));
    v = f(v, row_ror<2>(v));
    v = f(v, row_ror<1>(v));
    if constexpr (LPT == 64) {
        v = f(v, (uint32_t)__shfl_xor((int)v, 16, 64));
        v = f(v, (uint32_t)__shfl_xor((int)v, 32, 64));
    }
    return v;
}
template <int LPT>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    return group_reduce<LPT>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int LPT>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
    return group_reduce<LPT>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
template <int LPT>
__device__ __forceinline__ float group_sum(float v) {
    return __uint_as_float(group_reduce<LPT>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

template <int DT>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
    if constexpr (DT == kInF32) return ((const float*)p)[i];
    else if constexpr (DT == kInBF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    else return (float)__builtin_bit_cast(_Float16, ((const uint16_t*)p)[i]);
}

}  // namespace

// Top-k of a token's logits with their weights.
//
// A token belongs to LPT lanes (16, or 64 for many experts or slots), each holding NV
// keys; k rounds take the largest key left, the lowest expert among equals, by one
// maximum over the keys and one minimum over the experts that hold it.  Lane j keeps
// slot j.  The weights are binary32: softmax exp(l - max) / sum over all experts (or over
// the taken ones), with exp(0) = 1 for the maximum itself, an infinite one included;
// sigmoid 1 / (1 + exp(-l)), divided by the taken ones' sum when renormalized.
// A slot without an expert (fewer than k logits above -inf) gets -1 and weight 0.
//
// What bounds it: the logits are read once, in registers; the k rounds cost about
// 5 NV + 20 instructions each.  Four tokens to a wave rather than one cut the cross-lane
// steps per token by four and stay within a row of 16 lanes (register permutes).
template <int DT, int LPT, int NV>
__global__ __launch_bounds__(256) void route_topk_kernel(RouteArgs p) {
    constexpr int TPB = 256 / LPT;
    const int64_t token = (int64_t)blockIdx.x * TPB + threadIdx.x / LPT;
    const int lane = threadIdx.x % LPT;
    const bool live = token < p.tokens;
    const int64_t row = (live ? token : 0) * p.ldl;
    uint32_t key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = i * LPT + lane;
        key[i] = live && e < p.experts ? logit_key(load_logit<DT>(p.logits, row + e)) : 0u;
    }
    uint32_t local = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) local = key[i] > local ? key[i] : local;
    const uint32_t top = group_max<LPT>(local);
    const float best = key_logit(top);
    float whole = 0.0f;
    if (p.scoring == kScoreSoftmax && !p.renormalize) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (key[i] != 0u) whole += key[i] == top ? 1.0f : expf(key_logit(key[i]) - best);
        whole = group_sum<LPT>(whole);
    }
    int mine = -1;
    float weight = 0.0f;
    for (int j = 0; j < p.top_k; ++j) {
        local = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) local = key[i] > local ? key[i] : local;
        const uint32_t m = group_max<LPT>(local);
        uint32_t e = 0xFFFFFFFFu;
#pragma unroll
        for (int i = NV - 1; i >= 0; --i)
            if (key[i] == m) e = (uint32_t)(i * LPT + lane);
        e = group_min<LPT>(e);
        if (m != 0u && j == lane) {
            mine = (int)e;
            const float l = key_logit(m);
            weight = p.scoring == kScoreSigmoid ? 1.0f / (1.0f + expf(-l)) : m == top ? 1.0f : expf(l - best);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((uint32_t)(i * LPT + lane) == e) key[i] = 0u;
    }
    if (p.renormalize) whole = group_sum<LPT>(weight);
    else if (p.scoring == kScoreSigmoid) whole = 1.0f;
    if (live && lane < p.top_k) {
        p.ids[token * p.top_k + lane] = mine;
        p.weights[token * p.top_k + lane] = whole > 0.0f ? weight / whole * p.scale : 0.0f;
    }
}

namespace {

template <int DT>
hipError_t launch_route_dt(const RouteArgs& a, hipStream_t st) {
    const bool wide = a.experts > 256 || a.top_k > 16;
    const int lpt = wide ? 64 : 16;
    const dim3 grid((unsigned)((a.tokens + 256 / lpt - 1) / (256 / lpt)));
    const int nv = (int)((a.experts + lpt - 1) / lpt);
#define H3Q_ROUTE(LPT, NV) hipLaunchKernelGGL((route_topk_kernel<DT, LPT, NV>), grid, dim3(256), 0, st, a)
    if (wide) {
        if (nv <= 4) H3Q_ROUTE(64, 4);
        else H3Q_ROUTE(64, 16);
    } else {
        if (nv <= 1) H3Q_ROUTE(16, 1);
        else if (nv <= 4) H3Q_ROUTE(16, 4);
        else if (nv <= 8) H3Q_ROUTE(16, 8);
        else H3Q_ROUTE(16, 16);
    }
#undef H3Q_ROUTE
    return hipGetLastError();
}

}  // namespace

hipError_t launch_route_topk(const RouteArgs& a, int dtype, hipStream_t st) {
    if (dtype == kInF32) return launch_route_dt<kInF32>(a, st);
    if (dtype == kInBF16) return launch_route_dt<kInBF16>(a, st);
    return launch_route_dt<kInF16>(a, st);
}

// Plan of an expert layer: the pairs (token * top_k + slot) sorted by expert, in pair
// order within an expert.  Workgroup e places expert e's pairs: its waves take
// consecutive spans of the pairs, count the ones of lower experts and its own, and after
// one exchange walk their spans again and write.  No atomics, so the order is the same
// every time; no workspace, one launch.  Pairs whose expert is not in
// [first, first + experts) get slot -1 (workgroup 0), and the rows past the last placed
// one order -1 (workgroup e for rows total + e, total + e + experts, ...).
//
// What bounds it: every workgroup reads all ids twice (from the L2 after the first), so
// the latency of a span's loads for few pairs, experts * pairs * 8 bytes for many.
__global__ __launch_bounds__(1024) void plan_experts_kernel(PlanArgs p) {
    constexpr int kWaves = 16;
    __shared__ int lower[kWaves], own[kWaves], valid[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int e = blockIdx.x;
    // spans in whole 256-pair trips of a wave (4 consecutive pairs a lane)
    const int64_t trips = (p.pairs + 255) / 256;
    const int64_t t0 = trips * wave / kWaves, t1 = trips * (wave + 1) / kWaves;
    auto load = [&](int64_t t, int (&id)[4]) __attribute__((always_inline)) {
        const int64_t i = t * 256 + lane * 4;
        if (p.vec && i + 4 <= p.pairs) {
            const int4 v = *reinterpret_cast<const int4*>(p.ids + i);
            id[0] = v.x, id[1] = v.y, id[2] = v.z, id[3] = v.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) id[c] = i + c < p.pairs ? p.ids[i + c] : -1;
        }
        // expert of this plan, or `experts` for none (ids below 0 or outside the range;
        // the difference is taken unsigned, so no id wraps into the range)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t r = (uint32_t)id[c] - (uint32_t)p.first;
            id[c] = id[c] >= 0 && id[c] >= p.first && r < (uint32_t)p.experts ? (int)r : p.experts;
        }
    };
    int n_lower = 0, n_own = 0, n_valid = 0;
    for (int64_t t = t0; t < t1; ++t) {
        int id[4];
        load(t, id);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            n_lower += __popcll(__ballot(id[c] < e));
            n_own += __popcll(__ballot(id[c] == e));
            n_valid += __popcll(__ballot(id[c] < p.experts));
        }
    }
    if (lane == 0) {
        lower[wave] = n_lower;
        own[wave] = n_own;
        valid[wave] = n_valid;
    }
    __syncthreads();
    int base = 0, before = 0, count = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        base += lower[w];
        if (w < wave) before += own[w];
        count += own[w];
        total += valid[w];
    }
    if (threadIdx.x == 0) {
        p.offsets[e] = base;
        if (e == p.experts - 1) p.offsets[p.experts] = base + count;
    }
    int pos = base + before;
    for (int64_t t = t0; t < t1; ++t) {
        int id[4];
        load(t, id);
        uint64_t b[4];
        int rank = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            b[c] = __ballot(id[c] == e);
            rank += __popcll(b[c] & ((uint64_t(1) << lane) - 1));
        }
        const int64_t i = t * 256 + lane * 4;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (id[c] == e) {
                p.order[pos + rank] = (int)(i + c);
                p.slots[i + c] = pos + rank;
                ++rank;
            } else if (e == 0 && id[c] == p.experts && i + c < p.pairs) {
                p.slots[i + c] = -1;
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) pos += __popcll(b[c]);
    }
    for (int64_t i = total + e + (int64_t)threadIdx.x * p.experts; i < p.pairs; i += 1024 * (int64_t)p.experts)
        p.order[i] = -1;
}

hipError_t launch_plan_experts(const PlanArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(plan_experts_kernel, dim3((unsigned)a.experts), dim3(1024), 0, st, a);
    return hipGetLastError();
}

namespace {

template <bool F32>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (F32) {
        const float4 a = *reinterpret_cast<const float4*>((const float*)p + i);
        const float4 b = *reinterpret_cast<const float4*>((const float*)p + i + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>((const uint16_t*)p + i);
        v[0] = bf16_lo(a.x), v[1] = bf16_hi(a.x), v[2] = bf16_lo(a.y), v[3] = bf16_hi(a.y);
        v[4] = bf16_lo(a.z), v[5] = bf16_hi(a.z), v[6] = bf16_lo(a.w), v[7] = bf16_hi(a.w);
    }
}

}  // namespace

// out[t] = bf16(sum_j weights[t, j] * rows[slots[t, j]]), binary32 products and sums in
// slot order, one rounding.  A thread takes 8 columns of a token, four slots' loads in
// flight at a time; a slot outside [0, rows) adds nothing.  Bound by reading the rows.
template <bool F32>
__global__ __launch_bounds__(256) void combine_experts_kernel(CombineArgs p) {
    const int64_t vecs = p.cols / 8, total = p.tokens * vecs;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t token = i / vecs, col = (i - token * vecs) * 8;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 < p.top_k; j0 += 4) {
        float v[4][8], w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int j = j0 + c;
            const int slot = j < p.top_k ? p.slots[token * p.top_k + j] : -1;
            const bool in = slot >= 0 && slot < p.rows;
            w[c] = in ? p.weights[token * p.top_k + j] : 0.0f;
            if (in) load8<F32>(p.y, slot * p.ldy + col, v[c]);
            else
                for (int x = 0; x < 8; ++x) v[c][x] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int x = 0; x < 8; ++x) sum[x] = __builtin_fmaf(w[c], v[c][x], sum[x]);
    }
    *reinterpret_cast<uint4*>(p.out + token * p.ldo + col) =
        make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]), pack_bf16x2(sum[4], sum[5]),
                   pack_bf16x2(sum[6], sum[7]));
}

hipError_t launch_combine_experts(const CombineArgs& a, bool f32, hipStream_t st) {
    const dim3 grid((unsigned)((a.tokens * (a.cols / 8) + 255) / 256));
    if (f32) hipLaunchKernelGGL((combine_experts_kernel<true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((combine_experts_kernel<false>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace h3q
