// Routing of a mixture-of-experts layer, gfx950: the top-k of the router's logits, the
// plan that sorts the (token, slot) pairs by expert, and the weighted sum that brings
// the experts' rows back to their tokens.
#include <type_traits>

#include "h3q_common.hpp"
#include "h3q_kernels.hpp"
#include "row_quant.hpp"

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

// One step of a wave's reduction over its rows of 16: lane 15 (31) of the row before.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t row_bcast(uint32_t old, uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 0xF, false);
}

// Reductions over the LPT lanes (16 or 64) of a token; every lane gets the result.  neutral:
// what leaves the other operand of f as it is.
template <int LPT, class F>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, uint32_t neutral, F f) {
    v = f(v, row_ror<8>(v));
    v = f(v, row_ror<4>(v));
    v = f(v, row_ror<2>(v));
    v = f(v, row_ror<1>(v));
    if constexpr (LPT == 64) {
        v = f(v, row_bcast<0x142, 0xA>(neutral, v));
        v = f(v, row_bcast<0x143, 0xC>(neutral, v));
        v = (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
    }
    return v;
}
template <int LPT>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    return group_reduce<LPT>(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int LPT>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
    return group_reduce<LPT>(v, 0xFFFFFFFFu, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
template <int LPT>
__device__ __forceinline__ float group_sum(float v) {
    return __uint_as_float(group_reduce<LPT>(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

// exp(x) for x <= 0 or a logit: the hardware exp2 of x / ln 2, within (|x| + 2) 2^-23 of exp(x).
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 0x1.715476p+0f); }

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
// sigmoid 1 / (1 + exp(-l)), divided by the taken ones' sum when renormalized.  Below -18,
// 1 + exp(l) is 1 in binary32 and the score is exp(l); where the largest logit is below it,
// renormalized scores are taken as exp(l - max), whose common factor exp(max) falls out of the
// shares (the scores themselves underflow from -88 on, and their sum would be 0).
// A slot without an expert (fewer than k logits above -inf) gets -1 and weight 0.
//
// What bounds it: instructions.  The logits are read once, into registers; the k rounds cost
// about 5 NV + 20 instructions each.  Four tokens to a wave rather than one cut the
// cross-lane steps per token by four and stay within a row of 16 lanes (register permutes):
// 32768 tokens of 128 experts, top 4, take 9.8 us (16.8 MB of logits: 3 us at the HBM's rate).
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
            if (key[i] != 0u) whole += key[i] == top ? 1.0f : fast_exp(key_logit(key[i]) - best);
        whole = group_sum<LPT>(whole);
    }
    const bool logistic = p.scoring == kScoreSigmoid && !(p.renormalize && best < -18.0f);
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
            weight = logistic ? 1.0f / (1.0f + fast_exp(-l)) : m == top ? 1.0f : fast_exp(l - best);
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

// Lanes of a token.  A wave per token also for few tokens: a quarter of the work per wave while there
// are SIMDs for all of them (4093 tokens of 256 experts: 7.2 -> 6.5 us; 32768 of 128: 9.8 -> 16.4).
int route_lanes(const RouteArgs& a) { return a.experts > 256 || a.top_k > 16 || a.tokens <= 4096 ? 64 : 16; }

template <int DT>
hipError_t launch_route_dt(const RouteArgs& a, hipStream_t st) {
    const int lpt = route_lanes(a);
    const dim3 grid((unsigned)((a.tokens + 256 / lpt - 1) / (256 / lpt)));
    const int nv = (int)((a.experts + lpt - 1) / lpt);
#define H3Q_ROUTE(LPT, NV) hipLaunchKernelGGL((route_topk_kernel<DT, LPT, NV>), grid, dim3(256), 0, st, a)
    if (lpt == 64) {
        if (nv <= 1) H3Q_ROUTE(64, 1);
        else if (nv <= 4) H3Q_ROUTE(64, 4);
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

// A grid of n workgroups of 256 threads takes n * 256 < 2^32.
bool route_topk_fits(const RouteArgs& a) { return (a.tokens + 15) / 16 * 16 * route_lanes(a) < (int64_t(1) << 32); }

hipError_t launch_route_topk(const RouteArgs& a, int dtype, hipStream_t st) {
    if (dtype == kInF32) return launch_route_dt<kInF32>(a, st);
    if (dtype == kInBF16) return launch_route_dt<kInBF16>(a, st);
    return launch_route_dt<kInF16>(a, st);
}

// Plan of an expert layer: the pairs (token * top_k + slot) sorted by expert, in pair
// order within an expert (a stable counting sort).  A block of the plan is a chunk of
// consecutive pairs; its 16 waves take consecutive spans of it, 64 pairs a trip.
//
//   count   every wave counts its span's experts in its own row of an LDS table: the lanes
//           with the same expert find each other by one ballot per bit of the expert's number,
//           and the first of them adds their count (no atomics).
//   place   with the table summed over the waves below, and the counts of the blocks below
//           and of the lower experts added, the span is walked again, and every pair's row
//           is the table's entry plus its rank among its peers of the trip.
//
// Up to kPlanWholePairs pairs one workgroup does both; more take a counting launch, whose
// blocks leave their counts in the workspace, and a placing one, whose blocks each sum all
// the counts they need (blocks * experts integers, by all threads).  Deterministic.
// Pairs whose expert is not in [first, first + experts) get slot -1, and the rows past the
// last placed one order -1.
//
// What bounds it: dependent round trips and two launches; the work is log2(experts) ballots a
// trip.  131072 pairs of 128 experts: 3.7 + 7.6 us (one workgroup per expert over all pairs,
// in one launch: 46 us); 8 pairs: 3.6 us.
constexpr int kPlanWaves = 16;
constexpr int kPlanWholePairs = 2048;

namespace {

// Lanes of the wave with the same value (of `bits` bits) as this one, among `valid`.
__device__ __forceinline__ uint64_t match(int v, int bits, uint64_t valid) {
    uint64_t peers = valid;
    for (int i = 0; i < bits; ++i) {
        const bool one = v >> i & 1;
        const uint64_t b = __ballot(one);
        peers &= one ? b : ~b;
    }
    return peers;
}

}  // namespace

enum PlanPhase : int { kPlanWhole = 0, kPlanCount = 1, kPlanPlace = 2 };

// Block `block` of `blocks` of a plan.  table: LDS of kPlanWaves * experts integers,
// [wave][expert]: counts, then the next row of that expert in the wave's span.
template <int PHASE>
__device__ __forceinline__ void plan_block(const PlanArgs& p, int64_t chunk, int bits, int block, int blocks, int* table) {
    __shared__ int wave_sum[kPlanWaves];
    __shared__ int rows_all[kMaxExperts], rows_below[kMaxExperts];  // of each expert, over the blocks
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = p.experts;
    const int64_t begin = block * chunk, end = begin + chunk < p.pairs ? begin + chunk : p.pairs;
    const int64_t trips = (end - begin + 63) / 64;
    const int64_t t0 = trips * wave / kPlanWaves, t1 = trips * (wave + 1) / kPlanWaves;
    int* const mine = table + wave * n;
    for (int i = threadIdx.x; i < kPlanWaves * n; i += kPlanWaves * 64) table[i] = 0;
    if (threadIdx.x < n) rows_all[threadIdx.x] = rows_below[threadIdx.x] = 0;
    __syncthreads();

    // Expert of pair i relative to the plan's first, or n for none (ids below 0 or outside the
    // range; the difference is taken unsigned, so no id wraps into it).
    auto expert_of = [&](int64_t i) __attribute__((always_inline)) -> int {
        if (i >= end) return n;
        const int id = p.ids[i];
        const uint32_t r = (uint32_t)id - (uint32_t)p.first;
        return id >= p.first && r < (uint32_t)n ? (int)r : n;
    };
    auto walk = [&](auto place) __attribute__((always_inline)) {
        constexpr bool PLACE = decltype(place)::value;
        for (int64_t t = t0; t < t1; t += 4) {  // four trips' loads in flight
            int e4[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) e4[c] = t + c < t1 ? expert_of(begin + (t + c) * 64 + lane) : n;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (t + c >= t1) break;
                const int64_t i = begin + (t + c) * 64 + lane;
                const int e = e4[c];
                const uint64_t peers = match(e, bits, __ballot(e < n));
                const int rank = __popcll(peers & ((uint64_t(1) << lane) - 1));
                if (e < n) {
                    const int row = mine[e] + rank;
                    if constexpr (PLACE) {
                        p.order[row] = (int)i;
                        p.slots[i] = row;
                    }
                    // after every peer has read the entry: a wave's LDS operations are in order
                    if (rank == 0) mine[e] = row + __popcll(peers);
                } else if (PLACE && i < end) {
                    p.slots[i] = -1;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes read it in the next trip
            }
        }
    };
    walk(std::false_type());
    __syncthreads();

    if constexpr (PHASE == kPlanCount) {
        for (int e = threadIdx.x; e < n; e += kPlanWaves * 64) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < kPlanWaves; ++w) sum += table[w * n + e];
            p.workspace[(int64_t)block * n + e] = sum;
        }
        return;
    }
    // Rows of every expert in all blocks and in those below, each thread a share of the blocks
    // (LDS additions of integers: their order changes nothing).
    if constexpr (PHASE == kPlanPlace) {
        const int shares = kPlanWaves * 64 / n, share = threadIdx.x / n, e = threadIdx.x - share * n;
        if (share < shares) {
            int all = 0, below = 0;
#pragma unroll 8
            for (int b = share; b < blocks; b += shares) {
                const int c = p.workspace[(int64_t)b * n + e];
                all += c;
                if (b < block) below += c;
            }
            atomicAdd(&rows_all[e], all);
            atomicAdd(&rows_below[e], below);
        }
        __syncthreads();
    }
    const int e = threadIdx.x;
    int all = 0;
    if (e < n) {
        if constexpr (PHASE == kPlanPlace) {
            all = rows_all[e];
        } else {
#pragma unroll
            for (int w = 0; w < kPlanWaves; ++w) all += table[w * n + e];
        }
    }
    // Rows of the lower experts: a prefix sum over the threads.
    int sum = all;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(sum, d, 64);
        if (lane >= d) sum += o;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int lower = sum - all, total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        if (w < wave) lower += wave_sum[w];
        total += wave_sum[w];
    }
    if (e < n) {
        if (block == 0) {
            p.offsets[e] = lower;
            if (e == n - 1) p.offsets[n] = total;
        }
        int row = lower + rows_below[e];
#pragma unroll
        for (int w = 0; w < kPlanWaves; ++w) {
            const int c = table[w * n + e];
            table[w * n + e] = row;
            row += c;
        }
    }
    __syncthreads();
    walk(std::true_type());
    for (int64_t i = total + (int64_t)block * (kPlanWaves * 64) + threadIdx.x; i < p.pairs;
         i += (int64_t)blocks * (kPlanWaves * 64))
        p.order[i] = -1;
}

template <int PHASE>
__global__ __launch_bounds__(kPlanWaves * 64) void plan_experts_kernel(PlanArgs p, int64_t chunk, int bits) {
    extern __shared__ int table[];
    plan_block<PHASE>(p, chunk, bits, blockIdx.x, gridDim.x, table);
}

// The plan of up to kPlanWholePairs pairs (workgroup 0) and the codes of the tokens (a workgroup
// each of the others), in one launch: neither needs the other, and both are shorter than the
// launch that this saves.
template <int FMT, int ROUND>
__global__ __launch_bounds__(kPlanWaves * 64) void plan_quant_kernel(PlanArgs p, int bits, const uint16_t* x, int64_t ldx,
                                                                     int cols, uint8_t* codes, float* scales) {
    extern __shared__ int table[];
    if (blockIdx.x == 0) {
        plan_block<kPlanWhole>(p, kPlanWholePairs, bits, 0, 1, table);
        return;
    }
    __shared__ float wave_amax[kPlanWaves];
    const int64_t row = blockIdx.x - 1;
    const uint4* const src = reinterpret_cast<const uint4*>(x + row * ldx);
    const int nvec = cols >> 3, t = threadIdx.x;
    constexpr int THREADS = kPlanWaves * 64;
    const uint4 first = t < nvec ? src[t] : make_uint4(0, 0, 0, 0);
    uint32_t m = pk_abs_max(pk_abs_max(pk_abs_max(pk_abs_max(0, first.x), first.y), first.z), first.w);
    for (int v = t + THREADS; v < nvec; v += THREADS) {
        const uint4 w = src[v];
        m = pk_abs_max(pk_abs_max(pk_abs_max(pk_abs_max(m, w.x), w.y), w.z), w.w);
    }
    const float amax = wave_max(amax_from_packed(m));
    if ((t & 63) == 0) wave_amax[t >> 6] = amax;
    __syncthreads();
    float all = wave_amax[0];
#pragma unroll
    for (int w = 1; w < kPlanWaves; ++w) all = mag_max(all, wave_amax[w]);
    RowQuant<FMT, ROUND> q;
    q.init(all);
    v2u* const dst = reinterpret_cast<v2u*>(codes + row * cols);
    if (t < nvec) dst[t] = v2u{q.pack4(first.x, first.y), q.pack4(first.z, first.w)};
    for (int v = t + THREADS; v < nvec; v += THREADS) {
        const uint4 w = src[v];
        dst[v] = v2u{q.pack4(w.x, w.y), q.pack4(w.z, w.w)};
    }
    if (t == 0) scales[row] = q.s;
}

namespace {

int expert_bits(int experts) {
    int bits = 0;
    while ((1 << bits) < experts) ++bits;
    return bits;
}

// Pairs per block: one block for few, else at least 1024 and at most 256 blocks, so that a
// placing block's sum over them stays short.
int64_t plan_chunk(int64_t pairs) {
    if (pairs <= kPlanWholePairs) return kPlanWholePairs;
    return (pairs + 256 * 1024 - 1) / (256 * 1024) * 1024;
}

}  // namespace

int64_t plan_workspace_ints(int64_t pairs, int experts) {
    const int64_t chunk = plan_chunk(pairs);
    return pairs <= chunk ? 0 : (pairs + chunk - 1) / chunk * experts;
}

hipError_t launch_plan_experts(const PlanArgs& a, hipStream_t st) {
    const int64_t chunk = plan_chunk(a.pairs);
    const unsigned blocks = a.pairs <= chunk ? 1u : (unsigned)((a.pairs + chunk - 1) / chunk);
    const unsigned lds = (unsigned)(kPlanWaves * a.experts * sizeof(int));
    const int bits = expert_bits(a.experts);
    const dim3 threads(kPlanWaves * 64);
    if (blocks == 1) {
        hipLaunchKernelGGL((plan_experts_kernel<kPlanWhole>), dim3(1), threads, lds, st, a, chunk, bits);
    } else {
        hipLaunchKernelGGL((plan_experts_kernel<kPlanCount>), dim3(blocks), threads, lds, st, a, chunk, bits);
        hipLaunchKernelGGL((plan_experts_kernel<kPlanPlace>), dim3(blocks), threads, lds, st, a, chunk, bits);
    }
    return hipGetLastError();
}

bool plan_quant_supported(const PlanArgs& a, int64_t tokens) { return a.pairs <= kPlanWholePairs && tokens <= 512; }

hipError_t launch_plan_quant(const PlanArgs& a, int fmt, const uint16_t* x, int64_t ldx, int64_t tokens, int64_t cols,
                             uint8_t* codes, float* scales, hipStream_t st) {
    const dim3 grid((unsigned)(tokens + 1)), threads(kPlanWaves * 64);
    const unsigned lds = (unsigned)(kPlanWaves * a.experts * sizeof(int));
    const int bits = expert_bits(a.experts);
    if (fmt == kFmtInt8)
        hipLaunchKernelGGL((plan_quant_kernel<kFmtInt8, kRoundRcpMul>), grid, threads, lds, st, a, bits, x, ldx, (int)cols,
                           codes, scales);
    else
        hipLaunchKernelGGL((plan_quant_kernel<kFmtE4M3, kRoundDiv>), grid, threads, lds, st, a, bits, x, ldx, (int)cols,
                           codes, scales);
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
// slot order, one rounding.  A thread takes 8 columns of a token, eight slots' loads in
// flight at a time; a slot outside [0, rows) adds nothing.  Bound by
// reading the rows: 12288 of 2048 in binary32 (100 MB) 18.0 us, 5.6 TB/s.
template <bool F32>
__global__ __launch_bounds__(256) void combine_experts_kernel(CombineArgs p) {
    const int64_t vecs = p.cols / 8, total = p.tokens * vecs;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t token = i / vecs, col = (i - token * vecs) * 8;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 < p.top_k; j0 += 8) {
        float v[8][8], w[8];
        int slot[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int j = j0 + c;
            slot[c] = j < p.top_k ? p.slots[token * p.top_k + j] : -1;
            w[c] = j < p.top_k ? p.weights[token * p.top_k + j] : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (slot[c] >= 0 && slot[c] < p.rows) {
                load8<F32>(p.y, slot[c] * p.ldy + col, v[c]);
            } else {
                w[c] = 0.0f;
#pragma unroll
                for (int x = 0; x < 8; ++x) v[c][x] = 0.0f;
            }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
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
