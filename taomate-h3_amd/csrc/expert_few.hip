// The routed-expert FFN for a few tokens (up to 64 pairs) in two kernels, gfx950.
//
// What bounds it: a handful of tokens reads each hit expert's 3 f d bytes of weights once
// and computes almost nothing, so time is the weight stream (50 MB for 8 experts of f =
// 1024, d = 2048: 9 us at the HBM's rate) plus launches and dependent round trips, and the
// usual chain (plan, quantize, product, quantize, product, sum) is mostly the latter.  Here:
//
//   few_gate_up   a workgroup per (expert, 16 columns of h).  Each wave finds the expert
//                 and its pairs from the ids with ballots (one id a lane, no plan kernel),
//                 asks for its first weights, and then the workgroup quantizes the tokens it
//                 needs into LDS under those loads.  h goes to memory as bf16, by pair.
//   few_down      a workgroup per 16 columns of the output, over all hit experts: rows of h
//                 quantized into LDS (each workgroup for itself: 16 KB of h against 128 KB of
//                 weights, say), the (expert, k-step) pairs laid end to end and split evenly
//                 over the waves, so that 2 experts or 60 fill them alike; partial sums
//                 meet in LDS, and the weighted sum over a token's experts is taken there
//                 in slot order.  No atomics, no third kernel for the sum.
//
// Measured (int8, one token, 8 of 64 experts, f = 1024, d = 2048, weights out of HBM): 13 to 17
// us in all over runs, 9.6 + 8.8 by themselves (medians), of which about 9 are the weights; the
// chain of five launches takes 32.
//
// With many or long rows the quantizing inside every workgroup costs more than a launch of
// the row quantizer; then that runs first and the kernels read codes (FUSED false).
#include "grouped_gemm.hpp"
#include "row_quant.hpp"

#pragma clang fp contract(off)

namespace h3q {

namespace {

constexpr int kRowPad = 16;  // LDS rows of codes: 128-byte steps + 16, so 16 rows' chunks hit distinct banks

__device__ __host__ inline int lds_pitch(int64_t cols) { return (int)((cols + 127) / 128 * 128) + kRowPad; }

// Codes of a bf16 row [cols] (cols % 8 == 0) into LDS, zeros up to the next multiple of 128,
// by the THREADS of one wave or of the workgroup (thread t takes vectors t, t + THREADS, ...);
// returns the scale.  The first four vectors a thread stay in registers between the maximum
// and the codes, the rest of a long row is read again.  max_of: the maximum over the threads.
template <int FMT, int ROUND, int THREADS, class F>
__device__ __forceinline__ float quantize_row(const uint16_t* row, int cols, H3Q_LDS uint8_t* dst, int t, F max_of) {
    constexpr int NV = 4;
    const uint4* src = reinterpret_cast<const uint4*>(row);
    const int nvec = cols >> 3, padded = (cols + 127) / 128 * 16;
    uint4 kept[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = t + i * THREADS;
        kept[i] = v < nvec ? src[v] : make_uint4(0, 0, 0, 0);
    }
    uint32_t m = 0;
    auto up = [&](const uint4& w) __attribute__((always_inline)) {
        m = pk_abs_max(pk_abs_max(pk_abs_max(pk_abs_max(m, w.x), w.y), w.z), w.w);
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) up(kept[i]);
    for (int v = t + NV * THREADS; v < nvec; v += THREADS) up(src[v]);
    RowQuant<FMT, ROUND> q;
    q.init(max_of(wave_max(amax_from_packed(m))));
    auto put = [&](int v, const uint4& w) __attribute__((always_inline)) {
        if (v < padded) *(H3Q_LDS v2u*)(dst + 8 * v) = v < nvec ? v2u{q.pack4(w.x, w.y), q.pack4(w.z, w.w)} : v2u{0u, 0u};
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) put(t + i * THREADS, kept[i]);
    for (int v = t + NV * THREADS; v < padded; v += THREADS) put(v, v < nvec ? src[v] : make_uint4(0, 0, 0, 0));
    return q.s;
}

// The pairs of a call, one a lane (at most 64): expert relative to the first, or -1.
__device__ __forceinline__ int pair_expert(const ExpertFfnArgs& p, int pairs, int lane) {
    const int id = lane < pairs ? p.ids[lane] : -1;
    const uint32_t r = (uint32_t)id - (uint32_t)p.first;
    return id >= p.first && r < (uint32_t)p.experts ? (int)r : -1;
}

// Calls fn(tile, expert, members, skip) for every tile of the call: experts in the order in
// which their pairs first appear, 16 pairs a tile (members: the expert's pairs, skip: those
// of its earlier tiles); stops when fn returns false.  Uniform over the wave.  Returns the
// number of tiles seen.
template <class F>
__device__ __forceinline__ int for_tiles(int expert, F fn) {
    uint64_t left = __ballot(expert >= 0);
    int tile = 0;
    while (left) {
        const int e = __builtin_amdgcn_readlane(expert, __builtin_ctzll(left));
        const uint64_t members = __ballot(expert == e);
        left &= ~members;
        for (int skip = 0; skip < __popcll(members); skip += 16)
            if (!fn(tile++, e, members, skip)) return tile;
    }
    return tile;
}

}  // namespace

// h[pair, c] = bf16(silu(gate) * up) for 16 columns and one tile of pairs.
template <int OP, bool TB, bool FUSED>
__global__ __launch_bounds__(256) void few_gate_up_kernel(ExpertFfnArgs p, FewBuffers w, int slices) {
    using Mfma = GroupedMfma<OP, true>;
    using acc_t = typename Mfma::acc_t;
    constexpr int FMT = OP == kOpInt8 ? kFmtInt8 : kFmtE4M3, ROUND = OP == kOpInt8 ? kRoundRcpMul : kRoundDiv;
    constexpr int WAVES = 4, SPW = 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_dyn[];  // FUSED: codes of the tokens
    __shared__ __attribute__((aligned(16))) acc_t red[WAVES * 2 * 64];
    __shared__ float lds_scale[64], lds_amax[WAVES];
    __shared__ int lds_pair[WAVES][16];
    H3Q_LDS uint8_t* const codes = (H3Q_LDS uint8_t*)lds_dyn;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int slice = blockIdx.x % slices, want = blockIdx.x / slices;
    const int pairs = (int)(p.tokens * p.top_k);
    int expert = 0, skip = 0;
    uint64_t members = 0;
    bool found = false;
    for_tiles(pair_expert(p, pairs, lane), [&](int tile, int e, uint64_t m, int s) {
        if (tile != want) return true;
        expert = e;
        members = m;
        skip = s;
        found = true;
        return false;
    });
    if (!found) return;
    const int count = __popcll(members) - skip < 16 ? __popcll(members) - skip : 16;
    const int rank = __popcll(members & ((uint64_t(1) << lane) - 1)) - skip;
    if ((members >> lane & 1) && rank >= 0 && rank < 16) lds_pair[wave][rank] = lane;

    const int64_t steps = (p.d + 127) / 128;
    const int64_t w_bytes = 2 * p.f * p.d;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc((const uint8_t*)p.w13 + expert * w_bytes, (uint32_t)w_bytes);
    uint32_t woff[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t row = j * p.f + 16 * slice;
        if constexpr (TB) woff[j] = (uint32_t)(row / 16 * steps * 2048 + 16 * lane);
        else woff[j] = (uint32_t)((row + r16) * p.d + 32 * kq);
    }
    auto load_w = [&](int c, v8i (&wf)[SPW][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const int64_t st = (int64_t)(c * SPW + i) * WAVES + wave;
            const int left = (int)(p.d - st * 128) - 32 * kq;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t lo, hi;
                if constexpr (TB) {
                    lo = st < steps ? woff[j] + (uint32_t)(st * 2048) : kOob;
                    hi = st < steps ? lo + 1024 : kOob;
                } else {
                    lo = left > 0 ? woff[j] + (uint32_t)(st * 128) : kOob;
                    hi = left > 16 ? woff[j] + (uint32_t)(st * 128) + 16 : kOob;
                }
                constexpr int policy = TB ? 2 : 0;
                wf[i][j] = join(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, lo, 0, policy)),
                                __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, hi, 0, policy)));
            }
        }
    };
    v8i wa[SPW][2], wb[SPW][2];
    load_w(0, wa);
    load_w(1, wb);
    __builtin_amdgcn_sched_barrier(0);
    // Column scales of the epilogue, in flight with the weights.
    const v4f sg = *reinterpret_cast<const v4f*>(p.s13 + expert * 2 * p.f + 16 * slice + 4 * kq);
    const v4f su = *reinterpret_cast<const v4f*>(p.s13 + expert * 2 * p.f + p.f + 16 * slice + 4 * kq);

    const int pitch = lds_pitch(p.d);
    if constexpr (FUSED) {
        // The tokens of the tile's pairs, a wave per token (a token with several pairs once).
        uint64_t tokens = 0, m = members;
        for (int i = 0; i < skip; ++i) m &= m - 1;
        for (int i = 0; i < count; ++i, m &= m - 1) tokens |= uint64_t(1) << (__builtin_ctzll(m) / p.top_k);
        if (__popcll(tokens) == 1) {  // one token: the whole workgroup quantizes it
            const int t = __builtin_ctzll(tokens);
            const float s = quantize_row<FMT, ROUND, WAVES * 64>(
                p.x + t * p.ldx, (int)p.d, codes + t * pitch, threadIdx.x, [&](float wave_amax) {
                    if (lane == 0) lds_amax[wave] = wave_amax;
                    __syncthreads();
                    float m = lds_amax[0];
#pragma unroll
                    for (int i = 1; i < WAVES; ++i) m = mag_max(m, lds_amax[i]);
                    return m;
                });
            if (threadIdx.x == 0) lds_scale[t] = s;
        } else {  // a wave per token
            int n = 0;
            while (tokens) {
                const int t = __builtin_ctzll(tokens);
                tokens &= tokens - 1;
                if (n++ % WAVES != wave) continue;
                const float s = quantize_row<FMT, ROUND, 64>(p.x + t * p.ldx, (int)p.d, codes + t * pitch, lane,
                                                             [](float m) { return m; });
                if (lane == 0) lds_scale[t] = s;
            }
        }
        __syncthreads();
    }
    const int pair = lds_pair[wave][r16 < count ? r16 : 0];
    const int token = pair / p.top_k;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(w.xq, (uint32_t)(p.tokens * p.d));  // FUSED: not read
    auto frag = [&](int64_t st) __attribute__((always_inline)) -> v8i {
        if constexpr (FUSED) {
            if (st >= steps) return v8i{};
            const H3Q_LDS uint8_t* q = codes + token * pitch + st * 128 + 32 * kq;
            return join(*(const H3Q_LDS v4i*)q, *(const H3Q_LDS v4i*)(q + 16));
        } else {
            const int left = r16 < count ? (int)(p.d - st * 128) - 32 * kq : 0;
            const uint32_t o = (uint32_t)(token * p.d + st * 128 + 32 * kq);
            return join(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, left > 0 ? o : kOob, 0, 0)),
                        __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, left > 16 ? o + 16 : kOob, 0, 0)));
        }
    };
    acc_t acc[2] = {acc_t{}, acc_t{}};
    auto mfma_chunk = [&](int c, const v8i (&wf)[SPW][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const typename Mfma::frag_t x = Mfma::frag(frag((int64_t)(c * SPW + i) * WAVES + wave));
            acc[0] = Mfma::run(Mfma::frag(wf[i][0]), x, acc[0]);
            acc[1] = Mfma::run(Mfma::frag(wf[i][1]), x, acc[1]);
        }
    };
    const int iters = (int)((steps + WAVES - 1) / WAVES);
    const int nc = (iters + SPW - 1) / SPW;
    for (int c = 0; c < nc; c += 2) {  // (an odd last chunk's partner was read as zeros)
        mfma_chunk(c, wa);
        if (c + 2 < nc) load_w(c + 2, wa);
        __builtin_amdgcn_sched_barrier(0);
        mfma_chunk(c + 1, wb);
        if (c + 2 < nc) load_w(c + 3, wb);
        __builtin_amdgcn_sched_barrier(0);
    }
    red[(wave * 2 + 0) * 64 + lane] = acc[0];
    red[(wave * 2 + 1) * 64 + lane] = acc[1];
    __syncthreads();
    if (wave != 0 || r16 >= count) return;
    acc_t g = red[lane], u = red[64 + lane];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        g += red[i * 128 + lane];
        u += red[i * 128 + 64 + lane];
    }
    const float sx = FUSED ? lds_scale[token] : w.xs[token];
    float y[4];
#pragma unroll
    for (int v = 0; v < 4; ++v)
        y[v] = swiglu_f32(__fmul_rn(sx, __fmul_rn(sg[v], (float)g[v])), __fmul_rn(sx, __fmul_rn(su[v], (float)u[v])));
    *reinterpret_cast<v2u*>(w.h + (int64_t)pair * p.f + 16 * slice + 4 * kq) =
        v2u{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
}

// COLS columns of the output, over all tiles.  8 columns (half a weight block: the other
// half's lanes load nothing) where 16 would leave CUs without a workgroup.
template <int OP, bool TB, bool FUSED, int COLS>
__global__ __launch_bounds__(512) void few_down_kernel(ExpertFfnArgs p, FewBuffers w, int max_tiles) {
    using Mfma = GroupedMfma<OP>;
    using acc_t = typename Mfma::acc_t;
    constexpr int FMT = OP == kOpInt8 ? kFmtInt8 : kFmtE4M3, ROUND = OP == kOpInt8 ? kRoundRcpMul : kRoundDiv;
    constexpr int WAVES = 8, SPW = FUSED ? 4 : 2;  // as many registers as two workgroups a CU leave
    // Segments (1 KB each: one tile's sum by one wave, tile t of wave w at t + w: both only
    // grow along the stream), then (FUSED) the codes of h.
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_dyn[];
    __shared__ float lds_scale[64], lds_weight[64], lds_y[64 * COLS];
    __shared__ int lds_pair[64 * 16];   // pair of [tile][row], -1 where there is none
    __shared__ int lds_at[64];          // tile * 16 + row of each pair, -1 without an expert
    __shared__ int lds_w0[64], lds_w1[64];  // waves that hold a tile's first and last steps
    H3Q_LDS float* const seg = (H3Q_LDS float*)lds_dyn;
    H3Q_LDS uint8_t* const codes = (H3Q_LDS uint8_t*)lds_dyn + (max_tiles + WAVES) * 1024;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * COLS;
    const int pairs = (int)(p.tokens * p.top_k);
    const int mine = pair_expert(p, pairs, lane);
    int at = -1, tile_expert = 0;  // of pair `lane`; of tile `lane`
    const int tiles = for_tiles(mine, [&](int tile, int e, uint64_t m, int skip) {
        const int rank = __popcll(m & ((uint64_t(1) << lane) - 1)) - skip;
        if ((m >> lane & 1) && rank >= 0 && rank < 16) at = tile * 16 + rank;
        if (lane == tile) tile_expert = e;
        return true;
    });
    const int steps = (int)((p.f + 127) / 128);
    const int total = tiles * steps;
    const int s0 = __builtin_amdgcn_readfirstlane(total * wave / WAVES);
    const int s1 = __builtin_amdgcn_readfirstlane(total * (wave + 1) / WAVES);

    // Weight steps s0 .. s1 - 1 of the stream, SPW at a time.
    const int64_t w_bytes = p.d * p.f;
    const int64_t block = TB ? (int64_t)(n0 / 16) * steps * 2048 : (int64_t)n0 * p.f;
    const uint32_t block_bytes = TB ? (uint32_t)steps * 2048u : (uint32_t)(COLS * p.f);
    const bool has_row = r16 < COLS;
    const uint32_t lane_off = TB ? (uint32_t)(16 * ((n0 & 15) + r16 + 16 * kq)) : (uint32_t)(r16 * p.f + 32 * kq);
    int lt = s0 / steps, lk = s0 - lt * steps;  // tile and k-step of the next load
    auto load_w = [&](int c, v8i (&wf)[SPW]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const bool in = s0 + c * SPW + i < s1;
            const int64_t e = __builtin_amdgcn_readlane(tile_expert, in ? lt : 0);
            const __amdgpu_buffer_rsrc_t rw = make_rsrc((const uint8_t*)p.w2 + e * w_bytes + block, block_bytes);
            uint32_t lo, hi;
            if constexpr (TB) {
                lo = in && has_row ? (uint32_t)(lk * 2048) + lane_off : kOob;
                hi = in && has_row ? lo + 1024 : kOob;
            } else {
                const int left = (int)(p.f - lk * 128) - 32 * kq;
                const uint32_t o = (uint32_t)(lk * 128) + lane_off;
                lo = in && has_row && left > 0 ? o : kOob;
                hi = in && has_row && left > 16 ? o + 16 : kOob;
            }
            constexpr int policy = TB ? 2 : 0;
            wf[i] = join(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, lo, 0, policy)),
                         __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, hi, 0, policy)));
            if (++lk == steps) {
                lk = 0;
                ++lt;
            }
        }
    };
    v8i wa[SPW], wb[SPW];
    load_w(0, wa);
    load_w(1, wb);
    __builtin_amdgcn_sched_barrier(0);

    // What the epilogue needs, in flight with the weights: the channel scale of the outputs
    // (pair, column) this thread finishes.
    float s2[2] = {0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int item = threadIdx.x + 512 * q, pair = item / COLS;
        const int e = __shfl(mine, pair & 63, 64);
        if (pair < pairs && e >= 0) s2[q] = p.s2[e * p.d + n0 + item % COLS];
    }
    if (wave == 0) {
        lds_at[lane] = at;
        lds_weight[lane] = lane < pairs && mine >= 0 ? p.weights[lane] : 0.0f;
        for (int i = 0; i < tiles; i += 4) lds_pair[i * 16 + lane] = -1;
        if (at >= 0) lds_pair[at] = lane;
        if (!FUSED) lds_scale[lane] = lane < pairs ? w.hs[lane] : 0.0f;
    }
    const int pitch = lds_pitch(p.f);
    if constexpr (FUSED) {
        for (int pair = wave; pair < pairs; pair += WAVES) {
            if (__builtin_amdgcn_readlane(mine, pair) < 0) continue;
            const float s = quantize_row<FMT, ROUND, 64>(w.h + (int64_t)pair * p.f, (int)p.f, codes + pair * pitch, lane,
                                                         [](float m) { return m; });
            if (lane == 0) lds_scale[pair] = s;
        }
    }
    __syncthreads();

    // Not FUSED: the codes' fragments are asked for with the weights of the same steps.
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(w.hq, (uint32_t)((int64_t)pairs * p.f));
    int xt = s0 / steps, xk = s0 - xt * steps, xrow = 0;
    v8i xa[FUSED ? 1 : SPW], xb[FUSED ? 1 : SPW];
    auto load_x = [&](int c, v8i (&xf)[FUSED ? 1 : SPW]) __attribute__((always_inline)) {
        if constexpr (!FUSED) {
#pragma unroll
            for (int i = 0; i < SPW; ++i) {
                const bool in = s0 + c * SPW + i < s1;
                if (in && (xk == 0 || c + i == 0)) xrow = lds_pair[xt * 16 + r16];
                const int left = xrow < 0 ? 0 : (int)(p.f - xk * 128) - 32 * kq;
                const uint32_t o = (uint32_t)(xrow * p.f + xk * 128 + 32 * kq);
                xf[i] = join(
                    __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, in && left > 0 ? o : kOob, 0, 0)),
                    __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, in && left > 16 ? o + 16 : kOob, 0, 0)));
                if (++xk == steps) {
                    xk = 0;
                    ++xt;
                }
            }
        }
    };
    load_x(0, xa);
    load_x(1, xb);
    __builtin_amdgcn_sched_barrier(0);
    int ct = s0 / steps, ck = s0 - ct * steps;  // tile and k-step of the next product
    int row = 0;                                // pair of this lane's row in tile ct
    acc_t acc = acc_t{};
    auto enter = [&]() __attribute__((always_inline)) {  // before a step of tile ct
        row = lds_pair[ct * 16 + r16];
        row = row < 0 ? 0 : row;  // a row without a pair: any codes, its sums are not used
        acc = acc_t{};
        if (ck == 0 && lane == 0) lds_w0[ct] = wave;
    };
    auto leave = [&]() __attribute__((always_inline)) {
        *(H3Q_LDS acc_t*)(seg + ((ct + wave) * 64 + lane) * 4) = acc;
        if (ck == steps - 1 && lane == 0) lds_w1[ct] = wave;
    };
    auto mfma_chunk = [&](int c, const v8i (&wf)[SPW], const v8i (&xf)[FUSED ? 1 : SPW]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const int s = s0 + c * SPW + i;
            if (s >= s1) break;
            v8i x;
            if constexpr (FUSED) {
                const H3Q_LDS uint8_t* q = codes + row * pitch + ck * 128 + 32 * kq;
                x = join(*(const H3Q_LDS v4i*)q, *(const H3Q_LDS v4i*)(q + 16));
            } else {
                x = xf[i];
            }
            acc = Mfma::run(wf[i], x, acc);
            if (ck == steps - 1 || s == s1 - 1) leave();
            if (++ck == steps) {
                ck = 0;
                ++ct;
                if (s + 1 < s1) enter();
            }
        }
    };
    if (s0 < s1) enter();
    const int nc = (s1 - s0 + SPW - 1) / SPW;
    for (int c = 0; c < nc; c += 2) {
        mfma_chunk(c, wa, xa);
        if (c + 2 < nc) {
            load_w(c + 2, wa);
            load_x(c + 2, xa);
        }
        __builtin_amdgcn_sched_barrier(0);
        mfma_chunk(c + 1, wb, xb);
        if (c + 2 < nc) {
            load_w(c + 3, wb);
            load_x(c + 3, xb);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();

    // y of each pair, its waves' sums in wave order; then the tokens' weighted sums.
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int item = threadIdx.x + 512 * q, pair = item / COLS, col = item % COLS;
        if (pair >= pairs) continue;
        float y = 0.0f;
        const int place = lds_at[pair];
        if (place >= 0) {
            const int tile = place / 16, r = place & 15, last = lds_w1[tile];
            acc_t sum = acc_t{};  // one element of it is used
            for (int v = lds_w0[tile]; v <= last; ++v)
                if (total * v / WAVES < total * (v + 1) / WAVES)  // with few steps some waves have none
                    sum[0] += ((const H3Q_LDS decltype(sum[0] + 0)*)seg)[((tile + v) * 64 + r + 16 * (col >> 2)) * 4 + (col & 3)];
            y = __fmul_rn(lds_scale[pair], __fmul_rn(s2[q], (float)sum[0]));
        }
        lds_y[item] = y;
    }
    __syncthreads();
    for (int item = threadIdx.x; item < (int)p.tokens * COLS; item += 512) {
        const int token = item / COLS, col = item % COLS;
        float out = 0.0f;
#pragma unroll 8
        for (int j = 0; j < p.top_k; ++j) {  // a pair without an expert: 0 * 0
            const int pair = token * p.top_k + j;
            out = __builtin_fmaf(lds_weight[pair], lds_y[pair * COLS + col], out);
        }
        p.out[token * p.ldo + n0 + col] = (uint16_t)f32_to_bf16_bits(out);
    }
}

namespace {

constexpr int kFewPairs = 64;           // one id a lane
constexpr int kFewLdsCodes = 40 * 1024;  // codes that a workgroup quantizes into its LDS

int few_tiles(const ExpertFfnArgs& a) {  // at most
    const int pairs = (int)(a.tokens * a.top_k);
    const int most = a.experts + pairs / 16;
    return most < pairs ? most : pairs;
}

// Quantizing inside the gate-up kernel pays while its workgroups are all resident at once; in
// further rounds each would pay again what one launch of the row quantizer costs.
bool fused_up(const ExpertFfnArgs& a) {
    return a.tokens * lds_pitch(a.d) <= kFewLdsCodes && a.f / 16 * few_tiles(a) <= 1024;
}
bool fused_down(const ExpertFfnArgs& a) { return a.tokens * a.top_k * lds_pitch(a.f) <= kFewLdsCodes; }

template <int OP, bool TB>
void launch_up(const ExpertFfnArgs& a, const FewBuffers& w, hipStream_t st) {
    const int slices = (int)(a.f / 16);
    const dim3 grid((unsigned)(slices * few_tiles(a)));
    if (fused_up(a))
        hipLaunchKernelGGL((few_gate_up_kernel<OP, TB, true>), grid, dim3(256), (unsigned)(a.tokens * lds_pitch(a.d)), st,
                           a, w, slices);
    else
        hipLaunchKernelGGL((few_gate_up_kernel<OP, TB, false>), grid, dim3(256), 0, st, a, w, slices);
}

template <int OP, bool TB, int COLS>
void launch_down_cols(const ExpertFfnArgs& a, const FewBuffers& w, hipStream_t st) {
    const int tiles = few_tiles(a);
    const unsigned segments = (unsigned)(tiles + 8) * 1024;
    const dim3 grid((unsigned)(a.d / COLS));
    if (fused_down(a))
        hipLaunchKernelGGL((few_down_kernel<OP, TB, true, COLS>), grid, dim3(512),
                           segments + (unsigned)(a.tokens * a.top_k * lds_pitch(a.f)), st, a, w, tiles);
    else
        hipLaunchKernelGGL((few_down_kernel<OP, TB, false, COLS>), grid, dim3(512), segments, st, a, w, tiles);
}

template <int OP, bool TB>
void launch_down(const ExpertFfnArgs& a, const FewBuffers& w, hipStream_t st) {
    if (a.d / 16 < 256) launch_down_cols<OP, TB, 8>(a, w, st);
    else launch_down_cols<OP, TB, 16>(a, w, st);
}

}  // namespace

bool expert_few_supported(const ExpertFfnArgs& a) {
    return a.tokens * a.top_k <= kFewPairs && a.f / 16 * few_tiles(a) < (int64_t(1) << 24);  // grid * 256 < 2^32
}

hipError_t launch_expert_few(const ExpertFfnArgs& a, const FewBuffers& w, hipStream_t st) {
    const int fmt = a.kind == kOpInt8 ? kFmtInt8 : kFmtE4M3, rounding = a.kind == kOpInt8 ? kRoundRcpMul : kRoundDiv;
    hipError_t e = hipSuccess;
    if (!fused_up(a)) e = launch_quant_rows(a.x, a.ldx, a.tokens, a.d, fmt, rounding, w.xq, a.d, w.xs, st);
    if (e != hipSuccess) return e;
    if (a.kind == kOpInt8) a.w13_tiled ? launch_up<kOpInt8, true>(a, w, st) : launch_up<kOpInt8, false>(a, w, st);
    else a.w13_tiled ? launch_up<kOpE4M3, true>(a, w, st) : launch_up<kOpE4M3, false>(a, w, st);
    e = hipGetLastError();
    const int64_t pairs = a.tokens * a.top_k;
    if (e == hipSuccess && !fused_down(a)) e = launch_quant_rows(w.h, a.f, pairs, a.f, fmt, rounding, w.hq, a.f, w.hs, st);
    if (e != hipSuccess) return e;
    if (a.kind == kOpInt8) a.w2_tiled ? launch_down<kOpInt8, true>(a, w, st) : launch_down<kOpInt8, false>(a, w, st);
    else a.w2_tiled ? launch_down<kOpE4M3, true>(a, w, st) : launch_down<kOpE4M3, false>(a, w, st);
    return hipGetLastError();
}

}  // namespace h3q
