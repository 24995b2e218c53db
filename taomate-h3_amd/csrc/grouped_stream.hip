// Scaled product of rows grouped by expert, weight streaming, gfx950.
//
//   y[i, n] = s_a[r] * (s_w[e, n] * sum_k A[r, k] * W[e, n, k]),   i in expert e's rows,
//   r = order[i] / top_k, or i without an order
//   out = round(y), or with SwiGLU (W's rows [gate | up]) round(silu(y_gate) * y_up)
//
// With few rows to an expert the product is bound by reading every hit expert's weights
// once from HBM, as the dense weight-streaming kernel (gemm_skinny.hip) is, and this one
// is built alike: weights go from memory straight into the registers of the one wave that
// uses them.  A workgroup owns up to 16 MT rows of one expert and NBLK 16-row weight
// blocks (SwiGLU: as many gate blocks as up blocks of the same columns, so gate and up
// meet in the epilogue); its four waves take every fourth 128-byte k-step, in chunks of
// SPW steps, the next chunk's loads in flight during the current chunk's products.  The
// activation fragments come through the L2 (every column slice reads the same few rows).
// The waves' partial sums meet in LDS.
//
// k need not be a multiple of 128 with row-major weights: bytes past it read as zero.
#include "grouped_gemm.hpp"

namespace h3q {

namespace {

constexpr int kStreamWaves = 4;

}  // namespace

template <int OP, int MT, int SPW, bool TB, bool SWIGLU, bool F32>
__global__ __launch_bounds__(kStreamWaves * 64) void grouped_stream_kernel(GroupedArgs p, int slices) {
    using Mfma = GroupedMfma<OP, SWIGLU>;  // what SwiGLU gives is quantized again: wide products
    using acc_t = typename Mfma::acc_t;
    constexpr int WAVES = kStreamWaves, NBLK = 2, BM = 16 * MT;
    constexpr int ITEMS = SWIGLU ? MT : NBLK * MT;  // 16 x 16 output blocks of the workgroup
    constexpr int PER_WAVE = (ITEMS + WAVES - 1) / WAVES;
    __shared__ __attribute__((aligned(16))) acc_t red[WAVES * NBLK * MT * 64];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int slice = blockIdx.x % slices;
    const GroupTile tile = group_tile(p.offsets, p.experts, p.rows, BM, blockIdx.x / slices);
    if (tile.rows <= 0) return;
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert);
    const int rows = __builtin_amdgcn_readfirstlane(tile.rows);
    const int half = p.n / 2;  // SwiGLU: first up row

    // First weight row of block j, or n for none.
    auto block_row = [&](int j) __attribute__((always_inline)) -> int {
        if constexpr (SWIGLU) return j * half + 16 * slice;
        const int r = 32 * slice + 16 * j;
        return r < p.n ? r : p.n;
    };
    const int64_t steps = (p.k + 127) / 128;
    const int64_t w_bytes = (int64_t)p.n * p.k;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc((const uint8_t*)p.b + expert * w_bytes, (uint32_t)w_bytes);
    uint32_t woff[NBLK];
#pragma unroll
    for (int j = 0; j < NBLK; ++j) {
        const int row = block_row(j);
        if constexpr (TB) woff[j] = row < p.n ? (uint32_t)(row / 16 * steps * 2048 + 16 * lane) : kOob;
        else woff[j] = row < p.n ? (uint32_t)((int64_t)(row + r16) * p.k + 32 * kq) : kOob;
    }
    // Activation rows: gathered from all of them, or the tile's own.
    const bool gather = p.order != nullptr;
    const __amdgpu_buffer_rsrc_t rx =
        gather ? make_rsrc(p.a, (uint32_t)(p.a_rows * p.lda))
               : make_rsrc((const uint8_t*)p.a + tile.row0 * p.lda, (uint32_t)((int64_t)rows * p.lda));
    uint32_t xoff[MT];
    float sa[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = 16 * t + r16;
        int64_t r = -1;
        if (m < rows) {
            r = tile.row0 + m;
            if (gather) {
                r = p.order[r] / p.top_k;
                if (r >= p.a_rows) r = -1;  // also the -1 of a row without a pair
            }
        }
        sa[t] = r >= 0 ? p.a_scale[r] : 0.0f;
        xoff[t] = r >= 0 ? (uint32_t)((gather ? r : m) * p.lda + 32 * kq) : kOob;
    }
    // Column scales of this wave's output blocks: item i covers row block i % MT of
    // weight block i / MT (SwiGLU: of the gate and the up block).
    v4f sw[PER_WAVE][SWIGLU ? 2 : 1];
#pragma unroll
    for (int q = 0; q < PER_WAVE; ++q) {
        const int i = q * WAVES + wave;
#pragma unroll
        for (int g = 0; g < (SWIGLU ? 2 : 1); ++g) {
            const int row = block_row(SWIGLU ? g : i / MT);
            sw[q][g] = i < ITEMS && row < p.n
                           ? *reinterpret_cast<const v4f*>(p.b_scale + (int64_t)expert * p.n + row + 4 * kq)
                           : v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    acc_t acc[NBLK][MT];
#pragma unroll
    for (int j = 0; j < NBLK; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = acc_t{};

    // Chunk c of this wave: its steps c SPW .. c SPW + SPW - 1 (k bytes from 128 st).
    auto load_chunk = [&](int c, v8i (&wf)[SPW][NBLK], v8i (&xf)[SPW][MT]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const int64_t st = (int64_t)(c * SPW + i) * WAVES + wave;
            const int left = (int)(p.k - st * 128) - 32 * kq;  // bytes of the lane's 32 that exist
#pragma unroll
            for (int j = 0; j < NBLK; ++j) {
                uint32_t lo, hi;
                if constexpr (TB) {
                    lo = st < steps && woff[j] != kOob ? woff[j] + (uint32_t)(st * 2048) : kOob;
                    hi = lo == kOob ? kOob : lo + 1024;
                } else {
                    lo = left > 0 && woff[j] != kOob ? woff[j] + (uint32_t)(st * 128) : kOob;
                    hi = left > 16 && woff[j] != kOob ? woff[j] + (uint32_t)(st * 128) + 16 : kOob;
                }
                constexpr int policy = TB ? 2 : 0;  // tiled weights pass once: non-temporal (see gemm_skinny.hip)
                wf[i][j] = join(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, lo, 0, policy)),
                                __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, hi, 0, policy)));
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const bool in = xoff[t] != kOob;
                const uint32_t lo = in && left > 0 ? xoff[t] + (uint32_t)(st * 128) : kOob;
                const uint32_t hi = in && left > 16 ? xoff[t] + (uint32_t)(st * 128) + 16 : kOob;
                xf[i][t] = join(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, lo, 0, 0)),
                                __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, hi, 0, 0)));
            }
        }
    };
    auto mfma_chunk = [&](const v8i (&wf)[SPW][NBLK], const v8i (&xf)[SPW][MT]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            typename Mfma::frag_t w[NBLK];
#pragma unroll
            for (int j = 0; j < NBLK; ++j) w[j] = Mfma::frag(wf[i][j]);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const typename Mfma::frag_t x = Mfma::frag(xf[i][t]);
#pragma unroll
                for (int j = 0; j < NBLK; ++j) acc[j][t] = Mfma::run(w[j], x, acc[j][t]);
            }
        }
    };
    const int iters = (int)((steps + WAVES - 1) / WAVES);
    const int nc = (iters + SPW - 1) / SPW;
    v8i wa[SPW][NBLK], xa[SPW][MT], wb[SPW][NBLK], xb[SPW][MT];
    load_chunk(0, wa, xa);
    int c = 0;
    for (; c + 2 < nc; c += 2) {
        load_chunk(c + 1, wb, xb);
        __builtin_amdgcn_sched_barrier(0);
        mfma_chunk(wa, xa);
        load_chunk(c + 2, wa, xa);
        __builtin_amdgcn_sched_barrier(0);
        mfma_chunk(wb, xb);
    }
    if (c + 1 < nc) {
        load_chunk(c + 1, wb, xb);
        __builtin_amdgcn_sched_barrier(0);
        mfma_chunk(wa, xa);
        mfma_chunk(wb, xb);
    } else {
        mfma_chunk(wa, xa);
    }

#pragma unroll
    for (int j = 0; j < NBLK; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[((wave * NBLK + j) * MT + t) * 64 + lane] = acc[j][t];
    __syncthreads();

    // Sum over the waves in wave order, scales, output: lane holds columns 4 kq .. + 3 of
    // row 16 t + r16.
    auto total = [&](int j, int t) __attribute__((always_inline)) -> acc_t {
        acc_t s = red[(j * MT + t) * 64 + lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += red[((w * NBLK + j) * MT + t) * 64 + lane];
        return s;
    };
#pragma unroll
    for (int q = 0; q < PER_WAVE; ++q) {
        const int i = q * WAVES + wave;
        if (i >= ITEMS) break;
        const int t = i % MT;
        const int row = block_row(SWIGLU ? 0 : i / MT);
        float scale = sa[0];
#pragma unroll
        for (int x = 1; x < MT; ++x) scale = t == x ? sa[x] : scale;
        float y[4];
        const acc_t s0 = total(SWIGLU ? 0 : i / MT, t);
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = __fmul_rn(scale, __fmul_rn(sw[q][0][v], (float)s0[v]));
        if constexpr (SWIGLU) {
            const acc_t s1 = total(1, t);
#pragma unroll
            for (int v = 0; v < 4; ++v)
                y[v] = swiglu_f32(y[v], __fmul_rn(scale, __fmul_rn(sw[q][SWIGLU ? 1 : 0][v], (float)s1[v])));
        }
        const int m = 16 * t + r16;
        if (m < rows && row < p.n) {
            const int64_t at = (tile.row0 + m) * p.ldo + row + 4 * kq;
            if constexpr (F32) *reinterpret_cast<v4f*>((float*)p.out + at) = v4f{y[0], y[1], y[2], y[3]};
            else
                *reinterpret_cast<v2u*>((uint16_t*)p.out + at) =
                    v2u{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        }
    }
}

namespace {

// Row blocks of a tile, from the mean rows of an expert.
int stream_row_blocks(const GroupedArgs& a) { return a.rows / a.experts <= 16 ? 1 : 4; }

bool tile_kernel(const GroupedArgs& a) { return a.rows / a.experts > 64 && grouped_tile_supported(a); }

int stream_slices(const GroupedArgs& a) { return a.swiglu ? a.n / 32 : (a.n + 31) / 32; }

int64_t stream_grid(const GroupedArgs& a) {
    return (a.experts + a.rows / (16 * stream_row_blocks(a))) * stream_slices(a);
}

template <int OP, int MT, int SPW, bool TB>
hipError_t launch_stream_tb(const GroupedArgs& a, hipStream_t st) {
    const int slices = stream_slices(a);
    const dim3 grid((unsigned)stream_grid(a)), block(kStreamWaves * 64);
    if (a.swiglu)
        hipLaunchKernelGGL((grouped_stream_kernel<OP, MT, SPW, TB, true, false>), grid, block, 0, st, a, slices);
    else if (a.f32)
        hipLaunchKernelGGL((grouped_stream_kernel<OP, MT, SPW, TB, false, true>), grid, block, 0, st, a, slices);
    else
        hipLaunchKernelGGL((grouped_stream_kernel<OP, MT, SPW, TB, false, false>), grid, block, 0, st, a, slices);
    return hipGetLastError();
}

template <int OP>
hipError_t launch_stream_op(const GroupedArgs& a, hipStream_t st) {
    if (stream_row_blocks(a) == 1)
        return a.b_tiled ? launch_stream_tb<OP, 1, 2, true>(a, st) : launch_stream_tb<OP, 1, 2, false>(a, st);
    return a.b_tiled ? launch_stream_tb<OP, 4, 1, true>(a, st) : launch_stream_tb<OP, 4, 1, false>(a, st);
}

}  // namespace

// A grid of n workgroups of 256 threads takes n * 256 < 2^32.
bool grouped_mm_fits(const GroupedArgs& a) { return tile_kernel(a) || stream_grid(a) < (int64_t(1) << 24); }

hipError_t launch_grouped_mm(int kind, const GroupedArgs& a, hipStream_t st) {
    if (tile_kernel(a)) return launch_grouped_tile(kind, a, st);
    return kind == kOpInt8 ? launch_stream_op<kOpInt8>(a, st) : launch_stream_op<kOpE4M3>(a, st);
}

}  // namespace h3q
