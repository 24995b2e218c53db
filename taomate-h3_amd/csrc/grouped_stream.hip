// Scaled product of rows grouped by expert, weight streaming, gfx950.
//
//   y[i, n] = s_a[r] * (s_w[e, n] * sum_k A[r, k] * W[e, n, k]),   i in expert e's rows,
//   r = order[i] / top_k, or i without an order
//   out = round(y), or with SwiGLU (W's rows [gate | up]) round(silu(y_gate) * y_up)
//
// With few rows to an expert the product is bound by reading every hit expert's weights
// once from HBM, as the dense weight-streaming kernel (gemm_skinny.hip) is, and this one
// is built alike: weights go from memory straight into the registers of the one wave that
// uses them.  A workgroup owns up to 16 rows of one expert and two 16-row weight blocks
// (SwiGLU: a gate block and the up block of the same columns, so the two meet in the
// epilogue); its four waves take every fourth 128-byte k-step, in chunks of two steps,
// the next chunk's loads in flight during the current chunk's products.  The activation
// fragments come through the L2 (every column slice reads the same few rows).  The waves'
// partial sums meet in LDS.
//
// k need not be a multiple of 128 with row-major weights: bytes past it read as zero.
//
// Measured (int8, tiled weights, three sets in turn): 32 experts of 2816 x 2048 with SwiGLU,
// 4 rows each on average, 28.5 us (6.5 TB/s); 8 of 14336 x 5376, 89.5 us (6.9 TB/s).
#include "grouped_gemm.hpp"

namespace h3q {

namespace {

constexpr int kStreamWaves = 4;

}  // namespace

template <int OP, bool TB, int OUT>
__global__ __launch_bounds__(kStreamWaves * 64) void grouped_stream_kernel(GroupedArgs p, int slices) {
    constexpr bool SWIGLU = OUT == kOutSwiglu || OUT == kOutWide, F32 = OUT == kOutF32;
    using Mfma = GroupedMfma<OP, OUT == kOutWide>;
    using acc_t = typename Mfma::acc_t;
    constexpr int WAVES = kStreamWaves, SPW = 2, BM = 16;
    constexpr int ITEMS = SWIGLU ? 1 : 2;  // 16 x 16 output blocks of the workgroup, a wave each
    __shared__ __attribute__((aligned(16))) acc_t red[WAVES * 2 * 64];

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
    uint32_t woff[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = block_row(j);
        if constexpr (TB) woff[j] = row < p.n ? (uint32_t)(row / 16 * steps * 2048 + 16 * lane) : kOob;
        else woff[j] = row < p.n ? (uint32_t)((int64_t)(row + r16) * p.k + 32 * kq) : kOob;
    }
    // Activation rows: gathered from all of them, or the tile's own.
    const bool gather = p.order != nullptr;
    const __amdgpu_buffer_rsrc_t rx =
        gather ? make_rsrc(p.a, (uint32_t)(p.a_rows * p.lda))
               : make_rsrc((const uint8_t*)p.a + tile.row0 * p.lda, (uint32_t)((int64_t)rows * p.lda));
    int64_t r = -1;  // row of a behind this lane's row of the tile
    if (r16 < rows) {
        r = tile.row0 + r16;
        if (gather) {
            const int pair = p.order[r];
            r = pair >= 0 && pair / p.top_k < p.a_rows ? pair / p.top_k : -1;
        }
    }
    const uint32_t xoff = r >= 0 ? (uint32_t)((gather ? r : r16) * p.lda + 32 * kq) : kOob;

    // Chunk c of this wave: its steps c SPW .. c SPW + SPW - 1 (k bytes from 128 st).
    auto load_w = [&](int c, v8i (&wf)[SPW][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const int64_t st = (int64_t)(c * SPW + i) * WAVES + wave;
            const int left = (int)(p.k - st * 128) - 32 * kq;  // bytes of the lane's 32 that exist
#pragma unroll
            for (int j = 0; j < 2; ++j) {
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
        }
    };
    auto load_x = [&](int c, v8i (&xf)[SPW]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const int64_t st = (int64_t)(c * SPW + i) * WAVES + wave;
            const int left = (int)(p.k - st * 128) - 32 * kq;
            const uint32_t lo = xoff != kOob && left > 0 ? xoff + (uint32_t)(st * 128) : kOob;
            const uint32_t hi = xoff != kOob && left > 16 ? xoff + (uint32_t)(st * 128) + 16 : kOob;
            xf[i] = join(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, lo, 0, 0)),
                         __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rx, hi, 0, 0)));
        }
    };
    acc_t acc[2] = {acc_t{}, acc_t{}};
    auto mfma_chunk = [&](const v8i (&wf)[SPW][2], const v8i (&xf)[SPW]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const typename Mfma::frag_t x = Mfma::frag(xf[i]);
            acc[0] = Mfma::run(Mfma::frag(wf[i][0]), x, acc[0]);
            acc[1] = Mfma::run(Mfma::frag(wf[i][1]), x, acc[1]);
        }
    };
    const int iters = (int)((steps + WAVES - 1) / WAVES);
    const int nc = (iters + SPW - 1) / SPW;
    v8i wa[SPW][2], xa[SPW], wb[SPW][2], xb[SPW];
    auto load_chunk = [&](int c, v8i (&wf)[SPW][2], v8i (&xf)[SPW]) __attribute__((always_inline)) {
        load_w(c, wf);
        load_x(c, xf);
    };
    load_chunk(0, wa, xa);
    // Scales of the epilogue, in flight with the weights: this lane's row, and four columns of
    // the wave's output block (SwiGLU: of the gate and the up block).
    const float sa = r >= 0 ? p.a_scale[r] : 0.0f;
    v4f sw[SWIGLU ? 2 : 1];
#pragma unroll
    for (int g = 0; g < (SWIGLU ? 2 : 1); ++g) {
        const int row = wave < ITEMS ? block_row(SWIGLU ? g : wave) : p.n;
        sw[g] = row < p.n ? *reinterpret_cast<const v4f*>(p.b_scale + (int64_t)expert * p.n + row + 4 * kq)
                          : v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
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

    red[(wave * 2 + 0) * 64 + lane] = acc[0];
    red[(wave * 2 + 1) * 64 + lane] = acc[1];
    __syncthreads();
    if (wave >= ITEMS) return;

    // Sum over the waves in wave order, scales, output: lane holds columns 4 kq .. + 3 of row r16.
    auto total = [&](int j) __attribute__((always_inline)) -> acc_t {
        acc_t s = red[j * 64 + lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += red[(w * 2 + j) * 64 + lane];
        return s;
    };
    const int row = block_row(SWIGLU ? 0 : wave);
    const acc_t s0 = total(SWIGLU ? 0 : wave);
    float y[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) y[v] = __fmul_rn(sa, __fmul_rn(sw[0][v], (float)s0[v]));
    if constexpr (SWIGLU) {
        const acc_t s1 = total(1);
#pragma unroll
        for (int v = 0; v < 4; ++v)
            y[v] = swiglu_f32(y[v], __fmul_rn(sa, __fmul_rn(sw[SWIGLU ? 1 : 0][v], (float)s1[v])));
    }
    if (r >= 0 && row < p.n) {  // rows past the tile, or without a row of a, keep what out held
        const int64_t at = (tile.row0 + r16) * p.ldo + row + 4 * kq;
        if constexpr (F32) *reinterpret_cast<v4f*>((float*)p.out + at) = v4f{y[0], y[1], y[2], y[3]};
        else *reinterpret_cast<v2u*>((uint16_t*)p.out + at) = v2u{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    }
}

namespace {

int stream_slices(const GroupedArgs& a) { return a.swiglu ? a.n / 32 : (a.n + 31) / 32; }

template <int OP, bool TB>
hipError_t launch_stream_tb(const GroupedArgs& a, hipStream_t st) {
    const int slices = stream_slices(a);
    const dim3 grid((unsigned)grouped_stream_grid(a)), block(kStreamWaves * 64);
    if (OP == kOpE4M3 && a.swiglu && a.wide)
        hipLaunchKernelGGL((grouped_stream_kernel<kOpE4M3, TB, kOutWide>), grid, block, 0, st, a, slices);
    else if (a.swiglu)
        hipLaunchKernelGGL((grouped_stream_kernel<OP, TB, kOutSwiglu>), grid, block, 0, st, a, slices);
    else if (a.f32)
        hipLaunchKernelGGL((grouped_stream_kernel<OP, TB, kOutF32>), grid, block, 0, st, a, slices);
    else
        hipLaunchKernelGGL((grouped_stream_kernel<OP, TB, kOutBF16>), grid, block, 0, st, a, slices);
    return hipGetLastError();
}

}  // namespace

int64_t grouped_stream_grid(const GroupedArgs& a) { return (a.experts + a.rows / 16) * stream_slices(a); }

hipError_t launch_grouped_stream(int kind, const GroupedArgs& a, hipStream_t st) {
    if (kind == kOpInt8) return a.b_tiled ? launch_stream_tb<kOpInt8, true>(a, st) : launch_stream_tb<kOpInt8, false>(a, st);
    return a.b_tiled ? launch_stream_tb<kOpE4M3, true>(a, st) : launch_stream_tb<kOpE4M3, false>(a, st);
}

}  // namespace h3q
