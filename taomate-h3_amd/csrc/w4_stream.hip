// Product with 4-bit weights for few rows (m <= 32), gfx950: bound by the weights' bytes, n k / 2 from HBM once.
//
// A workgroup owns 16 NB output columns and all rows (MT tiles of 16); its waves split k, wave w taking the
// 128-column blocks w, w + WAVES, ...  A block's codes go from memory into the operand registers with no LDS
// between; its x rows (all of x is in the L2) the same way, rows past m as out-of-range offsets that move
// no bytes.  Block i + 1 is asked for before block i is used.  sum(x) of a group comes from one more matrix
// instruction with ones for weights: it lands in the lanes that need it.  The waves' sums meet in LDS and are
// added in wave order.
#include "w4.hpp"

namespace h3q {

namespace {

template <bool F16, bool ZEROS, int GPB, int MT, int NB>
struct W4Stage {
    v4u codes[NB], x[MT][4];
    v2u scales[NB][GPB];
    uint32_t zeros[NB][GPB];
};

// GPB: groups of a 128-column block (1: the group is a multiple of 128).
template <bool F16, bool ZEROS, int GPB, int MT, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void w4_stream_kernel(W4Args p) {
    __shared__ __attribute__((aligned(16))) v4f red[WAVES * NB * MT * 64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int blk0 = blockIdx.x * NB, blocks = (int)((p.n + 15) / 16);
    const int nblk = blocks - blk0 < NB ? blocks - blk0 : NB;
    const int steps = (int)((p.k + 127) / 128), groups = p.groups;
    const __amdgpu_buffer_rsrc_t rw =
        make_rsrc(p.codes + (int64_t)blk0 * steps * 1024, (uint32_t)(nblk * steps * 1024));
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.scales + (int64_t)blk0 * groups * 16, (uint32_t)(nblk * groups * 32));
    const __amdgpu_buffer_rsrc_t rz =
        make_rsrc(p.zeros + (ZEROS ? (int64_t)blk0 * groups * 16 : 0), ZEROS ? (uint32_t)(nblk * groups * 16) : 0);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x, (uint32_t)(((p.m - 1) * p.ldx + p.k) * 2));

    uint32_t xoff[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        xoff[t] = 16 * t + r16 < p.m ? (uint32_t)((16 * t + r16) * p.ldx * 2 + 16 * kq) : kW4Oob;

    using Stage = W4Stage<F16, ZEROS, GPB, MT, NB>;
    auto load = [&](Stage& s, int b) __attribute__((always_inline)) {
        const bool in = b < steps;
#pragma unroll
        for (int j = 0; j < NB; ++j)
            s.codes[j] = w4_load16(rw, in && j < nblk ? (uint32_t)((j * steps + b) * 1024 + 16 * lane) : kW4Oob, kW4Stream);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 128 * b + 32 * i + 8 * kq;
                const bool inside = xoff[t] != kW4Oob && k < p.k;
                s.x[t][i] = w4_load16(rx, inside ? xoff[t] + (uint32_t)(256 * b + 64 * i) : kW4Oob, 0);
            }
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int q = 0; q < GPB; ++q) {
                const int g = GPB == 1 ? b / p.blocks_per_group : b * GPB + q;
                const bool inside = in && j < nblk && g < groups;
                s.scales[j][q] = __builtin_amdgcn_raw_buffer_load_b64(
                    rs, inside ? (uint32_t)((j * groups + g) * 32 + 8 * kq) : kW4Oob, 0, 0);
                if constexpr (ZEROS)
                    s.zeros[j][q] = __builtin_amdgcn_raw_buffer_load_b32(
                        rz, inside ? (uint32_t)((j * groups + g) * 16 + 4 * kq) : kW4Oob, 0, 0);
                else
                    s.zeros[j][q] = 0;
            }
    };

    v4f acc[NB][MT];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = v4f{};
    constexpr uint32_t one = F16 ? 0x3C003C00u : 0x3F803F80u;
    const v4u ones = {one, one, one, one};

    auto multiply = [&](const Stage& s) __attribute__((always_inline)) {
        constexpr int SPG = 4 / GPB;  // matrix steps of a group
#pragma unroll
        for (int q = 0; q < GPB; ++q) {
            v4f sum[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                sum[t] = v4f{};
#pragma unroll
                for (int i = q * SPG; i < (q + 1) * SPG; ++i) sum[t] = w4_mfma<F16>(ones, s.x[t][i], sum[t]);
            }
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                v4f part[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) part[t] = v4f{};
#pragma unroll
                for (int i = q * SPG; i < (q + 1) * SPG; ++i) {
                    const v4u w = w4_unpack<F16>(s.codes[j][i]);
#pragma unroll
                    for (int t = 0; t < MT; ++t) part[t] = w4_mfma<F16>(w, s.x[t][i], part[t]);
                }
                const v4f scale = w4_scales(s.scales[j][q], p.scales_f16), off = w4_offsets<ZEROS>(s.zeros[j][q]);
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[j][t][e] =
                            __builtin_fmaf(scale[e], __builtin_fmaf(-off[e], sum[t][0], part[t][e]), acc[j][t][e]);
            }
        }
    };

    const int count = steps > wave ? (steps - wave + WAVES - 1) / WAVES : 0;
    if (count > 0) {
        Stage a, b;
        load(a, wave);
        int i = 0;
        for (; i + 2 < count; i += 2) {
            load(b, wave + (i + 1) * WAVES);
            __builtin_amdgcn_sched_barrier(0);
            multiply(a);
            load(a, wave + (i + 2) * WAVES);
            __builtin_amdgcn_sched_barrier(0);
            multiply(b);
        }
        if (i + 1 < count) {
            load(b, wave + (i + 1) * WAVES);
            __builtin_amdgcn_sched_barrier(0);
            multiply(a);
            multiply(b);
        } else {
            multiply(a);
        }
    }

#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[((wave * NB + j) * MT + t) * 64 + lane] = acc[j][t];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if ((j * MT + t) % WAVES != wave) continue;
            v4f s = red[(j * MT + t) * 64 + lane];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) s += red[((w * NB + j) * MT + t) * 64 + lane];
            w4_store<F16>(p, 16 * t + r16, 16 * (int64_t)(blk0 + j) + 4 * kq, s);
        }
}

template <bool F16, bool ZEROS, int GPB, int MT, int NB, int WAVES>
hipError_t launch_cfg(const W4Args& a, hipStream_t st) {
    const unsigned grid = (unsigned)(((a.n + 15) / 16 + NB - 1) / NB);
    hipLaunchKernelGGL((w4_stream_kernel<F16, ZEROS, GPB, MT, NB, WAVES>), dim3(grid), dim3(WAVES * 64), 0, st, a);
    return hipGetLastError();
}

template <bool F16, bool ZEROS, int GPB>
hipError_t launch_rows(const W4Args& a, hipStream_t st) {
    if (a.m <= 16) return launch_cfg<F16, ZEROS, GPB, 1, 1, 8>(a, st);
    return launch_cfg<F16, ZEROS, GPB, 2, 1, 8>(a, st);
}

template <bool F16, bool ZEROS>
hipError_t launch_groups(const W4Args& a, hipStream_t st) {
    if (a.group == 32) return launch_rows<F16, ZEROS, 4>(a, st);
    if (a.group == 64) return launch_rows<F16, ZEROS, 2>(a, st);
    return launch_rows<F16, ZEROS, 1>(a, st);
}

}  // namespace

hipError_t launch_w4_stream(const W4Args& a, hipStream_t st) {
    if (a.f16) return a.zeros ? launch_groups<true, true>(a, st) : launch_groups<true, false>(a, st);
    return a.zeros ? launch_groups<false, true>(a, st) : launch_groups<false, false>(a, st);
}

}  // namespace h3q
