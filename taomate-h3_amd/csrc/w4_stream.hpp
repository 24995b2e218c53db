// Product with 4-bit weights for few rows (m <= 16), gfx950: bound by the weights' bytes, n k / 2 from HBM once, as
// long as the instructions that fetch them are few: a CU takes about 24 cycles for a vector load whatever it brings,
// and a first version that asked for x and scales beside every KiB of codes ran at half the memory's rate.
//
// A workgroup owns 16 NB output columns and all rows; its waves split k, wave w taking the 128-column blocks w, w + WAVES,
// ...  A block's codes, scales and zero points go from memory into registers DEPTH
// blocks ahead.  x is the small operand: for up to 3 rows (XLDS) it is copied into LDS once (chunk by chunk
// where it is long), and the lanes of the rows behind m read row 0; above that its fragments come out of the L2, once
// for the NB column blocks of a wave.
//
// Weights stay integers here (u, exact in x's type) and the scale is applied to a group's sum in binary32:
//   y += s * (sum x u - z sum x)
// with sum(x) from one more matrix instruction, whose other operand is ones.  This takes 28 operations to unpack
// 32 codes and 8 to add a group, where rounding scaled weights takes 76: at one row of 14336 x 14336 22.3 us against
// 26.8, at 16 rows of 10752 x 5376 the same way.  x is the first operand of the matrix
// instruction, so that a lane's sums belong to one output column, whose scale it holds.
#pragma once

#include "w4.hpp"

namespace h3q {

namespace {

template <bool F16>
__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0,
                                                       0);
}

// Eight codes -> the integers 0 .. 15 in x's type (an e4m3 byte times 2^9, see w4.hpp).
template <bool F16>
__device__ __forceinline__ v4u integers(uint32_t w) {
    const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
    if constexpr (F16)
        return v4u{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, true))};
    else
        return v4u{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, true))};
}

constexpr int kFewRows = 3;
// LDS for x of few rows: three workgroups of eight waves on a CU.  Rows are 64 bytes out of step with the banks.
constexpr int kFewBytes = 44 * 1024;
constexpr int few_blocks(int64_t m) { return (int)((kFewBytes / m - 64) / 256); }

// GPB: groups of a 128-column block (1: the group is a multiple of 128).
template <bool F16, bool ZEROS, int GPB, int NB, int WAVES, int DEPTH, bool XLDS>
__global__ __launch_bounds__(WAVES * 64) void w4_stream_kernel(W4Args p) {
    __shared__ __attribute__((aligned(16))) v4f red[WAVES * NB * 64];
    extern __shared__ __attribute__((aligned(16))) uint8_t x_raw[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int64_t blk0 = (int64_t)blockIdx.x * NB, blocks = (p.n + 15) / 16;
    const int nblk = blocks - blk0 < NB ? (int)(blocks - blk0) : NB;
    const int steps = (int)((p.k + 127) / 128), quads = (p.groups + 3) / 4;
    const __amdgpu_buffer_rsrc_t rw = w4_rsrc(p.codes + blk0 * steps * 1024, (int64_t)nblk * steps * 1024);
    const __amdgpu_buffer_rsrc_t rs = w4_rsrc(p.scales + blk0 * quads * 64, (int64_t)nblk * quads * 128);
    const __amdgpu_buffer_rsrc_t rz =
        w4_rsrc(p.zeros + (ZEROS ? blk0 * quads * 64 : 0), ZEROS ? (int64_t)nblk * quads * 64 : 0);
    const __amdgpu_buffer_rsrc_t rx = w4_rsrc(p.x, ((p.m - 1) * p.ldx + p.k) * 2);

    const uint32_t xoff = r16 < p.m ? (uint32_t)(r16 * p.ldx * 2 + 16 * kq) : kW4Oob;

    v4u codes[DEPTH][NB], x[XLDS ? 1 : DEPTH][4];
    v2u scales[DEPTH][NB];
    uint32_t zeros[DEPTH][NB];
    auto load = [&](int i, int b) __attribute__((always_inline)) {
        const int q = w4_group(p, b, 0) >> 2;
#pragma unroll
        for (int j = 0; j < NB; ++j) {  // codes: read once, kept out of the caches
            codes[i][j] = __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)((j * steps + b) * 1024 + 16 * lane), 0, 2);
            scales[i][j] = __builtin_amdgcn_raw_buffer_load_b64(rs, (uint32_t)((j * quads + q) * 128 + 8 * r16), 0, 0);
            zeros[i][j] = 0;
            if constexpr (ZEROS)
                zeros[i][j] = __builtin_amdgcn_raw_buffer_load_b32(rz, (uint32_t)((j * quads + q) * 64 + 4 * r16), 0, 0);
        }
        if constexpr (!XLDS) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const bool inside = xoff != kW4Oob && 128 * b + 32 * s + 8 * kq < p.k;
                x[i][s] = __builtin_amdgcn_raw_buffer_load_b128(rx, inside ? xoff + (uint32_t)(256 * b + 64 * s) : kW4Oob,
                                                                0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // blocks in order: a wait for one waits for none behind it
    };
    v4f acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = v4f{};
    constexpr uint32_t one = F16 ? 0x3C003C00u : 0x3F803F80u;
    const v4u ones = {one, one, one, one};
    auto multiply = [&](int i, int b, const v4u (&xf)[4]) __attribute__((always_inline)) {
        constexpr int SPG = 4 / GPB;  // matrix steps of a group
#pragma unroll
        for (int q = 0; q < GPB; ++q) {
            const int g = w4_group(p, b, q * SPG);
            v4f sum = {};
#pragma unroll
            for (int s = q * SPG; s < (q + 1) * SPG; ++s) sum = mfma16<F16>(xf[s], ones, sum);
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                v4f part = {};
#pragma unroll
                for (int s = q * SPG; s < (q + 1) * SPG; ++s) part = mfma16<F16>(xf[s], integers<F16>(codes[i][j][s]), part);
                float scale, shift;
                w4_scale<ZEROS>(scales[i][j], zeros[i][j], g, p.scales_f16, scale, shift);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[j][e] = __builtin_fmaf(scale, __builtin_fmaf(shift, sum[e], part[e]), acc[j][e]);
            }
        }
    };

    // The chunks of k that LDS holds (one, but for few long rows), and in each the blocks of this wave.
    const int chunk = XLDS ? few_blocks(p.m) : steps;
    for (int c0 = 0; c0 < steps; c0 += chunk) {
        const int c1 = c0 + chunk < steps ? c0 + chunk : steps;
        const int first = c0 + wave, count = c1 > first ? (c1 - first + WAVES - 1) / WAVES : 0;
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (d < count) load(d, first + d * WAVES);
        H3Q_LDS uint8_t* const xs = (H3Q_LDS uint8_t*)x_raw;
        const int pitch = (c1 - c0) * 256 + 64;
        if constexpr (XLDS) {
            if (c0 > 0) __syncthreads();
            const int vectors = (c1 - c0) * 16;
            for (int64_t r = 0; r < p.m; ++r)
                for (int v = threadIdx.x; v < vectors; v += WAVES * 64) {
                    const int64_t k = 128 * (int64_t)c0 + 8 * v;
                    v4u w = {};
                    if (k < p.k) w = *reinterpret_cast<const v4u*>(p.x + r * p.ldx + k);
                    *(H3Q_LDS v4u*)(xs + r * pitch + 16 * v) = w;
                }
            __syncthreads();
        }
        const H3Q_LDS uint8_t* const xr = xs + (r16 < p.m ? r16 : 0) * pitch + 16 * kq;
        for (int i = 0; i < count; i += DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                if (i + d >= count) break;
                const int b = first + (i + d) * WAVES;
                if constexpr (XLDS) {
                    v4u xf[4];
#pragma unroll
                    for (int s = 0; s < 4; ++s) xf[s] = *(const H3Q_LDS v4u*)(xr + (b - c0) * 256 + 64 * s);
                    multiply(d, b, xf);
                } else {
                    multiply(d, b, x[d]);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (i + d + DEPTH < count) load(d, b + DEPTH * WAVES);
            }
        }
    }

#pragma unroll
    for (int j = 0; j < NB; ++j) red[(wave * NB + j) * 64 + lane] = acc[j];
    __syncthreads();
    if (wave >= NB) return;
    v4f sum = red[wave * 64 + lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += red[(w * NB + wave) * 64 + lane];
    const int64_t n = 16 * (blk0 + wave) + r16;
    if (n >= p.n) return;
    const float bias = p.bias ? out_lo(p.bias[n], F16) : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (4 * kq + e < p.m) p.out[(4 * kq + e) * p.ldo + n] = (uint16_t)pack_out2(sum[e] + bias, 0.0f, F16);
}

template <bool F16, bool ZEROS, int GPB, int NB, int WAVES, int DEPTH, bool XLDS>
hipError_t launch_cfg(const W4Args& a, hipStream_t st) {
    const unsigned grid = (unsigned)(((a.n + 15) / 16 + NB - 1) / NB);
    size_t lds = 0;
    if (XLDS) {
        const int64_t steps = (a.k + 127) / 128, held = few_blocks(a.m);
        lds = (size_t)(a.m * ((steps < held ? steps : held) * 256 + 64));
    }
    hipLaunchKernelGGL((w4_stream_kernel<F16, ZEROS, GPB, NB, WAVES, DEPTH, XLDS>), dim3(grid), dim3(WAVES * 64), lds,
                       st, a);
    return hipGetLastError();
}

// The column blocks of a workgroup: as few as leave at most one workgroup to a CU, because every one of them brings
// all of x (measured at 13 rows of 7003 x 4096, 438 blocks: 7.9 us with two, 10.4 with one, 10.9 with four; at 16
// rows of 10752 x 5376, 672 blocks: 11.1 us with four, 15.3 with two).  With x in LDS there is less to
// bring: one block, two from three workgroups a CU on (14336 x 14336: 21.1 us against 23.6), and sixteen waves where there
// are fewer workgroups than CUs (1024 x 14336: 8.0 us against 9.7).  x goes there for up to 3 rows: 3 rows of 5376 x
// 7168 8.6 us against 8.9, of 10752 x 5376 at groups of 32 11.1 against 11.6; 4 rows 9.9 against 9.1, and 11.3 against 11.6.
template <bool F16, bool ZEROS, int GPB>
hipError_t launch_w4_stream_rows(const W4Args& a, hipStream_t st) {
    const int64_t blocks = (a.n + 15) / 16;
    if (a.m <= kFewRows) {
        if (blocks <= 256) return launch_cfg<F16, ZEROS, GPB, 1, 16, 2, true>(a, st);
        if (blocks < 768) return launch_cfg<F16, ZEROS, GPB, 1, 8, 2, true>(a, st);
        return launch_cfg<F16, ZEROS, GPB, 2, 8, 2, true>(a, st);
    }
    if (blocks <= 256) return launch_cfg<F16, ZEROS, GPB, 1, 8, 2, false>(a, st);
    if (blocks <= 512) return launch_cfg<F16, ZEROS, GPB, 2, 8, 1, false>(a, st);
    return launch_cfg<F16, ZEROS, GPB, 4, 8, 1, false>(a, st);
}

template <bool F16, bool ZEROS>
hipError_t launch_w4_stream_groups(const W4Args& a, hipStream_t st) {
    if (a.group == 32) return launch_w4_stream_rows<F16, ZEROS, 4>(a, st);
    if (a.group == 64) return launch_w4_stream_rows<F16, ZEROS, 2>(a, st);
    return launch_w4_stream_rows<F16, ZEROS, 1>(a, st);
}

}  // namespace

}  // namespace h3q
