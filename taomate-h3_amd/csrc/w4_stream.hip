// Product with 4-bit weights for few rows (m <= 32), gfx950: bound by the weights' bytes, n k / 2 from HBM once.
//
// A workgroup owns 16 output columns and all rows (MT tiles of 16); its waves split k, wave w taking the
// 128-column blocks w, w + WAVES, ...  A block's codes, scales and zero points go from memory into registers, DEPTH
// blocks ahead (a few KiB a wave, so that a whole call's weights are under way at once); its x rows come out of
// the L2 one block ahead, rows past m as out-of-range offsets that move no bytes.  The waves' sums meet in LDS
// and are added in wave order.
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

template <bool F16, int MT, int WAVES, int DEPTH>
__global__ __launch_bounds__(WAVES * 64) void w4_stream_kernel(W4Args p) {
    __shared__ __attribute__((aligned(16))) v4f red[WAVES * MT * 64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int64_t blk = blockIdx.x;
    const int steps = (int)((p.k + 127) / 128), quads = (p.groups + 3) / 4;
    const __amdgpu_buffer_rsrc_t rw = w4_rsrc(p.codes + blk * steps * 1024, (int64_t)steps * 1024);
    const __amdgpu_buffer_rsrc_t rs = w4_rsrc(p.scales + blk * quads * 64, (int64_t)quads * 128);
    const __amdgpu_buffer_rsrc_t rz = w4_rsrc(p.zeros + (p.zeros ? blk * quads * 64 : 0), p.zeros ? quads * 64 : 0);
    const __amdgpu_buffer_rsrc_t rx = w4_rsrc(p.x, ((p.m - 1) * p.ldx + p.k) * 2);

    uint32_t xoff[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        xoff[t] = 16 * t + r16 < p.m ? (uint32_t)((16 * t + r16) * p.ldx * 2 + 16 * kq) : kW4Oob;

    v4u codes[DEPTH], x[2][MT][4];
    v2u scales[DEPTH];
    uint32_t zeros[DEPTH];
    auto load = [&](int i, int b) __attribute__((always_inline)) {  // past the end: zeros
        const int q = w4_quad(p, b);
        codes[i] = __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)(b * 1024 + 16 * lane), 0, 2);  // read once
        scales[i] = __builtin_amdgcn_raw_buffer_load_b64(rs, (uint32_t)(q * 128 + 8 * r16), 0, 0);
        zeros[i] = 0x08080808u;
        if (p.zeros) zeros[i] = __builtin_amdgcn_raw_buffer_load_b32(rz, (uint32_t)(q * 64 + 4 * r16), 0, 0);
    };
    auto load_x = [&](int i, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const bool inside = xoff[t] != kW4Oob && 128 * b + 32 * s + 8 * kq < p.k;
                x[i][t][s] = __builtin_amdgcn_raw_buffer_load_b128(
                    rx, inside ? xoff[t] + (uint32_t)(256 * b + 64 * s) : kW4Oob, 0, 0);
            }
    };
    v4f acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = v4f{};
    auto multiply = [&](int i, int j, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            float scale, shift;
            w4_group(scales[i], zeros[i], w4_element(p, b, s), p.scales_f16, scale, shift);
            const v4u w = w4_weights<F16>(codes[i][s], scale, shift);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = mfma16<F16>(w, x[j][t][s], acc[t]);
        }
    };

    const int count = steps > wave ? (steps - wave + WAVES - 1) / WAVES : 0;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(d, wave + d * WAVES);
    load_x(0, wave);
    for (int i = 0; i < count; i += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (i + d >= count) break;
            const int b = wave + (i + d) * WAVES;
            load_x((d + 1) & 1, b + WAVES);
            __builtin_amdgcn_sched_barrier(0);
            multiply(d, d & 1, b);
            load(d, b + DEPTH * WAVES);
        }
    }

#pragma unroll
    for (int t = 0; t < MT; ++t) red[(wave * MT + t) * 64 + lane] = acc[t];
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (t % WAVES != wave) continue;
        v4f s = red[t * 64 + lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += red[(w * MT + t) * 64 + lane];
        w4_store<F16>(p, 16 * t + r16, 16 * blk + 4 * kq, s);
    }
}

template <bool F16, int MT>
hipError_t launch_cfg(const W4Args& a, hipStream_t st) {
    hipLaunchKernelGGL((w4_stream_kernel<F16, MT, 8, 4>), dim3((unsigned)((a.n + 15) / 16)), dim3(512), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_w4_stream(const W4Args& a, hipStream_t st) {
    if (a.m <= 16) return a.f16 ? launch_cfg<true, 1>(a, st) : launch_cfg<false, 1>(a, st);
    return a.f16 ? launch_cfg<true, 2>(a, st) : launch_cfg<false, 2>(a, st);
}

}  // namespace h3q
