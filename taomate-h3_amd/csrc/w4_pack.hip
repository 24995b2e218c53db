// 4-bit weights as the products read them, gfx950: the quantizer of weight rows and the layout of w4.hpp.  Both run
// once, when a model is loaded.
#include "w4.hpp"

namespace h3q {

namespace {

// One thread a word of the layout: eight codes of a row.
__global__ __launch_bounds__(256) void w4_pack_kernel(W4PackArgs p, int64_t words, int steps) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const int s = (int)(i & 3), lane = (int)(i >> 2) & 63;
        const int64_t block = i >> 8, b = block % steps;
        const int64_t row = block / steps * 16 + (lane & 15), k = b * 128 + 32 * s + 8 * (lane >> 4);
        uint32_t w = 0;
        if (row < p.n && k < p.k) {
            const uint8_t* const c = p.codes + row * p.ldc + k / 2;
#pragma unroll
            for (int e = 0; e < 8; ++e) w |= (uint32_t)(c[e / 2] >> 4 * (e & 1) & 15) << (8 * (e & 3) + (e & 4));
        }
        ((uint32_t*)p.codes_out)[i] = w;
    }
}

__global__ __launch_bounds__(256) void w4_pack_scales_kernel(W4PackArgs p, int64_t count) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t quads = (p.groups + 3) / 4, panel = i >> 6;
        const int64_t g = panel % quads * 4 + (i & 3), row = panel / quads * 16 + (i >> 2 & 15);
        const bool in = row < p.n && g < p.groups;
        p.scales_out[i] = in ? p.scales[row * p.lds + g] : 0;
        if (p.zeros) p.zeros_out[i] = in ? p.zeros[row * p.ldz + g] & 15 : 0;
    }
}

__device__ __forceinline__ float weight_at(const W4QuantArgs& p, int64_t i) {
    if (p.dtype == kInF32) return ((const float*)p.w)[i];
    return out_lo(((const uint16_t*)p.w)[i], p.dtype == kInF16);
}

// Sixteen lanes a group.  s is rounded to its 16-bit type before the codes are made with it.  A NaN among a group's
// weights makes s a NaN (an infinity makes it one that is not finite by itself), so that no product hides it.
__global__ __launch_bounds__(256) void w4_quant_kernel(W4QuantArgs p, int groups) {
    const int l = threadIdx.x & 15;
    const int64_t teams = p.n * groups;  // of 16 lanes, which stay together
    for (int64_t team = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); team < teams; team += (int64_t)gridDim.x * 16) {
        const int64_t row = team / groups;
        const int g = (int)(team - row * groups);
        const int64_t k0 = (int64_t)g * p.group, k1 = k0 + p.group < p.k ? k0 + p.group : p.k;
        float low = 0.0f, high = 0.0f;
        int nan = 0;
        for (int64_t k = k0 + l; k < k1; k += 16) {
            const float v = weight_at(p, row * p.ldw + k);
            nan |= v != v;
            low = v < low ? v : low;
            high = v > high ? v : high;
        }
        for (int off = 8; off >= 1; off >>= 1) {
            const float a = __shfl_xor(low, off, 16), b = __shfl_xor(high, off, 16);
            low = a < low ? a : low;
            high = b > high ? b : high;
            nan |= __shfl_xor(nan, off, 16);
        }
        const float reach = nan ? __builtin_nanf("") : p.zeros ? (high - low) / 15.0f : (high > -low ? high : -low) / 7.0f;
        const bool f16 = p.dtype == kInF16;
        const uint16_t bits = (uint16_t)pack_out2(reach, 0.0f, f16);
        const float s = out_lo(bits, f16);
        float z = 8.0f;
        if (p.zeros) z = s > 0.0f ? fminf(fmaxf(__builtin_rintf(-low / s), 0.0f), 15.0f) : 0.0f;
        for (int64_t k = k0 + 2 * l; k < k1; k += 32) {
            uint32_t byte = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float q = s > 0.0f ? __builtin_rintf(weight_at(p, row * p.ldw + k + e) / s) : 0.0f;
                byte |= (uint32_t)fminf(fmaxf(q + z, 0.0f), 15.0f) << (4 * e);
            }
            p.codes[row * (p.k / 2) + k / 2] = (uint8_t)byte;
        }
        if (l == 0) {
            p.scales[team] = bits;
            if (p.zeros) p.zeros[team] = (uint8_t)z;
        }
    }
}

// At most 65536 blocks, which loop: a grid of 2^32 threads or more is cut off without an error.
unsigned blocks_for(int64_t threads) {
    const int64_t b = (threads + 255) / 256;
    return (unsigned)(b < 65536 ? b : 65536);
}

}  // namespace

hipError_t launch_w4_pack(const W4PackArgs& a, hipStream_t st) {
    const int64_t blocks = (a.n + 15) / 16, steps = (a.k + 127) / 128;
    const int64_t words = blocks * steps * 256, count = blocks * ((a.groups + 3) / 4) * 64;
    hipLaunchKernelGGL(w4_pack_kernel, dim3(blocks_for(words)), dim3(256), 0, st, a, words, (int)steps);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(w4_pack_scales_kernel, dim3(blocks_for(count)), dim3(256), 0, st, a, count);
    return hipGetLastError();
}

hipError_t launch_w4_quant(const W4QuantArgs& a, hipStream_t st) {
    const int groups = (int)((a.k + a.group - 1) / a.group);
    hipLaunchKernelGGL(w4_quant_kernel, dim3(blocks_for(a.n * groups * 16)), dim3(256), 0, st, a, groups);
    return hipGetLastError();
}

}  // namespace h3q
