// 4-bit weights with group scales: layout, unpacking and the arguments that the kernels share.
//
//   y[m, n] = sum_g s[n, g] * sum_{k in g} x[m, k] (u[n, k] - z[n, g])  [+ bias[n]]
//
// Layout.  Codes lie in blocks of 16 rows x 128 columns, 1 KiB, [row blocks][column blocks]: lane L's 16 bytes
// are four words, word s the eight codes k = 128 b + 32 s + 8 (L / 16) .. + 7 of row L % 16, which is the
// operand of one v_mfma_f32_16x16x32 (a wave's load of a block is one contiguous KiB).  Scales (bf16 or binary16)
// and zero points (bytes) lie as [row blocks][groups][16].
//
// Unpacking.  A code in the middle of a 16-bit float's mantissa is a number: with the exponent of 16 and the
// nibble in the top mantissa bits the float is 16 + u exactly.  The word holds the pairs (k0, k1), (k2, k3),
// (k4, k5), (k6, k7) at bits {3, 19}, {7, 23}, {11, 27}, {15, 31 wrapped}, so a pair takes one shift or rotation
// and one and-or: 7 operations for 8 codes (bf16; 8 in binary16, whose mantissa is longer).  Each group's
// product then carries (16 + z) sum(x) too much, which is taken off in binary32 before the group's scale; an
// offset of 16 costs the sum under 3 bits of binary32's 24, where the 128 of a whole bf16 mantissa would cost 5.
#pragma once

#include "h3q_common.hpp"
#include "h3q_kernels.hpp"

namespace h3q {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr uint32_t kW4Oob = 0x80000000u;  // beyond every descriptor's range: loads return 0
constexpr int kW4Stream = 2;              // cache policy of loads that are read once: non-temporal

template <bool F16>
__device__ __forceinline__ v4u w4_unpack(uint32_t w) {
    constexpr uint32_t mask = F16 ? 0x03C003C0u : 0x00780078u, one = F16 ? 0x4C004C00u : 0x41804180u;
    v4u d;
    d[0] = ((F16 ? w << 3 : w) & mask) | one;
    d[1] = ((F16 ? w >> 1 : w >> 4) & mask) | one;
    d[2] = ((F16 ? w >> 5 : w >> 8) & mask) | one;
    d[3] = (__builtin_amdgcn_alignbit(w, w, F16 ? 9 : 12) & mask) | one;
    return d;
}

template <bool F16>
__device__ __forceinline__ v4f w4_mfma(v4u a, v4u b, v4f c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0,
                                                       0);
}

__device__ __forceinline__ v4u w4_load16(__amdgpu_buffer_rsrc_t r, uint32_t off, int policy) {
    return policy == kW4Stream ? __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, kW4Stream)
                               : __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}

// A lane's four scales (one of four consecutive rows each) and zero points of a group.
__device__ __forceinline__ v4f w4_scales(v2u w, bool f16) {
    return f16 ? v4f{f16_lo(w[0]), f16_hi(w[0]), f16_lo(w[1]), f16_hi(w[1])}
               : v4f{bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
}
template <bool ZEROS>
__device__ __forceinline__ v4f w4_offsets(uint32_t z) {
    if constexpr (!ZEROS) return v4f{24.0f, 24.0f, 24.0f, 24.0f};  // 16 and a zero point of 8
    return v4f{16.0f + (float)(z & 255), 16.0f + (float)(z >> 8 & 255), 16.0f + (float)(z >> 16 & 255),
               16.0f + (float)(z >> 24)};
}

// out[m, n .. n + 3] = y + bias, rounded once; rows and columns past the end are dropped.
template <bool F16>
__device__ __forceinline__ void w4_store(const W4Args& p, int64_t m, int64_t n, v4f y) {
    if (m >= p.m || n >= p.n) return;
    const int cols = p.n - n < 4 ? (int)(p.n - n) : 4;
    if (p.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < cols) y[e] += out_lo(p.bias[n + e], F16);
    }
    uint16_t* const to = p.out + m * p.ldo + n;
    const uint32_t a = pack_out2(y[0], y[1], F16), b = pack_out2(y[2], y[3], F16);
    if (cols == 4 && p.out_vec) {
        *reinterpret_cast<uint2*>(to) = make_uint2(a, b);
    } else {
        const uint16_t h[4] = {(uint16_t)a, (uint16_t)(a >> 16), (uint16_t)b, (uint16_t)(b >> 16)};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < cols) to[e] = h[e];
    }
}

}  // namespace h3q
