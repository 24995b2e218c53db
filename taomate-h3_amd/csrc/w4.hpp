// 4-bit weights with group scales: layout, unpacking and what the kernels share.
//
//   y[m, n] = sum_k x[m, k] * w[n, k]  [+ bias[n]],   w[n, k] = rn(s[n, g] * (u[n, k] - z[n, g])), g = k / group
//
// The weight is rounded once, to x's 16-bit type, because the matrix instructions multiply that type; the product
// before it is exact in binary32 (an 11-bit scale times a 5-bit integer), so w is one definite matrix, the same
// for every kernel and row count.  It costs 1.1 times the rounding error of the output alone.  The other way, the
// integers in the matrix instructions and the scale on every group's sum, was built and measured first: 4096 rows of
// 14336 x 5376 took 600 us at groups of 128 without zero points, but 1330 us at groups of 32 with them, because
// each group costs an fma and an offset for every output, where rounding costs the same for all groups.
//
// Layout.  Codes lie in blocks of 16 rows x 128 columns, 1 KiB, [row blocks][column blocks]: lane L's 16 bytes
// are four words, word s the eight codes k = 128 b + 32 s + 8 (L / 16) .. + 7 of row L % 16, from the low nibble
// k0 k2 k4 k6 k1 k3 k5 k7: the operand of one v_mfma_f32_16x16x32, and with the lanes' 16 bytes taken as row L % 32
// and k quarter L / 32 (+ 2) of two blocks, of two v_mfma_f32_32x32x16.  Scales (bf16 or binary16) and zero
// points (bytes) lie as [row blocks][groups / 4][16][4]: a lane's row has four groups in one load.
//
// Unpacking.  A byte 0 .. 15 is the e4m3 number of 2^-9 times its value (subnormals up to 7, then the first
// binade, of the same step), so v_cvt_pk_f32_fp8 turns two masked nibbles into binary32 at once: three mask
// operations, four conversions, eight fmas with 2^9 s and -z s, four roundings to pairs for eight codes.
#pragma once

#include "h3q_common.hpp"
#include "h3q_kernels.hpp"

namespace h3q {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr uint32_t kW4Oob = 0x80000000u;  // beyond every descriptor's range: loads return 0

template <bool F16>
__device__ __forceinline__ uint32_t w4_pair(float lo, float hi) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{lo, hi}, v2h));
    else return pack_bf16x2(lo, hi);
}

// Eight codes of a row -> its weights: scale = 2^9 s, shift = -z s.
template <bool F16>
__device__ __forceinline__ v4u w4_weights(uint32_t w, float scale, float shift) {
    const int even = (int)(w & 0x0F0F0F0Fu), odd = (int)(w >> 4 & 0x0F0F0F0Fu);
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(even, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(even, true);
    const v2f c = __builtin_amdgcn_cvt_pk_f32_fp8(odd, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(odd, true);
    const auto f = [&](float v) { return __builtin_fmaf(v, scale, shift); };
    return v4u{w4_pair<F16>(f(a[0]), f(b[0])), w4_pair<F16>(f(c[0]), f(d[0])), w4_pair<F16>(f(a[1]), f(b[1])),
               w4_pair<F16>(f(c[1]), f(d[1]))};
}

// Scale and shift of a row for its group `e` of the four in `s` and `z` (e wave-uniform).
__device__ __forceinline__ void w4_group(v2u s, uint32_t z, int e, bool f16, float& scale, float& shift) {
    const uint32_t pair = e & 2 ? s[1] : s[0], bits = e & 1 ? pair >> 16 : pair;
    const float v = f16 ? f16_lo(bits) : bf16_lo(bits);
    scale = v * 512.0f;
    shift = -v * (float)(z >> (8 * e) & 255u);
}

// A descriptor whose words are in scalar registers for sure: where the compiler loses sight of that, every load
// through it becomes a loop over the lanes' values.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_rsrc(const void* base, int64_t bytes) {
    const uint64_t b = (uint64_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)b), hi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    return make_rsrc((const void*)((uint64_t)hi << 32 | lo), __builtin_amdgcn_readfirstlane((uint32_t)bytes));
}

// The four-group entry of block b's first group, and the group of its 32-column step s in that entry.
__device__ __forceinline__ int w4_quad(const W4Args& p, int b) {
    return p.group_shift >= 0 ? b >> p.group_shift : b / (4 * p.blocks_per_group);
}
__device__ __forceinline__ int w4_element(const W4Args& p, int b, int s) {
    if (p.group < 128) return p.group == 32 ? s : 2 * (b & 1) + (s >> 1);
    return (p.group_shift >= 0 ? b >> (p.group_shift - 2) : b / p.blocks_per_group) & 3;
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
