// 4-bit weights with group scales: layout, unpacking and what the kernels share.
//
//   y[m, n] = sum_k x[m, k] * s[n, g] * (u[n, k] - z[n, g])  [+ bias[n]],   g = k / group
//
// Up to 16 rows (w4_stream.hpp) the integers go into the matrix instructions and a group's sum is scaled in
// binary32: bound by the weights' bytes, it has room for that.  Above (w4_slab.hip, w4_tile.hip) the weight s (u - z),
// which binary32 holds exactly, is rounded once to x's 16-bit type and summed over all of k in the matrix instructions'
// accumulators.  Against 64 bits the result is off by 1.3 times what the output's own rounding costs; what it saves is an
// fma and an offset for every output and group: scaling the sums was built for many rows too, and took 600 us for 4096
// rows of 14336 x 5376 at groups of 128 without zero points, 1330 us at groups of 32 with them, where this takes 492
// and 501 (each a loop of one call; 503 and more with inputs that change).  binary16 holds weights from 2^-14 to 65504 in
// full: below, where only bf16 scales reach, its subnormal steps are left of them.
//
// Layout.  Codes lie in blocks of 16 rows x 128 columns, 1 KiB, [row blocks][column blocks]: lane L's 16 bytes
// are four words, word s the eight codes k = 128 b + 32 s + 8 (L / 16) .. + 7 of row L % 16, the low nibbles of
// its bytes k0 .. k3 and the high ones k4 .. k7: the operand of one v_mfma_f32_16x16x32, and with the lanes' 16 bytes
// taken as row L % 32 and k quarter L / 32 (+ 2) of two blocks, of two v_mfma_f32_32x32x16.  Scales (bf16 or binary16) and zero
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

// Group of the 32-column step s of block b: floor((4 b + s) / (group / 32)), by a multiplication that is exact for
// k <= 2^22 and groups up to 2^18 (numerator and divisor are doubled so that a divisor of 1 has a reciprocal).
__device__ __forceinline__ int w4_group(const W4Args& p, int b, int s) {
    return (int)__umulhi((uint32_t)(8 * b + 2 * s + 1), p.group_magic);
}

// Scale and -(zero point) of a row for group e & 3 of the four in `s` and `z`; e is wave-uniform, so the choice is
// one byte permutation with a selector from a scalar register.  f16 is a mask: a condition would become a branch,
// which keeps the compiler from mixing the unpacking of one step with the matrix instructions of another.
template <bool ZEROS>
__device__ __forceinline__ void w4_scale(v2u s, uint32_t z, int e, uint32_t f16, float& scale, float& shift) {
    const uint32_t at = (uint32_t)(e & 3) * 0x0202u + 0x0100u;  // its two bytes
    const uint32_t bits = __builtin_amdgcn_perm(s[1], s[0], at << 16 | 0x0C0Cu);
    scale = __uint_as_float((__float_as_uint(f16_hi(bits)) & f16) | (bits & ~f16));
    shift = ZEROS ? -(float)(__builtin_amdgcn_perm(0u, z, (uint32_t)(e & 3)) & 255u) : -8.0f;
}

// A row's scale and zero point, and the weights that they make of its codes: s (u - z), rounded once to x's type.
// With binary16 on both sides u - z (exact) and the product are packed binary16 (15 operations for 8 codes); else an fma
// of u with s and -z s (exact in binary32) and a rounding (19): 4096 binary16 rows of 14336 x 5376 502 and 526 us.
template <bool F16, bool SF16, bool ZEROS>
struct W4Row {
    static constexpr bool PACKED = F16 && SF16;
    float scale, shift;  // 2^9 s and -z s
    v2h scale2, shift2;  // s and -z, twice

    __device__ __forceinline__ void set(v2u s, uint32_t z, int e) {
        if constexpr (PACKED) {
            const uint32_t at = (uint32_t)(e & 3) * 0x0202u + 0x0100u, place = (uint32_t)(e & 3) | 0x0C00u;
            scale2 = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(s[1], s[0], at << 16 | at));
            const v2h top = {(_Float16)1024.0f, (_Float16)1024.0f};  // with z in its last bits: 1024 + z
            if (ZEROS)
                shift2 = top - __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0u, z, place << 16 | place) | 0x64006400u);
            else
                shift2 = v2h{(_Float16)-8.0f, (_Float16)-8.0f};
        } else {
            w4_scale<ZEROS>(s, z, e, SF16 ? ~0u : 0u, scale, shift);
            shift *= scale;
            scale *= 512.0f;
        }
    }
    // Weights 2 q and 2 q + 1 of a word's eight.
    __device__ __forceinline__ uint32_t pair(uint32_t w, int q) const {
        const uint32_t codes = (q < 2 ? w : w >> 4) & 0x0F0F0F0Fu;
        if constexpr (PACKED) {
            const v2h u = q & 1 ? __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 512.0f, true))
                                : __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 512.0f, false));
            return __builtin_bit_cast(uint32_t, (u + shift2) * scale2);
        } else {
            const v2f u = q & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true)
                                : __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
            return w4_pair<F16>(__builtin_fmaf(u[0], scale, shift), __builtin_fmaf(u[1], scale, shift));
        }
    }
};

// A descriptor whose words are in scalar registers for sure: where the compiler loses sight of that, every load
// through it becomes a loop over the lanes' values.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_rsrc(const void* base, int64_t bytes) {
    const uint64_t b = (uint64_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)b), hi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    return make_rsrc((const void*)((uint64_t)hi << 32 | lo), __builtin_amdgcn_readfirstlane((uint32_t)bytes));
}

template <bool F16>
__device__ __forceinline__ v16f w4_mfma(v4u a, v4u b, v16f c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0,
                                                       0);
}

struct W4Tile {
    int m, n, z;  // row tile, column tile, part of k; in scalar registers
};

// Workgroups b, b + 8, ... share an XCD: each gets a contiguous run of tiles, in bands of 8 row tiles with the row
// tile fastest.
__device__ __forceinline__ W4Tile w4_tile_of(int mtiles, int ntiles, int splits) {
    const int total = mtiles * ntiles * splits;
    int id = blockIdx.x;
    const int q = total / 8, r = total % 8, x = id % 8;
    id = x * q + (x < r ? x : r) + id / 8;
    const int z = id % splits;
    id /= splits;
    const int band = id / (8 * ntiles), in = id % (8 * ntiles);
    const int high = mtiles - band * 8 < 8 ? mtiles - band * 8 : 8;
    // A division leaves the scalar registers.
    return {__builtin_amdgcn_readfirstlane(band * 8 + in % high), __builtin_amdgcn_readfirstlane(in / high),
            __builtin_amdgcn_readfirstlane(z)};
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
