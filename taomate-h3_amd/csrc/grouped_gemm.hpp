// What the grouped products share: the matrix instructions, the tile of a workgroup and
// the SwiGLU of an epilogue.
#pragma once

#include "h3q_common.hpp"
#include "h3q_kernels.hpp"

namespace h3q {

constexpr uint32_t kOob = 0x80000000u;  // beyond every descriptor's range: loads return 0

__device__ __forceinline__ v8i join(v4u lo, v4u hi) {
    return v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
__device__ __forceinline__ v8i join(v4i lo, v4i hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// 16 x 16 products of 128-byte fragments (row = lane % 16, bytes 32 (lane / 16) .. + 31
// of each operand); the first operand's rows are accumulator rows 4 (lane / 16) + v.
// WIDE (e4m3): the codes become bf16, exactly, and four bf16 instructions take the place of
// the FP8 one.  The FP8 instruction drops the low bits of small products inside each group
// of 8 (2^-13 of the largest): 1.5e-5 to 3e-5 of the result, which the rounding of an
// output hides, but which moves one code in a thousand to its neighbour where the output is
// quantized again; bf16 products leave 5e-8 to 1e-7 (K = 1024 to 5376, measured).  Where
// weights are streamed the conversions and the slower instruction hide under the loads.
template <int OP, bool WIDE = false>
struct GroupedMfma;
template <>
struct GroupedMfma<kOpE4M3, false> {
    using acc_t = v4f;
    using frag_t = v8i;
    static __device__ __forceinline__ frag_t frag(v8i codes) { return codes; }
    static __device__ __forceinline__ acc_t run(frag_t a, frag_t b, acc_t c) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
    }
};
template <>
struct GroupedMfma<kOpE4M3, true> {
    using acc_t = v4f;
    struct frag_t {
        v8bf q[4];
    };
    static __device__ __forceinline__ frag_t frag(v8i codes) {
        frag_t f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v2bf lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)codes[2 * i + h], 1.0f, false);
                const v2bf hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)codes[2 * i + h], 1.0f, true);
                f.q[i][4 * h] = lo[0];
                f.q[i][4 * h + 1] = lo[1];
                f.q[i][4 * h + 2] = hi[0];
                f.q[i][4 * h + 3] = hi[1];
            }
        return f;
    }
    static __device__ __forceinline__ acc_t run(const frag_t& a, const frag_t& b, acc_t c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.q[i], b.q[i], c, 0, 0, 0);
        return c;
    }
};
template <bool WIDE>
struct GroupedMfma<kOpInt8, WIDE> {
    using acc_t = v4i;
    using frag_t = v8i;
    static __device__ __forceinline__ frag_t frag(v8i codes) { return codes; }
    static __device__ __forceinline__ acc_t run(frag_t a, frag_t b, acc_t c) {
        const v4i alo = {a[0], a[1], a[2], a[3]}, ahi = {a[4], a[5], a[6], a[7]};
        const v4i blo = {b[0], b[1], b[2], b[3]}, bhi = {b[4], b[5], b[6], b[7]};
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(alo, blo, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(ahi, bhi, c, 0, 0, 0);
    }
};

// What a grouped product stores.  kOutWide: SwiGLU from wide products.
enum GroupedOut : int { kOutBF16 = 0, kOutF32 = 1, kOutSwiglu = 2, kOutWide = 3 };

// silu(g) * u in binary32: exp(-g) by the hardware exp2, the quotient by its reciprocal (one
// unit in the last place; an IEEE division is ten instructions, which an epilogue without
// another wave to hide it pays in full).  The reciprocal instruction makes 0 of results below
// 2^-126, which 1 / (1 + e) is for g in (-88.7, -87.3): quotient and gate are taken at 8 times
// and an eighth of their size, powers of two that change no other result.  Below -88.7 e is
// infinite and the result 0, as the quotient's.  g = -inf gives NaN, as -inf / inf does.
__device__ __forceinline__ float swiglu_f32(float g, float u) {
    const float e = __builtin_amdgcn_exp2f(-g * 0x1.715476p+0f);
    return 0.125f * g * __builtin_amdgcn_rcpf(__builtin_fmaf(e, 0.125f, 0.125f)) * u;
}

// Rows of one expert that a workgroup's tile covers.
struct GroupTile {
    int expert;
    int64_t row0;
    int rows;  // 0: no tile
};

// Tiles of BM rows.  Expert e owns the tile numbers from e + offsets[e] / BM on: floor(hi /
// BM) - floor(lo / BM) + 1 of them, always enough for its hi - lo rows, so experts + rows /
// BM numbers cover every split of the rows, and a workgroup finds its own from the offsets
// alone (one load a lane per 64 experts), without a prefix sum over the experts' tile counts.
// The bounds come from device memory and are clamped to the rows that the call was given.
__device__ __forceinline__ int64_t tile_number(const int* offsets, int bm, int e) {
    return e + (int64_t)offsets[e] / bm;
}

// The expert that owns a tile number.
__device__ __forceinline__ int tile_expert(const int* offsets, int experts, int bm, int64_t tile) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int i = 0; i < experts; i += 64) {
        const int e = i + lane;
        n += __popcll(__ballot(e < experts && tile_number(offsets, bm, e < experts ? e : 0) <= tile));
    }
    return __builtin_amdgcn_readfirstlane(n > 0 ? n - 1 : 0);
}

__device__ __forceinline__ GroupTile tile_rows(const int* offsets, int64_t rows, int bm, int expert, int64_t m) {
    GroupTile t;
    t.expert = expert;
    int64_t lo = offsets[expert], hi = offsets[expert + 1];
    lo = lo < 0 ? 0 : (lo > rows ? rows : lo);
    hi = hi < lo ? lo : (hi > rows ? rows : hi);
    t.row0 = lo + m * bm;
    const int64_t left = m < 0 ? 0 : hi - t.row0;
    t.rows = (int)(left < 0 ? 0 : (left > bm ? bm : left));
    return t;
}

// Tile number `tile`.
__device__ __forceinline__ GroupTile group_tile(const int* offsets, int experts, int64_t rows, int bm, int tile) {
    const int e = tile_expert(offsets, experts, bm, tile);
    return tile_rows(offsets, rows, bm, e, tile - tile_number(offsets, bm, e));
}

// Work item of workgroup bid among the experts' tiles (whole ones and a last, partial one, no
// empty ones) x column slices: each XCD (bid % 8) gets a contiguous run of equal length, and in
// an expert the tiles of one slice are neighbours, so an expert's weights and rows pass
// through one L2, about once.  (Numbers of group_tile would leave gaps, uneven over the
// XCDs.)  Every wave sums the experts' tile counts for itself.  False: no item.
__device__ __forceinline__ bool group_item(const int* offsets, int experts, int64_t rows, int bm, int slices, int bid,
                                           GroupTile& tile, int& slice) {
    const int lane = threadIdx.x & 63;
    // Tiles of expert i + lane, and (first) those of the experts below it in its 64.
    auto tiles = [&](int i, int& own, int& upto) __attribute__((always_inline)) {
        own = 0;
        if (i + lane < experts) {
            int64_t lo = offsets[i + lane], hi = offsets[i + lane + 1];
            lo = lo < 0 ? 0 : (lo > rows ? rows : lo);
            hi = hi < lo ? lo : (hi > rows ? rows : hi);
            own = (int)((hi - lo + bm - 1) / bm);
        }
        upto = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d, 64);
            if (lane >= d) upto += o;
        }
    };
    int own, upto;
    int64_t total = 0;
    for (int i = 0; i < experts; i += 64) {
        tiles(i, own, upto);
        total += __builtin_amdgcn_readlane(upto, 63);
    }
    const int64_t items = total * slices, per = (items + 7) / 8, item = (bid & 7) * per + (bid >> 3);
    if ((bid >> 3) >= per || item >= items) return false;
    int64_t below = 0;
    for (int i = 0; i < experts; i += 64) {
        if (experts > 64) tiles(i, own, upto);
        const uint64_t past = __ballot((below + upto) * slices > item);  // the first of them holds the item
        if (past) {
            const int l = __builtin_ctzll(past);
            const int count = __builtin_amdgcn_readlane(own, l);
            const int rest = (int)(item - (below + __builtin_amdgcn_readlane(upto, l) - count) * slices);
            slice = rest / count;
            tile = tile_rows(offsets, rows, bm, i + l, rest % count);
            return tile.rows > 0;
        }
        below += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

}  // namespace h3q
