// Product with 4-bit weights for some dozens of rows, gfx950: one launch, no sums in memory.
//
// A workgroup owns 64 rows (up to 32 rows in all: 32) x 32 NT columns and all of k, which its eight waves split: wave
// w takes the 128-column blocks w, w + 8, ... on its own, from a ring of x and a place for a block's codes in LDS that
// only it fills (buffer_load ... lds) and reads, so that there is no barrier before the last sums are joined there, in
// order.  Where w4_tile.hip splits k over workgroups it writes and reads binary32 sums and takes a second launch: 100
// rows of 4096 x 4096 11.6 us against 18.3, 40 rows of 5376 x 7168 14.1 against 16.7, 200 rows 26.5 against 29.5
// (loops of one call; the last 27.4 to 29.4 over cards and changing inputs).  Up to 16 rows w4_stream.hpp keeps the
// weights exact; two of its row tiles took 32 rows of 5376 x 7168 in 18.3 us where this takes 12.4, 17 rows in 13.2 and
// 10.0.
//
// Everything that is fetched goes through LDS copies, whose count is known at every point; with a load into registers
// among them the compiler's own wait for it would count the copies behind it as done too early.  x comes in
// quarters of a block (32 columns, 64 bytes of a row; chunk c of a row lies in slot c ^ (row / 4 % 4), which
// keeps eight rows' reads of one chunk apart).  One step of 16 k ahead the operands are read and unpacked
// between the matrix instructions, and the copies are asked for there one at a time.  Eight waves and not four: a
// wave alone on its SIMD issues a vector instruction of 8 bytes every 8 cycles, two share them at one every 4.  What bounds
// it at 200 rows of 5376 x 7168: the vector port (some 560 instructions a wave and block, and 16 cycles of each
// of 48 matrix instructions) for 17 of the 26 us, without the copies 22 in all, and the copies' waits.
#include "w4.hpp"

namespace h3q {

namespace {

// One dword per lane, global -> LDS (as copy16).
__device__ __forceinline__ void copy4(const CopySrc& src, uint32_t lds_base, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(lds_base), "v"(voff), "s"(src.d)
                 : "memory");
}

// A block's loop has 8 MT steps, 2 MT to a quarter, each with one copy of x and, in the first half, as many of the
// next block's codes: how many of those come before step `at` of the block.
template <int MT, int CODE_COPIES>
constexpr int code_copies(int at) {
    const int n = (CODE_COPIES + 4 * MT - 1) / (4 * MT) * at;
    return n < CODE_COPIES ? n : CODE_COPIES;
}
// Copies that may be under way in the middle of quarter q, when the x of quarter q + 1 has to be there: those asked
// for behind it, which are RING - 3 quarters and a half.  (The codes, of quarters 0 and 1, are there in the third.)
template <int MT, int RING, int CODE_COPIES>
constexpr int asked(int q) {
    static_assert(RING == 3 || RING == 4, "a quarter of the last block that could be behind it has no codes");
    const int from = q + 3 - RING;  // the first quarter behind it; -1: the last block's last
    return 2 * MT * (q - from) + MT + code_copies<MT, CODE_COPIES>(2 * MT * q + MT) -
           code_copies<MT, CODE_COPIES>(2 * MT * (from < 0 ? 0 : from));
}

template <bool F16, bool SF16, bool ZEROS, int NT, int MT>
__global__ __launch_bounds__(512) void w4_slab_kernel(W4Args p, int mtiles, int ntiles) {
    constexpr int WAVES = 8, RING = NT == 1 || MT == 1 ? 4 : 3, XSTAGE = MT * 32 * 64;
    constexpr int CODES = NT * (2048 + 256 + (ZEROS ? 256 : 0)), COPIES = 2 * MT, CODE_COPIES = NT * (ZEROS ? 4 : 3);
    constexpr int WAVE = RING * XSTAGE + CODES;
    static_assert(WAVES * WAVE >= NT * 4 * WAVES * 1024, "the sums of a row tile");
    __shared__ __attribute__((aligned(1024))) uint8_t lds_raw[WAVES * WAVE];
    H3Q_LDS uint8_t* const lds = (H3Q_LDS uint8_t*)lds_raw;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, half = lane >> 5;
    const W4Tile at = w4_tile_of(mtiles, ntiles, 1);

    const int64_t m0 = (int64_t)at.m * 32 * MT;
    const int blk0 = at.n * 2 * NT, blocks = (int)((p.n + 15) / 16);
    const int nblk = blocks - blk0 < 2 * NT ? blocks - blk0 : 2 * NT;
    const int steps = (int)((p.k + 127) / 128), quads = (p.groups + 3) / 4;
    const int64_t rows = p.m - m0 < 32 * MT ? p.m - m0 : 32 * MT;
    const CopySrc rx(p.x + m0 * p.ldx, (uint32_t)(((rows - 1) * p.ldx + p.k) * 2));
    const CopySrc rw(p.codes + (int64_t)blk0 * steps * 1024, (uint32_t)((int64_t)nblk * steps * 1024));
    const CopySrc rs(p.scales + (int64_t)blk0 * quads * 64, (uint32_t)((int64_t)nblk * quads * 128));
    const CopySrc rz(p.zeros + (ZEROS ? (int64_t)blk0 * quads * 64 : 0), (uint32_t)(ZEROS ? (int64_t)nblk * quads * 64 : 0));
    const uint32_t row_bytes = (uint32_t)(p.ldx * 2);

    H3Q_LDS uint8_t* const mine = lds + wave * WAVE;
    const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)mine), codes_base = base + RING * XSTAGE;
    // A copy instruction takes 64 bytes of 16 rows; chunk c of a row lies in slot c ^ (row / 4 % 4).
    const int chunk = (lane & 3) ^ (lane >> 4);
    const uint32_t xat = (uint32_t)(lane >> 2) * row_bytes + 16u * chunk;
    auto ask_x = [&](int b, int q, int r, int i) __attribute__((always_inline)) {
        const bool ok = b < steps && 128 * b + 32 * q + 8 * chunk < p.k;
        const uint32_t off = ok ? xat + 256u * b + 64u * q : kW4Oob;  // past the range from there on, too
        copy16(rx, base + r * XSTAGE + i * 1024, off + 16u * i * row_bytes);
    };
    auto ask_codes = [&](int b, int o) __attribute__((always_inline)) {  // copy o of CODE_COPIES
        const bool ok = b < steps;
        const int j = o - 2 * NT, quad = (2 * (j % NT) + (lane >> 5)) * quads + (w4_group(p, b, 0) >> 2);
        if (o < 2 * NT)
            copy16(rw, codes_base + o * 1024, (ok ? (uint32_t)b * 1024u + 16u * lane : kW4Oob) + (uint32_t)(o * steps) * 1024u);
        else if (j < NT)
            copy4(rs, codes_base + NT * 2048 + j * 256, ok ? (uint32_t)quad * 128u + 4u * (lane & 31) : kW4Oob);
        else if (o < CODE_COPIES)
            copy4(rz, codes_base + NT * 2304 + (j - NT) * 256,
                  ok && (lane & 16) == 0 ? (uint32_t)quad * 64u + 4u * (lane & 15) : kW4Oob);
    };

    v16f acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = v16f{};
    v4u codes[NT][2], w[2][NT], x[2][MT];
    v2u scales[NT];
    uint32_t zeros[NT];
    W4Row<F16, SF16, ZEROS> row[NT];
    auto fetch = [&]() __attribute__((always_inline)) {
        const H3Q_LDS uint8_t* const from = mine + RING * XSTAGE;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const H3Q_LDS uint8_t* const c = from + (2 * j + (r32 >> 4)) * 1024 + ((r32 & 15) + 16 * half) * 16;
            codes[j][0] = *(const H3Q_LDS v4u*)c;
            codes[j][1] = *(const H3Q_LDS v4u*)(c + 512);
            scales[j] = *(const H3Q_LDS v2u*)(from + NT * 2048 + j * 256 + r32 * 8);
            zeros[j] = ZEROS ? *(const H3Q_LDS uint32_t*)(from + NT * 2304 + j * 256 + (r32 >> 4) * 128 + (r32 & 15) * 4) : 0u;
        }
    };
    uint32_t xoff[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) xoff[c] = r32 * 64 + 16 * ((2 * c + half) ^ (r32 >> 2 & 3));
    auto read = [&](int g, int t, int r) __attribute__((always_inline)) {
        x[g & 1][t] = *(const H3Q_LDS v4u*)(mine + r * XSTAGE + xoff[g & 1] + t * 32 * 64);
    };
    auto unpack = [&](int b, int g, int t) __attribute__((always_inline)) {  // part t of MT for step g of block b
#pragma unroll
        for (int q = 4 * NT / MT * t; q < 4 * NT / MT * (t + 1); ++q) {
            const int j = q / 4;
            if (q % 4 == 0 && g % 2 == 0) row[j].set(scales[j], zeros[j], w4_group(p, b, g / 2));
            w[g & 1][j][q % 4] = row[j].pair(codes[j][g & 1][g / 2], q % 4);
        }
    };

    const int b0 = wave;
#pragma unroll
    for (int o = 0; o < CODE_COPIES; ++o) ask_codes(b0, o);
#pragma unroll
    for (int q = 0; q < RING - 1; ++q)
#pragma unroll
        for (int i = 0; i < COPIES; ++i) ask_x(b0, q, q, i);
    wait_vmcnt<(RING - 2) * COPIES>();
    fetch();
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        read(0, t, 0);
        unpack(b0, 0, t);
    }
    int r = 0;
    for (int b = b0; b < steps; b += WAVES) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r1 = r == RING - 1 ? 0 : r + 1, last = r == 0 ? RING - 1 : r - 1;
            if (q == 0) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the fetch: its place is filled again
#pragma unroll
            for (int g = 2 * q; g < 2 * q + 2; ++g) {
                if (g & 1) {
                    if (q == 0) wait_vmcnt<asked<MT, RING, CODE_COPIES>(0)>();
                    else if (q == 1) wait_vmcnt<asked<MT, RING, CODE_COPIES>(1)>();
                    else if (q == 2) wait_vmcnt<asked<MT, RING, CODE_COPIES>(2)>();
                    else wait_vmcnt<asked<MT, RING, CODE_COPIES>(3)>();
                    if (q == 3) fetch();
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    read(g + 1, t, g & 1 ? r1 : r);
                    unpack(g == 7 ? b + WAVES : b, (g + 1) & 7, t);
                    ask_x(q + RING - 1 < 4 ? b : b + WAVES, (q + RING - 1) & 3, last, (g & 1) * MT + t);
#pragma unroll
                    for (int o = code_copies<MT, CODE_COPIES>(g * MT + t); o < code_copies<MT, CODE_COPIES>(g * MT + t + 1); ++o)
                        ask_codes(b + WAVES, o);
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[j][t] = w4_mfma<F16>(w[g & 1][j], x[g & 1][t], acc[j][t]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            r = r1;
        }
    }
    wait_vmcnt0();

    H3Q_LDS v4f* const sums = (H3Q_LDS v4f*)lds;  // [column tile and quarter][wave][lane]
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                sums[((j * 4 + v) * WAVES + wave) * 64 + lane] =
                    v4f{acc[j][t][4 * v], acc[j][t][4 * v + 1], acc[j][t][4 * v + 2], acc[j][t][4 * v + 3]};
        __syncthreads();
        for (int u = wave; u < 4 * NT; u += WAVES) {
            const H3Q_LDS v4f* const from = sums + u * WAVES * 64 + lane;
            v4f y = from[0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) y += from[i * 64];
            w4_store<F16>(p, m0 + 32 * t + r32, 16 * (int64_t)blk0 + 8 * u + 4 * half, y);
        }
    }
}

template <bool F16, bool SF16, bool ZEROS, int MT>
hipError_t launch_cols(const W4Args& a, int nt, hipStream_t st) {
    const int mtiles = (int)((a.m + 32 * MT - 1) / (32 * MT)), ntiles = (int)((a.n + 32 * nt - 1) / (32 * nt));
    const dim3 grid((unsigned)(mtiles * ntiles));
    if (nt == 1) hipLaunchKernelGGL((w4_slab_kernel<F16, SF16, ZEROS, 1, MT>), grid, dim3(512), 0, st, a, mtiles, ntiles);
    else if (nt == 2) hipLaunchKernelGGL((w4_slab_kernel<F16, SF16, ZEROS, 2, MT>), grid, dim3(512), 0, st, a, mtiles, ntiles);
    else hipLaunchKernelGGL((w4_slab_kernel<F16, SF16, ZEROS, 3, MT>), grid, dim3(512), 0, st, a, mtiles, ntiles);
    return hipGetLastError();
}

template <bool F16, bool SF16, bool ZEROS>
hipError_t launch_rows(const W4Args& a, int nt, hipStream_t st) {
    return a.m <= 32 ? launch_cols<F16, SF16, ZEROS, 1>(a, nt, st) : launch_cols<F16, SF16, ZEROS, 2>(a, nt, st);
}

template <bool F16, bool SF16>
hipError_t launch_zeros(const W4Args& a, int nt, hipStream_t st) {
    return a.zeros ? launch_rows<F16, SF16, true>(a, nt, st) : launch_rows<F16, SF16, false>(a, nt, st);
}

}  // namespace

hipError_t launch_w4_slab(const W4Args& a, int nt, hipStream_t st) {
    if (a.f16) return a.scales_f16 ? launch_zeros<true, true>(a, nt, st) : launch_zeros<true, false>(a, nt, st);
    return a.scales_f16 ? launch_zeros<false, true>(a, nt, st) : launch_zeros<false, false>(a, nt, st);
}

}  // namespace h3q
