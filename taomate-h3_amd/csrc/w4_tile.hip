// Product with 4-bit weights for many rows, gfx950: bound by the matrix instructions (and, below 128 rows to a
// tile, by the unpacking: 19 operations for 8 codes, once for every row tile).
//
// A workgroup of four waves owns a tile of 32 MT rows x 128 NT columns, each wave all rows and 32 NT of the
// columns, so every code is unpacked once in a workgroup, straight into operand registers.  Per 128 columns of k the
// x tile is copied into one of two LDS stages (buffer_load ... lds, no registers; a row is 256 contiguous bytes, its
// 16-byte chunk c in slot c ^ (row % 16), so that 16 rows' reads of one chunk meet no bank twice), and the codes,
// scales and zero points into registers, one block ahead.  One barrier a block.  Inside a block the operands of the
// next 16 columns are read and unpacked between the matrix instructions of these, and the next block's copies and loads
// issued there one at a time, in pieces that the scheduler must not gather: 4096 rows of 14336 x 5376 492 us, 511 with
// the copies and loads together, 549 in the compiler's order (loops of one call; 502 to 527 over cards and changing inputs).
// The library's bf16 product with the unpacked weights takes 417 (481 with them as [k, n]).  A matrix
// instruction keeps the vector port for 16 of its 32 cycles, whoever wants it, so the unpacking hides behind half.
//
// Few tiles: k is split over several workgroups, whose binary32 sums a last kernel adds in order.
#include "w4.hpp"

namespace h3q {

namespace {

struct TileArgs {
    W4Args w;
    float* parts;  // [splits][m][npad], null: not split
    int npad, mtiles, ntiles, splits, per_split, steps;
};

// Four columns of a row: the result, or this part of k's share of it.
template <bool F16>
__device__ __forceinline__ void store_sums(const TileArgs& p, int z, int64_t m, int64_t n, v4f y) {
    if (p.parts) {
        if (m < p.w.m && n < p.npad) *reinterpret_cast<v4f*>(p.parts + (z * p.w.m + m) * p.npad + n) = y;
    } else {
        w4_store<F16>(p.w, m, n, y);
    }
}

template <bool F16, bool SF16, bool ZEROS, int NT, int MT>
__global__ __launch_bounds__(256, 2) void w4_tile_kernel(TileArgs p) {
    constexpr int D = 2, STAGE = MT * 32 * 256;
    __shared__ __attribute__((aligned(1024))) uint8_t lds_raw[D * STAGE];
    H3Q_LDS uint8_t* const lds = (H3Q_LDS uint8_t*)lds_raw;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, half = lane >> 5;

    const W4Tile at = w4_tile_of(p.mtiles, p.ntiles, p.splits);

    const int64_t m0 = (int64_t)at.m * 32 * MT;
    const int blk0 = at.n * 8 * NT + wave * 2 * NT, blocks = (int)((p.w.n + 15) / 16);
    const int nblk = blocks - blk0 < 0 ? 0 : blocks - blk0 < 2 * NT ? blocks - blk0 : 2 * NT;
    const int steps = p.steps, quads = (p.w.groups + 3) / 4;
    const int64_t rows = p.w.m - m0 < 32 * MT ? p.w.m - m0 : 32 * MT;
    const CopySrc rx(p.w.x + m0 * p.w.ldx, (uint32_t)(((rows - 1) * p.w.ldx + p.w.k) * 2));
    const int64_t first = nblk > 0 ? blk0 : 0;
    const __amdgpu_buffer_rsrc_t rw = w4_rsrc(p.w.codes + first * steps * 1024, (int64_t)nblk * steps * 1024);
    const __amdgpu_buffer_rsrc_t rs = w4_rsrc(p.w.scales + first * quads * 64, (int64_t)nblk * quads * 128);
    const __amdgpu_buffer_rsrc_t rz =
        w4_rsrc(p.w.zeros + (ZEROS ? first * quads * 64 : 0), ZEROS ? (int64_t)nblk * quads * 64 : 0);
    const uint32_t row_bytes = (uint32_t)(p.w.ldx * 2);

    // A copy instruction takes four rows; wave w the rows 4 w .. + 3 of every 16.
    const int crow = 4 * wave + (lane >> 4), chunk = (lane & 15) ^ crow;
    constexpr int COPIES = 2 * MT;
    auto copy = [&](int b, int stage, int i) __attribute__((always_inline)) {
        const uint32_t base = (uint32_t)(uintptr_t)(lds + stage * STAGE);
        const uint32_t off =
            128 * b + 8 * chunk < p.w.k ? crow * row_bytes + 256u * b + 16u * chunk : kW4Oob;
        copy16(rx, base + (wave + 4 * i) * 1024, off + 16u * i * row_bytes);  // past the range from kW4Oob on, too
    };
    // Row r32 of 32-column tile j: its block and place there; k quarters half and half + 2.
    uint32_t code_off[NT], scale_off[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int blk = 2 * j + (r32 >> 4);
        code_off[j] = (uint32_t)(blk * steps * 1024 + ((r32 & 15) + 16 * half) * 16);
        scale_off[j] = (uint32_t)(blk * quads * 16 + (r32 & 15));
    }
    v4u codes[D][NT][2];
    v2u scales[D][NT];
    uint32_t zeros[D][NT];
    constexpr int LOADS = NT * (ZEROS ? 4 : 3);
    auto load = [&](int b, int stage, int o) __attribute__((always_inline)) {
        const int j = o % NT, q = w4_group(p.w, b, 0) >> 2;
        if (o < 2 * NT)
            codes[stage][j][o / NT] = __builtin_amdgcn_raw_buffer_load_b128(rw, code_off[j] + 1024u * b + 512u * (o / NT), 0, 0);
        else if (o < 3 * NT)
            scales[stage][j] = __builtin_amdgcn_raw_buffer_load_b64(rs, (scale_off[j] + 16u * q) * 8, 0, 0);
        else
            zeros[stage][j] = __builtin_amdgcn_raw_buffer_load_b32(rz, (scale_off[j] + 16u * q) * 4, 0, 0);
    };
#pragma unroll
    for (int j = 0; j < NT; ++j) zeros[0][j] = zeros[1][j] = 0;

    v16f acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = v16f{};
    // This lane's chunk of step (s, h) in a row: 4 s + 2 h + half.
    uint32_t xoff[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) xoff[c] = r32 * 256 + 16 * ((2 * c + half) ^ (r32 & 15));

    const int b0 = at.z * p.per_split, b1 = b0 + p.per_split < steps ? b0 + p.per_split : steps;
    // A block's copies and loads, one at a time.  Past b1 the copies are out of range and the loads repeat.
    auto ask = [&](int b, int stage, int o) __attribute__((always_inline)) {
        if (o < COPIES) copy(b < b1 ? b : steps, stage, o);
        else if (o < COPIES + LOADS) load(b < b1 ? b : b1 - 1, stage, o - COPIES);
    };
#pragma unroll
    for (int o = 0; o < COPIES + LOADS; ++o) ask(b0, 0, o);
    static_assert(COPIES + LOADS <= 8 * MT, "one at each step of the loop");
    for (int b = b0; b < b1; b += D) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
            if (b + i >= b1) break;
            wait_vmcnt0();    // this wave's part of stage i has landed
            __syncthreads();  // everyone's has, and every wave is done with the stage before it
            const H3Q_LDS uint8_t* const tile = lds + i * STAGE;
            // Operands one step of 16 k ahead, the next block's copies and loads one at a time: between two matrix
            // instructions' issues a read, a part of the unpacking and one of those.
            v4u x[2][MT], w[2][NT];
            W4Row<F16, SF16, ZEROS> row[NT];
            auto prepare = [&](int g, int t) __attribute__((always_inline)) {  // part t of MT for step g
                x[g & 1][t] = *(const H3Q_LDS v4u*)(tile + xoff[g] + t * 32 * 256);
#pragma unroll
                for (int q = 4 * NT / MT * t; q < 4 * NT / MT * (t + 1); ++q) {
                    const int j = q / 4;
                    if (q % 4 == 0 && g % 2 == 0) row[j].set(scales[i][j], zeros[i][j], w4_group(p.w, b + i, g / 2));
                    w[g & 1][j][q % 4] = row[j].pair(codes[i][j][g & 1][g / 2], q % 4);
                }
            };
#pragma unroll
            for (int t = 0; t < MT; ++t) prepare(0, t);
#pragma unroll
            for (int g = 0; g < 8; ++g)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    if (g < 7) prepare(g + 1, t);
                    ask(b + i + 1, 1 - i, g * MT + t);
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[j][t] = w4_mfma<F16>(w[g & 1][j], x[g & 1][t], acc[j][t]);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
    wait_vmcnt0();  // the last copies

#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const v4f y = {acc[j][t][4 * v], acc[j][t][4 * v + 1], acc[j][t][4 * v + 2], acc[j][t][4 * v + 3]};
                const int64_t m = m0 + 32 * t + r32, n = 16 * (int64_t)blk0 + 32 * j + 8 * v + 4 * half;
                store_sums<F16>(p, at.z, m, n, y);
            }
}

template <bool F16>
__global__ __launch_bounds__(256) void w4_join_kernel(TileArgs p) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    const int64_t m = at / p.npad, n = at - m * p.npad;
    if (m >= p.w.m) return;
    v4f s = *reinterpret_cast<const v4f*>(p.parts + at);
    for (int z = 1; z < p.splits; ++z) s += *reinterpret_cast<const v4f*>(p.parts + z * p.w.m * p.npad + at);
    w4_store<F16>(p.w, m, n, s);
}

struct Plan {
    int nt, mt, splits, per_split, mtiles, ntiles, steps, npad, slab;  // slab: its 32-column tiles, or 0
    int64_t parts_bytes;
};

// 128 x 256 tiles where they fill the chip (4096 rows of 14336 x 5376 in a loop: 492 us, 1285 TFLOP/s; 128 x 128: 553,
// 64 x 128: 642).  Else 128 columns, of 128 rows or, where that pads the rows by over a seventh, of 64, and k in as many
// parts as give about two workgroups to a CU (600 rows of 5376 x 7168: 57 us with 128 rows in two parts, 70 with 64),
// each of at least four blocks.
//
// Or w4_slab.hip, whose waves split k inside a workgroup, when it is estimated to take less.  The estimate, in
// 1/20 of 0.87 us, is a line through 48 shapes (40 to 600 rows, 1024 to 14336 columns, k 4096 to 16384): a workgroup
// of it takes 20 (1 + NT) for eight blocks (13 up to 32 rows), a tile 22 or 15 (64 rows) a block, each once for 256 workgroups, beside
// 80 there, and 60 or, with sums in memory and their launch, 240 here.  Measured in loops of one call, us, slab and tile, the chosen one
// first: 64 rows of 1024 x 4096 8.2 and 10.6, 40 of 5376 x 7168 14.1 and 16.7, 200 of 4096 x 4096 14.0 and 20.2, 200 of
// 5376 x 7168 26.5 and 29.5; tile and slab: 64 of 2048 x 16384 19.3 and 32.5, 384 of 5376 x 7168 39 and 46, 600 of it
// 57 and 81, 256 of 14336 x 5376 48 and 63.  At two of the 48 the other one is better, by 4 and 19 % (128 of 10752 x
// 5376: tile 26.4, slab 22.2).
Plan plan_tiles(int64_t m, int64_t n, int64_t k) {
    Plan p{};
    p.steps = (int)((k + 127) / 128);
    const auto tiles = [&](int nt, int mt) { return ((m + 32 * mt - 1) / (32 * mt)) * ((n + 128 * nt - 1) / (128 * nt)); };
    p.nt = tiles(2, 4) >= 256 ? 2 : 1;
    p.mt = p.nt == 2 || (m + 127) / 128 * 128 * 7 <= m * 8 ? 4 : 2;
    p.mtiles = (int)((m + 32 * p.mt - 1) / (32 * p.mt));
    p.ntiles = (int)((n + 128 * p.nt - 1) / (128 * p.nt));
    const int64_t count = tiles(p.nt, p.mt);
    int64_t splits = p.nt == 2 ? 1 : (512 + count / 2) / count;
    if (splits > 8) splits = 8;
    if (splits > p.steps / 4) splits = p.steps / 4;
    if (splits < 1) splits = 1;
    p.per_split = (int)((p.steps + splits - 1) / splits);
    p.splits = (p.steps + p.per_split - 1) / p.per_split;
    p.npad = (int)((n + 15) / 16 * 16);
    if (p.nt == 1) {
        const auto rounds = [](int64_t workgroups) { return (workgroups + 255) / 256; };
        int64_t best = (p.splits > 1 ? 240 : 60) + rounds(count * p.splits) * p.per_split * (p.mt == 4 ? 22 : 15);
        for (int nt = 1; nt <= 3; ++nt) {
            const int64_t workgroups = (m + 63) / 64 * ((n + 32 * nt - 1) / (32 * nt));
            const int64_t cost = 80 + rounds(workgroups) * ((p.steps + 7) / 8) * (m <= 32 ? 13 : 20) * (1 + nt);
            if (cost < best) best = cost, p.slab = nt;
        }
    }
    p.parts_bytes = p.splits > 1 && !p.slab ? (int64_t)p.splits * m * p.npad * 4 : 0;
    return p;
}

template <bool F16, bool SF16, bool ZEROS>
hipError_t launch_cfg(const TileArgs& a, const Plan& p, hipStream_t st) {
    const dim3 grid((unsigned)(p.mtiles * p.ntiles * p.splits));
    if (p.nt == 2) hipLaunchKernelGGL((w4_tile_kernel<F16, SF16, ZEROS, 2, 4>), grid, dim3(256), 0, st, a);
    else if (p.mt == 4) hipLaunchKernelGGL((w4_tile_kernel<F16, SF16, ZEROS, 1, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((w4_tile_kernel<F16, SF16, ZEROS, 1, 2>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

template <bool F16>
hipError_t launch_type(const TileArgs& a, const Plan& p, hipStream_t st) {
    const hipError_t e = a.w.scales_f16 ? (a.w.zeros ? launch_cfg<F16, true, true>(a, p, st) : launch_cfg<F16, true, false>(a, p, st))
                                        : (a.w.zeros ? launch_cfg<F16, false, true>(a, p, st) : launch_cfg<F16, false, false>(a, p, st));
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL((w4_join_kernel<F16>), dim3((unsigned)((a.w.m * p.npad / 4 + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

// Of 256 and more tiles of 128 x 256 none is split and none goes to the slab; with fewer the other grids are small.
bool w4_tile_fits(int64_t m, int64_t n) { return (m + 127) / 128 * ((n + 255) / 256) < (int64_t(1) << 24); }

int64_t w4_tile_workspace_bytes(int64_t m, int64_t n, int64_t k) { return plan_tiles(m, n, k).parts_bytes; }

hipError_t launch_w4_tile(const W4Args& w, void* workspace, hipStream_t st) {
    const Plan p = plan_tiles(w.m, w.n, w.k);
    if (p.slab) return launch_w4_slab(w, p.slab, st);
    TileArgs a{};
    a.w = w;
    a.parts = p.splits > 1 ? (float*)workspace : nullptr;
    a.npad = p.npad;
    a.mtiles = p.mtiles;
    a.ntiles = p.ntiles;
    a.splits = p.splits;
    a.per_split = p.per_split;
    a.steps = p.steps;
    return w.f16 ? launch_type<true>(a, p, st) : launch_type<false>(a, p, st);
}

}  // namespace h3q
