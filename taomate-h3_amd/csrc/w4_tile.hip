// Product with 4-bit weights for many rows, gfx950: bound by the matrix instructions.
//
// A workgroup of four waves owns a tile of 16 TB rows x 64 JB columns, each wave all rows and 16 JB of the
// columns, so every code is unpacked once in a workgroup.  Per 128 columns of k the x tile is copied into LDS in
// operand order (double-buffered, buffer_load ... lds, no registers), the codes go straight into registers one
// block ahead, and one barrier a block closes both.  A group's product is accumulated apart from zero (rather:
// from -(16 + z) sum(x), the offset of the unpacked codes, so no subtraction follows), then added to the tile's
// sums with the group's scale: one binary32 fma for 128 (or 64, 32) multiply-adds.
//
// sum(x) of every group and row comes from a small kernel in front (x is read once more); a wave's own sums
// would cost it as many matrix instructions as one column block.
//
// Few tiles: k is split over several workgroups, whose binary32 sums a last kernel adds in order.
#include "w4.hpp"

namespace h3q {

namespace {

struct TileArgs {
    W4Args w;
    const float* sums;  // [steps * GPB][mpad]
    float* parts;       // [splits][m][npad], null: not split
    int mpad, npad, mtiles, ntiles, splits, per_split, steps;
};

template <bool F16, bool ZEROS, int GPB, int JB, int TB>
__global__ __launch_bounds__(256, 2) void w4_tile_kernel(TileArgs p) {
    constexpr int SPG = 4 / GPB;
    constexpr int XBYTES = TB * 4 * 1024, SBYTES = GPB * 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t lds_raw[2 * (XBYTES + SBYTES)];
    H3Q_LDS uint8_t* const lds = (H3Q_LDS uint8_t*)lds_raw;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;

    // Workgroups b, b + 8, ... share an XCD: each gets a contiguous run of tiles, in bands of 8 row tiles
    // with the row tile fastest.
    const int total = p.mtiles * p.ntiles * p.splits;
    int id = blockIdx.x;
    {
        const int q = total / 8, r = total % 8, x = id % 8;
        id = x * q + (x < r ? x : r) + id / 8;
    }
    const int z = id % p.splits;
    id /= p.splits;
    const int band = id / (8 * p.ntiles), in = id % (8 * p.ntiles);
    const int high = p.mtiles - band * 8 < 8 ? p.mtiles - band * 8 : 8;
    const int mt = band * 8 + in % high, nt = in / high;

    const int64_t m0 = (int64_t)mt * 16 * TB;
    const int blk0 = nt * 4 * JB + wave * JB, blocks = (int)((p.w.n + 15) / 16);
    const int nblk = blocks - blk0 < 0 ? 0 : blocks - blk0 < JB ? blocks - blk0 : JB;
    const int groups = p.w.groups, steps = p.steps;
    const int64_t rows = p.w.m - m0 < 16 * TB ? p.w.m - m0 : 16 * TB;
    const CopySrc rx(p.w.x + m0 * p.w.ldx, (uint32_t)(((rows - 1) * p.w.ldx + p.w.k) * 2));
    const CopySrc rsum(p.sums, (uint32_t)((int64_t)steps * GPB * p.mpad * 4));
    const int64_t first = nblk > 0 ? blk0 : 0;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w.codes + first * steps * 1024, (uint32_t)(nblk * steps * 1024));
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.w.scales + first * groups * 16, (uint32_t)(nblk * groups * 32));
    const __amdgpu_buffer_rsrc_t rz =
        make_rsrc(p.w.zeros + (ZEROS ? first * groups * 16 : 0), ZEROS ? (uint32_t)(nblk * groups * 16) : 0);
    const uint32_t row_bytes = (uint32_t)(p.w.ldx * 2);

    // Wave w copies the 32 columns 32 w .. + 31 of each 16-row block, and the sums of group w of the block.
    auto copy = [&](int b, int buf) __attribute__((always_inline)) {
        const uint32_t base = (uint32_t)(uintptr_t)(lds + buf * (XBYTES + SBYTES));
        const uint32_t off = 128 * b + 32 * wave + 8 * kq < p.w.k
                                 ? r16 * row_bytes + 256u * b + 64u * wave + 16u * kq : kW4Oob;
#pragma unroll
        for (int t = 0; t < TB; ++t)
            copy16(rx, base + (4 * t + wave) * 1024, off == kW4Oob ? kW4Oob : off + 16u * t * row_bytes);
        if (wave < GPB)
            copy16(rsum, base + XBYTES + wave * 1024,
                   lane < 4 * TB ? (uint32_t)(((b * GPB + wave) * p.mpad + m0) * 4 + 16 * lane) : kW4Oob);
    };
    v4u codes[JB];
    v2u scales[JB][GPB];
    uint32_t zeros[JB][GPB];
    auto load = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            codes[j] = w4_load16(rw, (uint32_t)((j * steps + b) * 1024 + 16 * lane), 0);
#pragma unroll
            for (int q = 0; q < GPB; ++q) {
                const int g = GPB == 1 ? b / p.w.blocks_per_group : b * GPB + q;
                scales[j][q] = __builtin_amdgcn_raw_buffer_load_b64(
                    rs, g < groups ? (uint32_t)((j * groups + g) * 32 + 8 * kq) : kW4Oob, 0, 0);
                zeros[j][q] = 0;
                if constexpr (ZEROS)
                    zeros[j][q] = __builtin_amdgcn_raw_buffer_load_b32(
                        rz, g < groups ? (uint32_t)((j * groups + g) * 16 + 4 * kq) : kW4Oob, 0, 0);
            }
        }
    };

    v4f acc[JB][TB];
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[j][t] = v4f{};

    const int b0 = z * p.per_split, b1 = b0 + p.per_split < steps ? b0 + p.per_split : steps;
    if (b0 < b1) {
        copy(b0, 0);
        load(b0);
    }
    for (int b = b0; b < b1; ++b) {
        const int buf = (b - b0) & 1;
        wait_vmcnt0();
        __syncthreads();  // block b is in LDS, and every wave is done with the other buffer
        v4u held[JB];
        v4f scale[JB][GPB], off[JB][GPB];
#pragma unroll
        for (int j = 0; j < JB; ++j) {
            held[j] = codes[j];
#pragma unroll
            for (int q = 0; q < GPB; ++q) {
                scale[j][q] = w4_scales(scales[j][q], p.w.scales_f16);
                off[j][q] = w4_offsets<ZEROS>(zeros[j][q]);
            }
        }
        if (b + 1 < b1) {
            copy(b + 1, buf ^ 1);
            load(b + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        const H3Q_LDS uint8_t* const tile = lds + buf * (XBYTES + SBYTES);
        const H3Q_LDS float* const sums = (const H3Q_LDS float*)(tile + XBYTES);
#pragma unroll
        for (int q = 0; q < GPB; ++q) {
            v4u w[JB][SPG];
#pragma unroll
            for (int j = 0; j < JB; ++j)
#pragma unroll
                for (int i = 0; i < SPG; ++i) w[j][i] = w4_unpack<F16>(held[j][q * SPG + i]);
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                v4u x[SPG];
#pragma unroll
                for (int i = 0; i < SPG; ++i)
                    x[i] = *(const H3Q_LDS v4u*)(tile + (4 * t + q * SPG + i) * 1024 + 16 * lane);
                const float sum = -sums[q * 256 + 16 * t + r16];
                const float plain = 24.0f * sum;
#pragma unroll
                for (int j = 0; j < JB; ++j) {
                    v4f part;
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[e] = ZEROS ? off[j][q][e] * sum : plain;
#pragma unroll
                    for (int i = 0; i < SPG; ++i) part = w4_mfma<F16>(w[j][i], x[i], part);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][t][e] = __builtin_fmaf(scale[j][q][e], part[e], acc[j][t][e]);
                }
            }
        }
    }

#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int64_t m = m0 + 16 * t + r16, n = 16 * (int64_t)(blk0 + j) + 4 * kq;
            if (p.parts) {
                if (m < p.w.m && j < nblk) *reinterpret_cast<v4f*>(p.parts + (z * p.w.m + m) * p.npad + n) = acc[j][t];
            } else {
                w4_store<F16>(p.w, m, n, acc[j][t]);
            }
        }
}

// sums[i][m] = sum of x[m, size i .. size i + size - 1] (zeros past k), size 32, 64 or 128: a wave takes 512
// columns of a row, 8 a lane.
template <bool F16>
__global__ __launch_bounds__(256) void w4_sums_kernel(W4Args p, float* sums, int mpad, int count, int lanes) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m = (int64_t)blockIdx.x * 4 + wave;
    if (m >= p.m) return;
    const int64_t k = (int64_t)blockIdx.y * 512 + 8 * lane;
    float s = 0.0f;
    if (k < p.k) {
        const uint4 v = *reinterpret_cast<const uint4*>(p.x + m * p.ldx + k);
        s = ((out_lo(v.x, F16) + out_hi(v.x, F16)) + (out_lo(v.y, F16) + out_hi(v.y, F16))) +
            ((out_lo(v.z, F16) + out_hi(v.z, F16)) + (out_lo(v.w, F16) + out_hi(v.w, F16)));
    }
    for (int off = lanes >> 1; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    const int i = (int)(k / (8 * lanes));
    if (lane % lanes == 0 && i < count) sums[(int64_t)i * mpad + m] = s;
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
    int jb, tb, splits, per_split, mtiles, ntiles, steps, mpad, npad, gpb;
    int64_t sums_bytes, parts_bytes;
};

Plan plan_tiles(int64_t m, int64_t n, int64_t k, int group) {
    Plan p{};
    p.steps = (int)((k + 127) / 128);
    p.gpb = group == 32 ? 4 : group == 64 ? 2 : 1;
    const auto tiles = [&](int jb, int tb) { return ((m + 16 * tb - 1) / (16 * tb)) * ((n + 64 * jb - 1) / (64 * jb)); };
    p.jb = 2;
    p.tb = tiles(2, 8) < 256 ? 4 : 8;
    p.mtiles = (int)((m + 16 * p.tb - 1) / (16 * p.tb));
    p.ntiles = (int)((n + 64 * p.jb - 1) / (64 * p.jb));
    const int64_t count = tiles(p.jb, p.tb);
    int64_t splits = count >= 512 ? 1 : 512 / count;
    if (splits > 8) splits = 8;
    if (splits > p.steps / 4) splits = p.steps / 4 > 0 ? p.steps / 4 : 1;
    p.per_split = (int)((p.steps + splits - 1) / splits);
    p.splits = (p.steps + p.per_split - 1) / p.per_split;
    p.mpad = p.mtiles * 16 * p.tb;
    p.npad = (int)((n + 15) / 16 * 16);
    p.sums_bytes = ((int64_t)p.steps * p.gpb * p.mpad * 4 + 255) / 256 * 256;
    p.parts_bytes = p.splits > 1 ? (int64_t)p.splits * m * p.npad * 4 : 0;
    return p;
}

template <bool F16, bool ZEROS, int GPB>
hipError_t launch_cfg(const TileArgs& a, const Plan& p, hipStream_t st) {
    const dim3 grid((unsigned)(p.mtiles * p.ntiles * p.splits));
    if (p.tb == 8) hipLaunchKernelGGL((w4_tile_kernel<F16, ZEROS, GPB, 2, 8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((w4_tile_kernel<F16, ZEROS, GPB, 2, 4>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

template <bool F16>
hipError_t launch_type(const TileArgs& a, const Plan& p, hipStream_t st) {
    const W4Args& w = a.w;
    hipLaunchKernelGGL((w4_sums_kernel<F16>), dim3((unsigned)((w.m + 3) / 4), (unsigned)((p.steps * 128 + 511) / 512)),
                       dim3(256), 0, st, w, const_cast<float*>(a.sums), p.mpad, p.steps * p.gpb, 16 / p.gpb);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (w.zeros)
        e = p.gpb == 4 ? launch_cfg<F16, true, 4>(a, p, st) : p.gpb == 2 ? launch_cfg<F16, true, 2>(a, p, st)
                                                                         : launch_cfg<F16, true, 1>(a, p, st);
    else
        e = p.gpb == 4 ? launch_cfg<F16, false, 4>(a, p, st) : p.gpb == 2 ? launch_cfg<F16, false, 2>(a, p, st)
                                                                          : launch_cfg<F16, false, 1>(a, p, st);
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL((w4_join_kernel<F16>), dim3((unsigned)((w.m * p.npad / 4 + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

bool w4_tile_fits(int64_t m, int64_t n, int64_t k, int group) {
    const int64_t rows = (m + 127) / 128 * 128, steps = (k + 127) / 128;
    return rows * steps * (group == 32 ? 4 : group == 64 ? 2 : 1) * 4 < (int64_t(1) << 31) &&
           rows / 64 * ((n + 127) / 128) * 8 < (int64_t(1) << 31) && rows * ((n + 15) / 16) / 64 < (int64_t(1) << 31);
}

int64_t w4_tile_workspace_bytes(int64_t m, int64_t n, int64_t k, int group) {
    const Plan p = plan_tiles(m, n, k, group);
    return p.sums_bytes + p.parts_bytes;
}

hipError_t launch_w4_tile(const W4Args& w, void* workspace, hipStream_t st) {
    const Plan p = plan_tiles(w.m, w.n, w.k, w.group);
    TileArgs a{};
    a.w = w;
    a.sums = (const float*)workspace;
    a.parts = p.splits > 1 ? (float*)((uint8_t*)workspace + p.sums_bytes) : nullptr;
    a.mpad = p.mpad;
    a.npad = p.npad;
    a.mtiles = p.mtiles;
    a.ntiles = p.ntiles;
    a.splits = p.splits;
    a.per_split = p.per_split;
    a.steps = p.steps;
    return w.f16 ? launch_type<true>(a, p, st) : launch_type<false>(a, p, st);
}

}  // namespace h3q
