// Scaled product of rows grouped by expert over 256 x 256 tiles, gfx950: the four-wave
// kernel of the dense GEMM (gemm_w4.hip: four waves of 128 x 128, 64-byte k-steps through
// a ring of four 32 KiB LDS stages filled by LDS-DMA, accumulators in AGPRs) on tiles that
// the device finds itself.
//
//   y[i, n] = s_a[r] * (s_w[e, n] * sum_k A[r, k] * W[e, n, k]),  r = order[i] / top_k or i
//
// Tiles.  An expert's rows are cut into blocks of 256; a block of at most 128 rows (the
// last of an expert's, as a rule) runs as a half tile with half the matrix instructions.
// Each workgroup sums the experts' block counts into LDS when it starts, and takes tiles
// blockIdx.x, + gridDim.x, ... of the blocks x column tiles, so a batch that leaves
// experts empty costs no workgroup.
//
// Gather.  The rows' indices of a tile are copied to LDS while the previous tile runs;
// each lane then adds its row's offset to its copies of A, which makes the gather free
// (16 lanes' chunks of 4 rows a copy either way).  The row scales are gathered by the same
// copies, 4 bytes a lane.
//
// SwiGLU.  The 256 weight rows of a tile are the gate and up rows of 128 columns, placed
// so that a wave's 128 columns are 64 gate columns and the same 64 up columns: accumulator
// blocks j and j + 2 of a lane then hold gate and up of the same element, and the epilogue
// stays in registers.
//
// What bounds it: as the dense kernel, the matrix instructions at their power-limited clock
// (int8 16384 rows over 8 experts of 14336 x 5376 with SwiGLU and gathered rows: 1126 to 1168 us
// over eight runs on four cards, 2.16 to 2.24 POP/s; the dense kernel's 2.31), and with a short k the
// epilogue, which no other wave hides (e4m3 32768 rows over 64 experts of 2816 x 2048: 215 to 224
// us, 1.68 to 1.75 PFLOP/s).
#include <type_traits>

#include "gemm_tiles.hpp"
#include "grouped_gemm.hpp"

namespace h3q {

namespace {

constexpr int kStages = 4;
constexpr int kStageBytes = (256 + 256) * 64;  // A and B, 64 bytes of k each
constexpr int kABytes = 256 * 64;
constexpr int kVecBytes = 3 * 256 * 4;  // a tile's row scales, column scales and pairs, 4 bytes each
constexpr int64_t kStreamOutBytes = int64_t(64) << 20;  // outputs stored past the caches (see gemm_w4.hip)

// Wave copies global -> LDS (see copy16 in h3q_common.hpp), with a scalar offset.  A scalar
// that a vector instruction wrote (readfirstlane, or a spilled one read back) may be read
// by a memory instruction five wait states later at the earliest; the compiler does not see
// the load inside the text, so the text waits for itself.
__device__ __forceinline__ void copy16_soff(const CopySrc& src, uint32_t lds_base, uint32_t voff, uint32_t soff) {
    const v4i d = {__builtin_amdgcn_readfirstlane(src.d[0]), __builtin_amdgcn_readfirstlane(src.d[1]),
                   __builtin_amdgcn_readfirstlane(src.d[2]), __builtin_amdgcn_readfirstlane(src.d[3])};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(voff), "s"(d),
                   "s"(__builtin_amdgcn_readfirstlane(soff))
                 : "memory");
}

// Lane L's 4 bytes at src + voff land at LDS byte lds_base + 4 L.
__device__ __forceinline__ void copy4(const CopySrc& src, uint32_t lds_base, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(voff), "s"(src.d)
                 : "memory");
}

__device__ __forceinline__ void mfma_e4m3(v16f& c, const v8i& b, const v8i& a) {
    asm volatile("v_mfma_f32_32x32x64_f8f6f4 %0, %1, %2, %0" : "+a"(c) : "v"(b), "v"(a));
}
__device__ __forceinline__ void mfma_e4m3_first(v16f& c, const v8i& b, const v8i& a) {
    asm volatile("v_mfma_f32_32x32x64_f8f6f4 %0, %1, %2, 0" : "=a"(c) : "v"(b), "v"(a));
}
__device__ __forceinline__ void mfma_i8(v16i& c, const v4i& b, const v4i& a) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %1, %2, %0" : "+a"(c) : "v"(b), "v"(a));
}
__device__ __forceinline__ void mfma_i8_first(v16i& c, const v4i& b, const v4i& a) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %1, %2, 0" : "=a"(c) : "v"(b), "v"(a));
}
__device__ __forceinline__ float agpr_read(float x) {
    float v;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(x));
    return v;
}
__device__ __forceinline__ float agpr_read(int x) {
    int v;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(x));
    return (float)v;
}

// Chunk swizzle of a 64-byte row-major stage row (see gemm_w4.hip).
__device__ __forceinline__ int swz64(int r) { return (((r >> 1) ^ (r >> 3)) & 1) | ((r >> 1) & 2); }

template <int OP>
struct TileOp;
template <>
struct TileOp<kOpE4M3> {
    using acc_t = v16f;
    using frag_t = v8i;
    static constexpr int kSteps = 1;  // matrix-instruction k-steps per 64-byte stage
};
template <>
struct TileOp<kOpInt8> {
    using acc_t = v16i;
    using frag_t = v4i;
    static constexpr int kSteps = 2;
};

}  // namespace

template <int OP, bool TB, int OUT>
__global__ __launch_bounds__(256, 1) void grouped_tile_kernel(GroupedArgs p, int tiles_n, int stream_out) {
    using acc_t = typename TileOp<OP>::acc_t;
    using frag_t = typename TileOp<OP>::frag_t;
    constexpr int KS = TileOp<OP>::kSteps;
    constexpr bool SWIGLU = OUT == kOutSwiglu;
    __shared__ __attribute__((aligned(1024))) uint8_t lds_ring[kStages * kStageBytes];
    // Per tile parity: row scales [256] f32 | column scales [256] f32 | order [256] i32.
    __shared__ __attribute__((aligned(1024))) uint8_t lds_vec[2 * kVecBytes];
    __shared__ uint32_t lds_live[2][8];  // a bit for each row of the tile that has a row of a
    __shared__ int lds_first[kMaxExperts];  // row blocks of the experts below, and each one's rows
    __shared__ int lds_lo[kMaxExperts], lds_hi[kMaxExperts];
    H3Q_LDS uint8_t* const ring = (H3Q_LDS uint8_t*)lds_ring;
    H3Q_LDS uint8_t* const vec = (H3Q_LDS uint8_t*)lds_vec;
    const uint32_t ring_addr = (uint32_t)(uintptr_t)ring;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn0 = (wave & 1) * 128;
    const int g = lane >> 5, c32 = lane & 31;
    const int kbytes = (int)p.k;
    const int ksteps = (kbytes + 127) / 128 * 2;  // even; the bytes past k read as zero
    const int64_t steps128 = p.k / 128;           // tiled weights
    const bool gather = p.order != nullptr;
    const int half_n = p.n / 2;

    // Row blocks before each expert, 64 experts at a time (every wave for itself; wave 0
    // keeps them).  The bounds come from device memory: clamped to the rows of the call.
    int total_blocks = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
        const int e = e0 + lane;
        int64_t lo = 0, hi = 0;
        if (e < p.experts) {
            lo = p.offsets[e];
            hi = p.offsets[e + 1];
            lo = lo < 0 ? 0 : (lo > p.rows ? p.rows : lo);
            hi = hi < lo ? lo : (hi > p.rows ? p.rows : hi);
        }
        const int own = (int)((hi - lo + 255) / 256);
        int sum = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d, 64);
            if (lane >= d) sum += o;
        }
        if (wave == 0 && e < p.experts) {
            lds_first[e] = total_blocks + sum - own;
            lds_lo[e] = (int)lo;
            lds_hi[e] = (int)hi;
        }
        total_blocks += __builtin_amdgcn_readlane(sum, 63);
    }
    const int64_t all_tiles = (int64_t)total_blocks * tiles_n;
    const int T = (int)(all_tiles < 0x7FFFFFFF ? all_tiles : 0x7FFFFFFF), G = (int)gridDim.x, b = (int)blockIdx.x;
    const int ntiles = b < T ? (T - b + G - 1) / G : 0;
    if (ntiles == 0) return;
    __syncthreads();

    // Tile j of this workgroup.  Each XCD gets a contiguous run of the tiles (tile_coords of
    // gemm_tiles.hpp); inside an expert they go column by column over groups of 8 row blocks.
    struct Tile {
        int expert, rows, cols, n0;  // cols: weight rows (SwiGLU: output columns) left from n0
        int64_t row0;
    };
    auto find_tile = [&](int j) __attribute__((always_inline)) -> Tile {
        constexpr int kXcds = 8, kGroupM = 8;
        const int bid = b + j * G, q = T / kXcds, rem = T % kXcds, xcd = bid % kXcds, local = bid / kXcds;
        const int t = xcd < rem ? xcd * (q + 1) + local : rem * (q + 1) + (xcd - rem) * q + local;
        const int block = t / tiles_n;  // some block of the same expert
        int n = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 64) {
            const int e = e0 + lane;
            n += __popcll(__ballot(e < p.experts && lds_first[e < p.experts ? e : 0] <= block));
        }
        // the last expert that starts at or before the block: empty ones before it start there too
        Tile r;
        r.expert = __builtin_amdgcn_readfirstlane(n - 1);
        const int first = lds_first[r.expert];
        const int lo = lds_lo[r.expert], own = lds_hi[r.expert] - lo;
        const int blocks = (own + 255) / 256;
        const int rest = t - first * tiles_n;
        const int group = rest / (kGroupM * tiles_n), first_m = group * kGroupM;
        const int gsize = blocks - first_m < kGroupM ? blocks - first_m : kGroupM;
        const int in_group = rest - group * kGroupM * tiles_n;
        const int tm = first_m + in_group % gsize, tn = in_group / gsize;
        const int left = own - tm * 256;
        r.row0 = __builtin_amdgcn_readfirstlane(lo + tm * 256);
        r.rows = __builtin_amdgcn_readfirstlane(left < 256 ? left : 256);
        r.n0 = __builtin_amdgcn_readfirstlane(tn * (SWIGLU ? 128 : 256));
        r.cols = (SWIGLU ? half_n : p.n) - r.n0;
        return r;
    };

    // ---------------------------------------------------------------- copies
    CopySrc ra(nullptr, 0), rb(nullptr, 0);
    uint32_t voff_a[4], voff_b[4];
    int chunk16 = 0;  // byte of the lane's 16-byte chunk in a row-major 64-byte step
    Tile cp;          // the tile being copied
    int cj = 0, cs = 0;
    // order[] of tile t (parity par) into LDS, by wave 3.
    auto issue_order = [&](const Tile& t, int par) __attribute__((always_inline)) {
        if (gather && wave == 3)
            copy16_soff(CopySrc(p.order + t.row0, (uint32_t)t.rows * 4u),
                        (uint32_t)(uintptr_t)(vec + par * kVecBytes + 2048), 16u * lane, 0);
    };
    // Row of a behind row i of the copy tile, or -1.
    auto source_row = [&](int i) __attribute__((always_inline)) -> int64_t {
        if (i >= cp.rows) return -1;
        if (!gather) return cp.row0 + i;
        const int pair = ((const H3Q_LDS int*)(vec + (cj & 1) * kVecBytes + 2048))[i];
        const int r = pair / p.top_k;
        return pair >= 0 && r < p.a_rows ? r : -1;
    };
    auto setup_copy_tile = [&](Tile t) __attribute__((always_inline)) {
        cp = t;
        const bool live = cj < ntiles;
        ra = gather ? CopySrc(p.a, live ? (uint32_t)(p.a_rows * p.lda) : 0u)
                    : CopySrc((const uint8_t*)p.a + cp.row0 * p.lda, live ? (uint32_t)(cp.rows * p.lda) : 0u);
        const int64_t w_bytes = (int64_t)p.n * p.k;
        rb = CopySrc((const uint8_t*)p.b + cp.expert * w_bytes, live ? (uint32_t)w_bytes : 0u);
        const int ln = opaque_lane();
        const int sub = ln >> 2;
        chunk16 = 16 * ((ln & 3) ^ swz64(sub));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = wave + 4 * i;  // 16 rows x 64 bytes per copy
            const int64_t r = source_row(c * 16 + sub);
            voff_a[i] = r >= 0 ? (uint32_t)((gather ? r : r - cp.row0) * p.lda) + (uint32_t)chunk16 : kOob;
            int row = c * 16;  // first weight row of block c, and whether it exists
            bool in = row < cp.cols;
            if constexpr (SWIGLU) {
                const int f = (c >> 3) * 64 + (c & 3) * 16;  // gate of columns f .., or up
                in = f < cp.cols;
                row = f + ((c & 4) ? half_n : 0);
            }
            row += cp.n0;
            if constexpr (TB)
                voff_b[i] = in ? (uint32_t)(row / 16 * steps128 * 2048) + (uint32_t)((ln >> 5) * 1024 + (ln & 31) * 16) : kOob;
            else
                voff_b[i] = in ? (uint32_t)((row + sub) * kbytes) + (uint32_t)chunk16 : kOob;
        }
        if (!live) return;
        // Epilogue vectors of the tile: its row scales (a row per lane of the four waves) and
        // column scales, and the next tile's order.
        H3Q_LDS uint8_t* const v = vec + (cj & 1) * kVecBytes;
        const int64_t r = source_row(threadIdx.x);
        const uint64_t rows_live = __ballot(r >= 0);
        if (lane < 2) lds_live[cj & 1][2 * wave + lane] = (uint32_t)(rows_live >> (32 * lane));
        copy4(gather ? CopySrc(p.a_scale, (uint32_t)(p.a_rows * 4)) : CopySrc(p.a_scale + cp.row0, (uint32_t)cp.rows * 4u),
              (uint32_t)(uintptr_t)(v + wave * 256), r >= 0 ? (uint32_t)((gather ? r : r - cp.row0) * 4) : kOob);
        const float* const sw = p.b_scale + (int64_t)cp.expert * p.n;
        if constexpr (SWIGLU) {
            if (wave < 2) {  // gate (up) scales of the tile's 128 columns
                if (lane < 32)  // the other lanes' zeros would land in the next 512 bytes
                    copy16_soff(CopySrc(sw + wave * half_n + cp.n0, (uint32_t)(cp.cols < 128 ? cp.cols : 128) * 4u),
                                (uint32_t)(uintptr_t)(v + 1024 + wave * 512), 16u * lane, 0);
            }
        } else {
            if (wave == 1)
                copy16_soff(CopySrc(sw + cp.n0, (uint32_t)(cp.cols < 256 ? cp.cols : 256) * 4u),
                            (uint32_t)(uintptr_t)(v + 1024), 16u * lane, 0);
        }
    };
    Tile nxt;  // tile cj + 1, its order on the way
    auto issue_copy = [&](int q, int st) __attribute__((always_inline)) {
        const uint32_t base = ring_addr + (uint32_t)(st * kStageBytes);
        const uint32_t soff_t = (uint32_t)((cs >> 1) * 2048 + (cs & 1) * 512), soff_r = (uint32_t)(cs * 64);
        const bool in = chunk16 < kbytes - cs * 64;  // the lane's chunk lies before k
        if (q < 4)
            copy16_soff(ra, base + (uint32_t)((wave + 4 * q) * 1024), in ? voff_a[q] : kOob, soff_r);
        else if constexpr (TB)
            copy16_soff(rb, base + (uint32_t)(kABytes + (wave + 4 * (q - 4)) * 1024), voff_b[q - 4], soff_t);
        else
            copy16_soff(rb, base + (uint32_t)(kABytes + (wave + 4 * (q - 4)) * 1024), in ? voff_b[q - 4] : kOob, soff_r);
    };
    auto advance_copy = [&]() __attribute__((always_inline)) {
        if (++cs == ksteps) {
            cs = 0;
            ++cj;
            setup_copy_tile(nxt);
            if (cj + 1 < ntiles) {
                nxt = find_tile(cj + 1);
                issue_order(nxt, (cj + 1) & 1);
            }
        }
    };

    // ------------------------------------------------------ fragment reads
    uint32_t rda[2], rda_full[2], rda_half[2], rdb[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int chunk = OP == kOpE4M3 ? 2 * g + h : 2 * h + g;  // logical 16-byte chunk of the row
        const int tiled_off = ((c32 & 15) + 16 * (OP == kOpE4M3 ? g : h)) * 16 + (OP == kOpE4M3 ? h : g) * 512;
        const uint32_t in_row = (uint32_t)((chunk ^ swz64(c32)) << 4);
        rda_full[h] = (uint32_t)(((wave >> 1) * 128 + c32) * 64) + in_row;
        rda_half[h] = (uint32_t)(((wave >> 1) * 64 + c32) * 64) + in_row;
        rdb[h] = kABytes + (TB ? (uint32_t)(((wn0 + c32) >> 4) * 1024 + tiled_off) : (uint32_t)((wn0 + c32) * 64) + in_row);
    }
    auto set_layout = [&](bool half) __attribute__((always_inline)) {
        rda[0] = half ? rda_half[0] : rda_full[0];
        rda[1] = half ? rda_half[1] : rda_full[1];
    };
    struct Frags {
        frag_t a[4 * KS], b[4 * KS];
    };
    auto ld16 = [&](const H3Q_LDS uint8_t* ptr) __attribute__((always_inline)) -> v4i { return *(const H3Q_LDS v4i*)ptr; };
    // Fragment x of stage st: x < 4 KS is A block x % 4 (k-step x / 4), the rest B.
    auto read_frag = [&](Frags& F, int x, int st) __attribute__((always_inline)) {
        const H3Q_LDS uint8_t* sb = ring + st * kStageBytes;
        const bool is_a = x < 4 * KS;
        const int xx = is_a ? x : x - 4 * KS;
        const int y = xx % 4, s = xx / 4;
        if constexpr (OP == kOpE4M3) {
            const uint32_t* off = is_a ? rda : rdb;
            const v8i f = __builtin_shufflevector(ld16(sb + off[0] + y * 2048), ld16(sb + off[1] + y * 2048), 0, 1, 2,
                                                  3, 4, 5, 6, 7);
            if (is_a) F.a[y] = f;
            else F.b[y] = f;
        } else {
            const v4i f = ld16(sb + (is_a ? rda[s] : rdb[s]) + y * 2048);
            if (is_a) F.a[y + 4 * s] = f;
            else F.b[y + 4 * s] = f;
        }
    };

    acc_t acc[4][4];
    Frags F0, F1;
    auto mfma = [&](auto mi, bool first, const Frags& Fc, int t) __attribute__((always_inline)) {
        constexpr int MI = decltype(mi)::value;
        const int s = t / (4 * MI), i = (t % (4 * MI)) / 4, j = t % 4;
        if constexpr (OP == kOpE4M3) {
            if (first) mfma_e4m3_first(acc[i][j], Fc.b[j], Fc.a[i]);
            else mfma_e4m3(acc[i][j], Fc.b[j], Fc.a[i]);
        } else {
            if (first && s == 0) mfma_i8_first(acc[i][j], Fc.b[j + 4 * s], Fc.a[i + 4 * s]);
            else mfma_i8(acc[i][j], Fc.b[j + 4 * s], Fc.a[i + 4 * s]);
        }
    };
    // One step: matrix instructions on Fc, the next stage's fragments into Fn, the copies of
    // four steps on; every slot kept in place by a scheduling barrier.
    auto body = [&](auto mi, bool first, const Frags& Fc, Frags& Fn, int rst, int cst) __attribute__((always_inline)) {
        constexpr int MI = decltype(mi)::value;
        constexpr int NM = 4 * MI * KS, NR = 8 * KS;
        constexpr int NT = NM > NR + 8 ? NM : NR + 8;
        constexpr int CP = NT / 8;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (t < NM) mfma(mi, first, Fc, t);
            if (t < NR) read_frag(Fn, t, rst);
            if (t % CP == CP - 1 && t / CP < 8) issue_copy(t / CP, cst);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // ------------------------------------------------------------- epilogue
    // Accumulator slot 4 q + x of block (i, jj): row 32 i + c32, column 32 jj + 8 q + 4 g + x of
    // the wave's.  Rows of up to 256 bytes are staged in LDS (the stage that the next
    // step's copies fill is free until then), 16-byte chunk c of row r at c ^ (r % 16).
    auto epilogue = [&](auto mi, const Tile& cur, int par, int st) __attribute__((always_inline)) {
        constexpr int MI = decltype(mi)::value;
        const int wm0 = (wave >> 1) * 32 * MI;
        const int ln = opaque_lane();
        const int gg = ln >> 5, cc = ln & 31;
        const H3Q_LDS uint8_t* e = vec + par * kVecBytes;
        H3Q_LDS uint8_t* const scratch = ring + st * kStageBytes + wave * 8192;
        constexpr int EL = OUT == kOutF32 ? 4 : 2;
        const __amdgpu_buffer_rsrc_t ro =
            make_rsrc((uint8_t*)p.out + cur.row0 * p.ldo * EL, (uint32_t)((int64_t)cur.rows * p.ldo * EL));
        float sa[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) sa[i] = ((const H3Q_LDS float*)e)[wm0 + 32 * i + cc];
        // VALU reads of matrix results: wait out the last instructions' passes.
        asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
        auto scaled = [&](int i, int jj, int q, const v4f& sw, int x) __attribute__((always_inline)) -> float {
            return __fmul_rn(sa[i], __fmul_rn(sw[x], agpr_read(acc[i][jj][4 * q + x])));
        };
        auto store = [&](const v4u& v, uint32_t off) __attribute__((always_inline)) {
            if (stream_out) __builtin_amdgcn_raw_buffer_store_b128(v, ro, off, 0, 2);
            else __builtin_amdgcn_raw_buffer_store_b128(v, ro, off, 0, 0);
        };
        // The wave's rows of a staged pass: `chunks` 16-byte chunks a row from byte column col0 of out.
        // A row without a row of a keeps what out held, as those past the tile do.
        auto flush = [&](int i, int chunks, int pitch, int col0, int limit) __attribute__((always_inline)) {
            const uint32_t live = lds_live[par][(wm0 >> 5) + i];
            const int per = 64 / chunks;  // rows a store covers
#pragma unroll
            for (int r = 0; r < 32 / per; ++r) {
                const int row = per * r + ln / chunks, c = ln % chunks;
                const v4u v = *(const H3Q_LDS v4u*)(scratch + row * pitch + ((c ^ (row & (chunks - 1))) << 4));
                const int m = wm0 + 32 * i + row;
                store(v, 16 * c < limit && (live >> row & 1) ? (uint32_t)m * (uint32_t)p.ldo * EL + (uint32_t)(col0 + 16 * c)
                                                        : 0xFFFFFFF0u);
            }
        };
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            if constexpr (SWIGLU) {
                const int f0 = (wave & 1) * 64;
#pragma unroll
                for (int g8 = 0; g8 < 8; ++g8) {
                    const int jj = g8 >> 2, q = g8 & 3;
                    const int col = f0 + 32 * jj + 8 * q + 4 * gg;
                    const v4f swg = *(const H3Q_LDS v4f*)(e + 1024 + 4 * col), swu = *(const H3Q_LDS v4f*)(e + 1536 + 4 * col);
                    float y[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) y[x] = swiglu_f32(scaled(i, jj, q, swg, x), scaled(i, jj + 2, q, swu, x));
                    *(H3Q_LDS v2u*)(scratch + cc * 128 + ((g8 ^ (cc & 7)) << 4) + gg * 8) =
                        v2u{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
                }
                flush(i, 8, 128, (cur.n0 + f0) * 2, (cur.cols - f0) * 2);
            } else if constexpr (OUT == kOutBF16) {
#pragma unroll
                for (int g16 = 0; g16 < 16; ++g16) {
                    const int jj = g16 >> 2, q = g16 & 3;
                    const v4f sw = *(const H3Q_LDS v4f*)(e + 1024 + 4 * (wn0 + 8 * g16 + 4 * gg));
                    float y[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) y[x] = scaled(i, jj, q, sw, x);
                    *(H3Q_LDS v2u*)(scratch + cc * 256 + ((g16 ^ (cc & 15)) << 4) + gg * 8) =
                        v2u{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
                }
                flush(i, 16, 256, (cur.n0 + wn0) * 2, (cur.cols - wn0) * 2);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // 64 columns of 4 bytes at a time
#pragma unroll
                    for (int g8 = 0; g8 < 8; ++g8) {
                        const int jj = 2 * h + (g8 >> 2), q = g8 & 3;
                        const v4f sw = *(const H3Q_LDS v4f*)(e + 1024 + 4 * (wn0 + 32 * jj + 8 * q + 4 * gg));
                        v4f y;
#pragma unroll
                        for (int x = 0; x < 4; ++x) y[x] = scaled(i, jj, q, sw, x);
                        *(H3Q_LDS v4f*)(scratch + cc * 256 + (((2 * g8 + gg) ^ (cc & 15)) << 4)) = y;
                    }
                    flush(i, 16, 256, (cur.n0 + wn0 + 64 * h) * 4, (cur.cols - wn0 - 64 * h) * 4);
                }
            }
        }
    };

    // ------------------------------------------------------------ main loop
    // The first tile's order has to be there before its copies are set up.
    {
        const Tile t0 = find_tile(0);
        issue_order(t0, 0);
        wait_vmcnt<0>();
        ring_barrier();
        setup_copy_tile(t0);
        nxt = t0;
        if (ntiles > 1) {
            nxt = find_tile(1);
            issue_order(nxt, 1);
        }
    }
    set_layout(cp.rows <= 128);
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
#pragma unroll
        for (int q = 0; q < 8; ++q) issue_copy(q, st);
        ++cs;  // ksteps > 4: the first tile's groups
    }
    wait_vmcnt<(kStages - 1) * 8>();
    ring_barrier();
#pragma unroll
    for (int x = 0; x < 8 * KS; ++x) read_frag(F0, x, 0);
    wait_vmcnt<(kStages - 2) * 8>();
    ring_barrier();

    int cur_st = 0;  // stage of the running step (its fragments are in registers)
    auto step = [&](auto mi, bool first, const Frags& Fc, Frags& Fn) __attribute__((always_inline)) {
        const int nxt_st = cur_st + 1 == kStages ? 0 : cur_st + 1;
        body(mi, first, Fc, Fn, nxt_st, cur_st);
        advance_copy();
        wait_vmcnt<(kStages - 2) * 8>();
        ring_barrier();
        cur_st = nxt_st;
    };
    auto run_tile = [&](auto mi, const Tile& cur, int mj) __attribute__((always_inline)) {
        const std::integral_constant<int, decltype(mi)::value> m;
        step(m, true, F0, F1);
        step(m, false, F1, F0);
        for (int s = 2; s < ksteps; s += 2) {
            step(m, false, F0, F1);
            // The last step reads the next tile's first fragments (cp is that tile by now).
            if (s + 2 == ksteps) set_layout(cp.rows <= 128);
            step(m, false, F1, F0);
        }
        epilogue(m, cur, mj & 1, cur_st);
        ring_barrier();
    };
    for (int mj = 0; mj < ntiles; ++mj) {
        const Tile cur = cp;  // the copies are still at this tile: ksteps > 4
        if (cur.rows <= 128) run_tile(std::integral_constant<int, 2>(), cur, mj);
        else run_tile(std::integral_constant<int, 4>(), cur, mj);
    }
    wait_vmcnt<0>();
}

namespace {

int64_t grouped_tiles(const GroupedArgs& a, int* tiles_n) {
    *tiles_n = a.swiglu ? (a.n / 2 + 127) / 128 : (a.n + 255) / 256;
    return (a.experts + a.rows / 256) * (int64_t)*tiles_n;
}

template <int OP, bool TB>
hipError_t launch_tile_tb(const GroupedArgs& a, hipStream_t st) {
    int tiles_n;
    const int64_t tiles = grouped_tiles(a, &tiles_n);  // at most
    const dim3 grid((unsigned)persistent_grid((int)tiles));
    const int cols = a.swiglu ? a.n / 2 : a.n;
    const int stream_out = a.rows * cols * (a.f32 ? 4 : 2) >= kStreamOutBytes;
    if (a.swiglu)
        hipLaunchKernelGGL((grouped_tile_kernel<OP, TB, kOutSwiglu>), grid, dim3(256), 0, st, a, tiles_n, stream_out);
    else if (a.f32)
        hipLaunchKernelGGL((grouped_tile_kernel<OP, TB, kOutF32>), grid, dim3(256), 0, st, a, tiles_n, stream_out);
    else
        hipLaunchKernelGGL((grouped_tile_kernel<OP, TB, kOutBF16>), grid, dim3(256), 0, st, a, tiles_n, stream_out);
    return hipGetLastError();
}

}  // namespace

bool grouped_tile_supported(const GroupedArgs& a) {
    // More than four 64-byte steps a tile (a tile's first four are copied under the one before),
    // tile-relative 32-bit offsets, and a tile count that an int holds.
    int tiles_n;
    return a.k > 256 && 256 * a.ldo * (a.f32 ? 4 : 2) < (int64_t(1) << 31) &&
           grouped_tiles(a, &tiles_n) < (int64_t(1) << 31);
}

hipError_t launch_grouped_tile(int kind, const GroupedArgs& a, hipStream_t st) {
    if (kind == kOpInt8) return a.b_tiled ? launch_tile_tb<kOpInt8, true>(a, st) : launch_tile_tb<kOpInt8, false>(a, st);
    return a.b_tiled ? launch_tile_tb<kOpE4M3, true>(a, st) : launch_tile_tb<kOpE4M3, false>(a, st);
}

}  // namespace h3q
