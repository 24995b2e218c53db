// Scaled product of rows grouped by expert, a band of rows per workgroup, gfx950: for
// groups of a few dozen to a few hundred rows (see grouped_stream.hip for the definition).
//
// What bounds it.  An expert's weights still come from HBM once and its rows are few enough
// that the matrix instructions take a third of that time, but every 16 columns need the same
// rows: with one wave per weight block (grouped_stream.hip) 64 rows cost twice the weights'
// bytes again through the L2.  Here a workgroup of four waves owns up to 16 MT rows of one
// expert and 128 weight rows; a wave streams its own 32 weight rows straight into registers,
// D k-steps of 128 bytes ahead, and the activation rows of a step come once into an LDS ring
// that the four waves share (LDS-DMA, gathered rows as cheaply as dense ones).  One barrier a
// step publishes the next stage and frees the last.  No split of K: the experts give
// workgroups enough.  Items (band x column slice) go to the XCDs in contiguous runs, an
// expert's bands of one slice side by side, so weights and rows pass through one L2 about
// once: spread over the XCDs, two bands an expert missed the L2s for 525 MB where 197 MB were
// needed, and that was the bound (32 experts of 2816 x 2048 with 200 rows each, int8: 84 -> 70 to
// 72 us; 8 of 14336 x 5376: 197 -> 185 to 192 us).  In runs the first misses for 227 MB (3.2 TB/s),
// with the matrix instructions busy 28% of the time: neither binds it now.
//
// SwiGLU: a wave's two 16-row blocks are gate and up rows of the same columns, so both sit in
// one lane.  The output tile is staged in LDS and stored as whole row pieces.
#include <type_traits>

#include "gemm_tiles.hpp"
#include "grouped_gemm.hpp"

namespace h3q {

namespace {

constexpr int kBandWaves = 4;

// See copy16_soff in grouped_tile.hip for the wait inside.
__device__ __forceinline__ void band_copy(const CopySrc& src, uint32_t lds_base, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(voff), "s"(src.d)
                 : "memory");
}

}  // namespace

template <int OP, int MT, bool TB, int OUT>
__global__ __launch_bounds__(kBandWaves * 64, MT == 8 || OUT == kOutWide ? 2 : 3) void grouped_band_kernel(GroupedArgs p, int slices) {
    constexpr bool SWIGLU = OUT == kOutSwiglu || OUT == kOutWide;
    using Mfma = GroupedMfma<OP, OUT == kOutWide>;
    using acc_t = typename Mfma::acc_t;
    // Loads complete in order, so the wait for a stage of rows also waits for the weights asked
    // for before it: the ring is as deep as the weights run ahead, and as two or three
    // workgroups a CU (64 rows) have LDS for.
    constexpr int BM = 16 * MT, SA = MT == 8 ? 5 : 6, D = 4;
    constexpr int STAGE = MT * 2048;   // one k-step of the rows
    constexpr int CA = MT / 2;         // 1 KiB copies per wave and step
    // Loads a wave has issued after the copies of stage s + 1 when it waits for them in step s:
    // the weights of that step and all of the SA - 3 steps since.
    constexpr int WAIT = 4 + (SA - 3) * (CA + 4);
    constexpr int WAIT_TAIL = (SA - 3) * CA;  // the last steps ask for no more weights
    static_assert((MT == 4 || MT == 8) && D * 4 + SA * CA < 63, "vmcnt range");
    __shared__ __attribute__((aligned(1024))) uint8_t lds_ring[SA * STAGE];
    __shared__ __attribute__((aligned(16))) float lds_scales[MT == 8 ? 4 : BM + 128 + BM / 32];
    H3Q_LDS uint8_t* const ring = (H3Q_LDS uint8_t*)lds_ring;
    // Row scales [BM], the column scales of the waves' blocks, a bit for each row of the band that
    // has a row of a (the others keep what out held); 128-row bands have no LDS
    // beside the ring (two workgroups share a CU's) and take its end, past the output tile.
    H3Q_LDS float* const lds_sa = MT == 8 ? (H3Q_LDS float*)(ring + BM * 512) : (H3Q_LDS float*)lds_scales;
    H3Q_LDS float* const lds_sw = lds_sa + BM;
    H3Q_LDS uint32_t* const lds_live = (H3Q_LDS uint32_t*)(lds_sw + 128);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    GroupTile tile;
    int slice;
    if (!group_item(p.offsets, p.experts, p.rows, BM, slices, blockIdx.x, tile, slice)) return;
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert);
    const int rows = __builtin_amdgcn_readfirstlane(tile.rows);
    const int half = p.n / 2;
    const int kbytes = (int)p.k;
    const int steps = (kbytes + 127) >> 7;

    // First weight row of this wave's block j (p.n: none).
    auto block_row = [&](int j) __attribute__((always_inline)) -> int {
        if constexpr (SWIGLU) {
            const int f = 64 * slice + 16 * wave;
            return f < half ? j * half + f : p.n;
        }
        const int r = 128 * slice + 32 * wave + 16 * j;
        return r < p.n ? r : p.n;
    };
    const int64_t w_bytes = (int64_t)p.n * p.k;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc((const uint8_t*)p.b + expert * w_bytes, (uint32_t)w_bytes);
    uint32_t woff[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = block_row(j);
        if constexpr (TB) woff[j] = row < p.n ? (uint32_t)((int64_t)(row / 16) * steps * 2048 + 16 * lane) : kOob;
        else woff[j] = row < p.n ? (uint32_t)((int64_t)(row + r16) * p.k + 32 * kq) : kOob;
    }
    auto load_w = [&](int st, v8i (&w)[2]) __attribute__((always_inline)) {
        // Past K: an offset beyond the descriptor.  Every load is issued (the wait counts need
        // them): the empty asm keeps the compiler from making branches of the conditions.
        const int left = kbytes - st * 128 - (TB ? 0 : 32 * kq);
        uint32_t k_lo = left > 0 ? (uint32_t)st * (TB ? 2048u : 128u) : kOob;
        uint32_t k_hi = left > (TB ? 0 : 16) ? (uint32_t)st * (TB ? 2048u : 128u) + (TB ? 1024u : 16u) : kOob;
        asm volatile("" : "+v"(k_lo), "+v"(k_hi));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t lo = (woff[j] | k_lo) & kOob ? kOob : woff[j] + k_lo;
            const uint32_t hi = (woff[j] | k_hi) & kOob ? kOob : woff[j] + k_hi;
            constexpr int policy = 0;  // cached: the bands of an expert read the same weights
            w[j] = join(__builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, lo, 0, policy)),
                        __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rw, hi, 0, policy)));
        }
    };

    // Activation rows.  A 1 KiB piece is 8 rows x 128 bytes: lane l holds row l / 8, 16-byte
    // chunk (l % 8) ^ swz(row); piece c is half c % 2 of row block c / 2 (see gemm_stream.hpp).
    const bool gather = p.order != nullptr;
    auto source_row = [&](int m) __attribute__((always_inline)) -> int64_t {
        if (m >= rows) return -1;
        if (!gather) return tile.row0 + m;
        const int pair = p.order[tile.row0 + m];
        const int r = pair / p.top_k;
        return pair >= 0 && r < p.a_rows ? r : -1;
    };
    auto swz = [](int r) __attribute__((always_inline)) { return (r ^ (r >> 3)) & 7; };
    const CopySrc rx = gather ? CopySrc(p.a, (uint32_t)(p.a_rows * p.lda))
                              : CopySrc((const uint8_t*)p.a + tile.row0 * p.lda, (uint32_t)((int64_t)rows * p.lda));
    const int a_half = wave & 1, lo_row = lane >> 3;
    const int a_byte = 16 * ((lane & 7) ^ swz(8 * a_half + lo_row));
    uint32_t aoff[CA];
#pragma unroll
    for (int i = 0; i < CA; ++i) {
        const int c = wave + kBandWaves * i;  // half wave % 2 of row block c / 2
        const int64_t r = source_row(16 * (c >> 1) + 8 * a_half + lo_row);
        aoff[i] = r >= 0 ? (uint32_t)((gather ? r : r - tile.row0) * p.lda + a_byte) : kOob;
    }
    auto copy_a = [&](int st, int slot) __attribute__((always_inline)) {
        const uint32_t base = (uint32_t)(uintptr_t)(ring + slot * STAGE);
        const bool in = a_byte < kbytes - st * 128;
#pragma unroll
        for (int i = 0; i < CA; ++i) {
            uint32_t off = in && aoff[i] != kOob ? aoff[i] + (uint32_t)(st * 128) : kOob;
            asm volatile("" : "+v"(off));
            band_copy(rx, base + (uint32_t)((wave + kBandWaves * i) * 1024), off);
        }
    };
    const uint32_t row_base = (uint32_t)((r16 >> 3) * 1024 + (r16 & 7) * 128);
    const uint32_t frag_lo = row_base + (uint32_t)(((2 * kq) ^ swz(r16)) << 4);
    const uint32_t frag_hi = row_base + (uint32_t)(((2 * kq + 1) ^ swz(r16)) << 4);
    auto frag = [&](int slot, int t) __attribute__((always_inline)) -> v8i {
        const H3Q_LDS uint8_t* q = ring + slot * STAGE + t * 2048;
        return join(*(const H3Q_LDS v4i*)(q + frag_lo), *(const H3Q_LDS v4i*)(q + frag_hi));
    };

    // Scales of the epilogue, one row's and one weight row's a thread until then.
    float my_sa = 0.0f, my_sw = 0.0f;
    uint64_t live;  // rows 64 wave .. + 63
    {
        const int64_t r = threadIdx.x < BM ? source_row(threadIdx.x) : -1;
        if (r >= 0) my_sa = p.a_scale[r];
        live = __ballot(r >= 0);
        const int row = block_row(lane >> 4 & 1);
        if (row < p.n) my_sw = p.b_scale[(int64_t)expert * p.n + row + r16];
    }
    __builtin_amdgcn_sched_barrier(0);

    acc_t acc[2][MT];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = acc_t{};

#pragma unroll
    for (int s = 0; s < SA - 1; ++s) copy_a(s, s);
    v8i w[D][2];
#pragma unroll
    for (int d = 0; d < D; ++d) load_w(d, w[d]);
    wait_vmcnt<(SA - 2) * CA + 4 * D>();  // stage 0 has landed
    asm volatile("s_barrier" ::: "memory");

    int slot = 0;
    auto step = [&](int s, v8i (&ws)[2], auto tail) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail)::value;
        const int next = slot + 1 == SA ? 0 : slot + 1, last = slot == 0 ? SA - 1 : slot - 1;
        const typename Mfma::frag_t w0 = Mfma::frag(ws[0]), w1 = Mfma::frag(ws[1]);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const typename Mfma::frag_t x = Mfma::frag(frag(slot, t));
            acc[0][t] = Mfma::run(w0, x, acc[0][t]);
            acc[1][t] = Mfma::run(w1, x, acc[1][t]);
        }
        __builtin_amdgcn_sched_barrier(0);
        // This wave has read its fragments of stage s and stage s + 1 has landed; after the
        // barrier that holds for every wave, and the slot of stage s - 1 takes stage s - 1 + SA
        // (every wave read that one before the previous barrier).
        wait_vmcnt<TAIL ? WAIT_TAIL : WAIT>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        copy_a(s - 1 + SA, last);
        if constexpr (!TAIL) load_w(s + D, ws);
        __builtin_amdgcn_sched_barrier(0);
        slot = next;
    };
    int s = 0;
    for (; s + D <= steps; s += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) step(s + d, w[d], std::false_type());
    }
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (s + d < steps) step(s + d, w[d], std::true_type());
    wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // The tile in LDS (16-byte chunk c of row r at c ^ (r % 8)), then whole row pieces.
    constexpr int EL = OUT == kOutF32 ? 4 : 2, COLS = SWIGLU ? 64 : 128, PITCH = COLS * EL, CH = PITCH / 16;
    static_assert(BM * PITCH + (MT == 8 ? 4 * (BM + 128 + BM / 32) : 0) <= SA * STAGE, "output tile");
    if (threadIdx.x < BM) lds_sa[threadIdx.x] = my_sa;
    if (lane < 32) lds_sw[32 * wave + lane] = my_sw;
    if (lane < 2 && wave < BM / 64) lds_live[2 * wave + lane] = (uint32_t)(live >> (32 * lane));
    __syncthreads();
    v4f sw[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) sw[j] = *(const H3Q_LDS v4f*)(lds_sw + 32 * wave + 16 * j + 4 * kq);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = 16 * t + r16;
        const float sa = lds_sa[m];
        float y[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) y[j][v] = __fmul_rn(sa, __fmul_rn(sw[j][v], (float)acc[j][t][v]));
        if constexpr (SWIGLU) {
            float h[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) h[v] = swiglu_f32(y[0][v], y[1][v]);
            const int c = 16 * wave + 4 * kq;
            *(H3Q_LDS v2u*)(ring + m * PITCH + (((c >> 3) ^ (m & 7)) << 4) + (c & 4) * 2) =
                v2u{pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3])};
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = 32 * wave + 16 * j + 4 * kq;
                if constexpr (OUT == kOutF32)
                    *(H3Q_LDS v4f*)(ring + m * PITCH + (((c >> 2) ^ (m & 7)) << 4)) =
                        v4f{y[j][0], y[j][1], y[j][2], y[j][3]};
                else
                    *(H3Q_LDS v2u*)(ring + m * PITCH + (((c >> 3) ^ (m & 7)) << 4) + (c & 4) * 2) =
                        v2u{pack_bf16x2(y[j][0], y[j][1]), pack_bf16x2(y[j][2], y[j][3])};
            }
        }
    }
    __syncthreads();
    const int cols = (SWIGLU ? half : p.n) - COLS * slice;
    for (int i = threadIdx.x; i < rows * CH; i += kBandWaves * 64) {
        const int r = i / CH, c = i % CH;
        const v4u v = *(const H3Q_LDS v4u*)(ring + r * PITCH + ((c ^ (r & 7)) << 4));
        if (16 / EL * c < cols && (lds_live[r >> 5] >> (r & 31) & 1))
            *reinterpret_cast<v4u*>((uint8_t*)p.out + ((tile.row0 + r) * p.ldo + COLS * slice) * EL + 16 * c) = v;
    }
}

namespace {

int band_slices(const GroupedArgs& a) { return a.swiglu ? (a.n / 2 + 63) / 64 : (a.n + 127) / 128; }

template <int OP, int MT, bool TB>
hipError_t launch_band_tb(const GroupedArgs& a, hipStream_t st) {
    const int slices = band_slices(a);
    const dim3 grid((unsigned)grouped_band_grid(a, MT)), block(kBandWaves * 64);
    if (OP == kOpE4M3 && a.swiglu && a.wide)
        hipLaunchKernelGGL((grouped_band_kernel<kOpE4M3, MT, TB, kOutWide>), grid, block, 0, st, a, slices);
    else if (a.swiglu)
        hipLaunchKernelGGL((grouped_band_kernel<OP, MT, TB, kOutSwiglu>), grid, block, 0, st, a, slices);
    else if (a.f32)
        hipLaunchKernelGGL((grouped_band_kernel<OP, MT, TB, kOutF32>), grid, block, 0, st, a, slices);
    else
        hipLaunchKernelGGL((grouped_band_kernel<OP, MT, TB, kOutBF16>), grid, block, 0, st, a, slices);
    return hipGetLastError();
}

template <int OP, int MT>
hipError_t launch_band_mt(const GroupedArgs& a, hipStream_t st) {
    return a.b_tiled ? launch_band_tb<OP, MT, true>(a, st) : launch_band_tb<OP, MT, false>(a, st);
}

template <int OP>
hipError_t launch_band_op(const GroupedArgs& a, int blocks, hipStream_t st) {
    return blocks == 4 ? launch_band_mt<OP, 4>(a, st) : launch_band_mt<OP, 8>(a, st);
}

}  // namespace

int64_t grouped_band_grid(const GroupedArgs& a, int blocks) {
    return ((a.experts + a.rows / (16 * blocks)) * band_slices(a) + 7) / 8 * 8;  // a run of each of 8 XCDs
}

hipError_t launch_grouped_band(int kind, const GroupedArgs& a, int blocks, hipStream_t st) {
    return kind == kOpInt8 ? launch_band_op<kOpInt8>(a, blocks, st) : launch_band_op<kOpE4M3>(a, blocks, st);
}

}  // namespace h3q
