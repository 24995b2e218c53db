// What stands between the qkv product and the attention, gfx950: rotary positions, the RMS norm of
// each query and key head, and the append of keys and values to a paged cache.
//
//   n  = x * (1 / sqrt(sum(x * x) / d + eps)) * weight            (rows with a norm)
//   (a, b) -> (a cos - b sin, a sin + b cos)                      (the first 2 * half channels, pair by pair)
//   q  = e4m3(clamp(RN(y / s), +-448)), s a head's own or max(max|y| / 448, 1e-12) of the row   (e4m3 pages)
//
// All of it in binary32 on the values as they are, rounded once where the row is stored.
//
// Bound by the rows' bytes, so one pass: a row of d channels belongs to G lanes (the power of two that
// holds d / (2 V)), each with V pairs of one 16-byte vector per side, and a wave takes 64 / G heads of one
// token at a time.  The token's cosines and sines (fp32: as many bytes as two bf16 rows) and the norm's
// weights stay in registers over the HEADS * 64 / G heads of the wave; its HEADS vectors are asked for
// together, ahead of the first use and of the position and the slot they are needed with.  The lanes that own a row
// read all of it before they store any of it, so a call may run in place.  The folds over a row go by lane
// permutation, two to four instructions where a shuffle takes a round trip through LDS.
//
// Measured, the kernel alone under the profiler: 18603 tokens of 28 + 28 heads of 128, bf16, 107 us, 5.0 TB/s (a copy
// reaches 5.1); 6201 tokens of 28 rotated 16 us, of which the caches hold a part; 8190 tokens of 32 query heads and
// 8 + 8 heads into e4m3 pages with a scale a row 41 us, 4.5 TB/s; one token 3.2 us, two dependent round trips (the call
// in a replayed graph 5.0 to 5.6).
//
// Pairs: (i, half + i), where a lane's two vectors at c V and half + c V hold both sides, or (2 i, 2 i + 1), where
// each of them holds V / 2 whole pairs.  Channels from 2 * half on go through as they are (a select, not a
// rotation by zero: 0 * inf would be a NaN).
#include "h3q_common.hpp"
#include "h3q_kernels.hpp"

namespace h3q {

namespace {

template <int DT>
struct Elem;
template <>
struct Elem<kInBF16> {
    using T = uint16_t;
    static __device__ __forceinline__ float up(T v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ T down(float v) { return (T)pack_bf16x2(v, 0.0f); }
};
template <>
struct Elem<kInF16> {
    using T = uint16_t;
    static __device__ __forceinline__ float up(T v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ T down(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};
template <>
struct Elem<kInF32> {
    using T = float;
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ T down(float v) { return v; }
};

template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Vec<T, 1> {
    typedef T type;
};
template <typename T, int V>
__device__ __forceinline__ T at(const typename Vec<T, V>::type& v, int i) {
    if constexpr (V == 1) return v;
    else return v[i];
}

// A value of the lane that differs in one bit of its number within a row of 16 (for the third and fourth step: of a
// lane whose quad, or half, the other is; the steps before have made those alike).
template <int CTRL>
__device__ __forceinline__ float lane_dpp(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

// f over the `lanes` (a power of two) lanes of a row, in every one of them.
template <typename F>
__device__ __forceinline__ float row_fold(float v, int lanes, F f) {
    if (lanes >= 2) v = f(v, lane_dpp<kDppXor1>(v));
    if (lanes >= 4) v = f(v, lane_dpp<kDppXor2>(v));
    if (lanes >= 8) v = f(v, lane_dpp<kDppHalfMirror>(v));
    if (lanes >= 16) v = f(v, lane_dpp<kDppMirror>(v));
    if (lanes >= 32) v = f(v, __shfl_xor(v, 16, 64));
    if (lanes >= 64) v = f(v, __shfl_xor(v, 32, 64));
    return v;
}

// 1 / sqrt(v), one rounding of the hardware's reciprocal root off, where that has no subnormals either.
__device__ __forceinline__ float inverse_root(float v) {
    const bool tiny = v < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(tiny ? v * 0x1p+100f : v);
    return tiny ? r * 0x1p+50f : r;
}

// V binary32 values -> V e4m3 codes at p.
template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&y)[V]) {
    if constexpr (V == 1) {
        *p = (uint8_t)cvt_e4m3x2(y[0], 0.0f);
    } else {
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            w[i] = cvt_e4m3x2(y[4 * i], y[4 * i + 1]) | (cvt_e4m3x2(y[4 * i + 2], y[4 * i + 3]) << 16);
        if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(p) = w[0];
    }
}

constexpr int kBlockRows = 65535;  // a grid's second extent

// DT: the rows' type.  V: channels a vector.  NC: chunks of 2 V channels a lane (1, or 4 at V = 1).
// HEADS: rows a lane group takes.  INTER: interleaved pairs.  CACHE: some rows go into pages.
template <int DT, int V, int NC, int HEADS, bool INTER, bool CACHE>
__global__ __launch_bounds__(256) void head_rotary_kernel(HeadArgs p) {
    using E = Elem<DT>;
    using T = typename E::T;
    using VT = typename Vec<T, V>::type;
    constexpr int HALF = INTER && V > 1 ? V / 2 : V;  // pairs of one of a lane's vectors
    constexpr int TABLES = V / HALF;                  // runs of cosines a lane
    using VF = typename Vec<float, V>::type;
    using VC = typename Vec<float, HALF>::type;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t token = (((int64_t)blockIdx.z * kBlockRows + blockIdx.y) * 8 + (blockIdx.x & 7)) * 4 + wave;
    if (token >= p.tokens) return;
    int unit = blockIdx.x >> 3, which = 0;
    while (which + 1 < p.segments && unit >= p.seg[which].units) unit -= p.seg[which++].units;
    const HeadSegment& s = p.seg[which];

    // Lanes and row groups past the end load what lies at it, and store nothing: the loads of a wave are one run.
    const int g = lane & (p.lanes - 1), rows = 64 / p.lanes;  // this lane of a row; rows of a wave at a time
    const int first = unit * rows * HEADS, head0 = first + lane / p.lanes;
    const int turned = s.rotate ? p.half / V : 0;  // chunks that are rotated; the others lie behind 2 * half
    const int chunks = p.d / (2 * V);
    // A lane's two vectors are as far apart as its region (the rotated channels, or those behind them) has chunks, so
    // that every access of a wave is whole runs.
    int off[NC][2];
    bool turns[NC];  // of the chunk that is loaded: past the row's end the last one again, values and angles
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int chunk = g + c * 64 < chunks ? g + c * 64 : chunks - 1;
        const bool turn = turns[c] = chunk < turned;
        off[c][0] = turn ? chunk * V : (turned + chunk) * V;
        off[c][1] = off[c][0] + (turn ? turned : chunks - turned) * V;
        if (INTER && V == 1 && turn) {
            off[c][0] = 2 * chunk;
            off[c][1] = 2 * chunk + 1;
        }
    }

    VT raw[HEADS][NC][2];
    const T* const x = (const T*)s.x + token * s.token_stride;
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (first + h * rows >= s.heads) break;  // the wave's last rows
        const int head = head0 + h * rows < s.heads ? head0 + h * rows : s.heads - 1;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                raw[h][c][i] = *reinterpret_cast<const VT*>(x + head * s.head_stride + off[c][i]);
    }

    // Behind the rows' loads: what a token's rows are multiplied by and where they go is one round trip further.
    int64_t pos = token;
    if (p.positions) pos = p.positions_i64 ? ((const int64_t*)p.positions)[token] : ((const int32_t*)p.positions)[token];
    if (pos < 0) return;  // padding: its rows are left as they were
    int64_t to = token * s.out_token_stride, scale_to = 0;
    if (CACHE && s.dest != kDestRows) {
        const int slot = p.slots[token];
        if (slot < 0 || slot >= p.cache_slots) return;  // no page for it
        const int page = slot / p.page_size, place = slot - page * p.page_size;
        to = page * s.cache.page_stride + place * s.cache.slot_stride;
        scale_to = page * s.cache.scale_page_stride + place * s.cache.scale_slot_stride;
    }

    float cs[NC][V], sn[NC][V];
    if (turned > 0) {
        const bool known = pos < p.table_rows;
        const int64_t row = (known ? pos : 0) * p.half;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < TABLES; ++i) {
                const int chunk = g + c * 64 < turned ? g + c * 64 : turned - 1;
                const VC co = *reinterpret_cast<const VC*>(p.cos + row + (chunk + i * turned) * HALF);
                const VC si = *reinterpret_cast<const VC*>(p.sin + row + (chunk + i * turned) * HALF);
#pragma unroll
                for (int e = 0; e < HALF; ++e) {
                    cs[c][i * HALF + e] = at<float, HALF>(co, e);
                    sn[c][i * HALF + e] = at<float, HALF>(si, e);
                }
            }
        if (p.inverse) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) sn[c][e] = -sn[c][e];
        }
        if (!known) {  // a position past the table gives NaN, never another one's angle
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) cs[c][e] = sn[c][e] = __builtin_nanf("");
        }
    }

    float w[NC][2][V];
    auto load_weight = [&](int head) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t o = head * s.weight_stride + off[c][i];
                if (p.weight_f32) {
                    const VF v = *reinterpret_cast<const VF*>((const float*)s.weight + o);
#pragma unroll
                    for (int e = 0; e < V; ++e) w[c][i][e] = at<float, V>(v, e);
                } else {
                    const VT v = *reinterpret_cast<const VT*>((const T*)s.weight + o);
#pragma unroll
                    for (int e = 0; e < V; ++e) w[c][i][e] = E::up(at<T, V>(v, e));
                }
            }
    };
    if (s.weight && s.weight_stride == 0) load_weight(0);

#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (first + h * rows >= s.heads) break;
        const int head = head0 + h * rows;
        float y[NC][2][V];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) y[c][i][e] = E::up(at<T, V>(raw[h][c][i], e));
        if (s.weight) {
            if (s.weight_stride != 0) load_weight(head < s.heads ? head : s.heads - 1);
            float ss = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) part = __builtin_fmaf(y[c][i][e], y[c][i][e], part);
                ss += g + c * 64 < chunks ? part : 0.0f;
            }
            ss = row_fold(ss, p.lanes, [](float a, float b) { return a + b; });
            const float rs = inverse_root(__builtin_fmaf(ss, p.inverse_d, p.eps));
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) y[c][i][e] = y[c][i][e] * rs * w[c][i][e];
        }
        if (turned > 0) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bool turn = turns[c];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    // interleaved: the pairs (2 e, 2 e + 1) of one vector, then of the other
                    float& a = INTER && V > 1 ? y[c][e / HALF][2 * (e % HALF)] : y[c][0][e];
                    float& b = INTER && V > 1 ? y[c][e / HALF][2 * (e % HALF) + 1] : y[c][1][e];
                    const float co = cs[c][e], si = sn[c][e];
                    const float ra = __builtin_fmaf(a, co, -(b * si)), rb = __builtin_fmaf(a, si, b * co);
                    a = turn ? ra : a;
                    b = turn ? rb : b;
                }
            }
        }
        if (!CACHE || s.dest <= kDestPages) {
            T* const row = (CACHE && s.dest != kDestRows ? (T*)s.cache.pages + head * s.cache.head_stride
                                                         : (T*)s.out + head * s.out_head_stride) + to;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    VT v;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        if constexpr (V == 1) v = E::down(y[c][i][e]);
                        else v[e] = E::down(y[c][i][e]);
                    }
                    if (head < s.heads && g + c * 64 < chunks) *reinterpret_cast<VT*>(row + off[c][i]) = v;
                }
            continue;
        }
        float scale;
        if (s.dest == kDestStatic) {
            scale = s.cache.scale[head < s.heads ? head * s.cache.scale_head_stride : 0];
        } else {
            float m = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        m = mag_max(m, __builtin_fabsf(y[c][i][e]));  // lanes past the row have its last chunk's
            m = row_fold(m, p.lanes, [](float a, float b) { return mag_max(a, b); });
            scale = amax_scale(m, kE4M3Recip);
            if (g == 0 && head < s.heads) s.cache.scale[scale_to + head * s.cache.scale_head_stride] = scale;
        }
        const float r = 1.0f / scale;
        uint8_t* const row = (uint8_t*)s.cache.pages + head * s.cache.head_stride + to;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // The quotient from r and one residual; where that leaves no finite value (s or r is 0, infinite or
                // NaN, or y is), IEEE division.
                float q[V];
                bool odd = false;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float v = div_rn_signed(y[c][i][e], scale, r);
                    odd |= !(__builtin_fabsf(v) < __builtin_inff());
                    q[e] = clamp_e4m3(v);
                }
                if (odd) {
#pragma unroll
                    for (int e = 0; e < V; ++e) q[e] = clamp_e4m3(y[c][i][e] / scale);
                }
                if (head < s.heads && g + c * 64 < chunks) store_codes<V>(row + off[c][i], q);
            }
    }
}

// cos and sin of position * frequency, times magnitude.  The angle is a binary64 product (positions of
// millions lose 1e-10 of a turn), taken to turns and reduced to half a turn there; the rest is binary32.
// V values a thread.
template <typename P, int V>
__global__ __launch_bounds__(256) void rotary_tables_kernel(const P* positions, const double* frequencies, int64_t n,
                                                            int half, double magnitude, float* cos_out,
                                                            float* sin_out) {
    using VF = typename Vec<float, V>::type;
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    const uint32_t per = (uint32_t)half / V;
    if (i >= (uint32_t)n * per) return;
    const uint32_t row = i / per, col = (i - row * per) * V;
    const double position = (double)positions[row];
    VF c, s;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const double turns = position * frequencies[col + e] * 0.15915494309189533577;
        const float part = 2.0f * (float)(turns - __builtin_rint(turns));
        float si, co;
        sincospif(part, &si, &co);
        if constexpr (V == 1) {
            c = co * (float)magnitude;
            s = si * (float)magnitude;
        } else {
            c[e] = co * (float)magnitude;
            s[e] = si * (float)magnitude;
        }
    }
    *reinterpret_cast<VF*>(cos_out + (int64_t)row * half + col) = c;
    *reinterpret_cast<VF*>(sin_out + (int64_t)row * half + col) = s;
}

// Position and slot of each token of a step, one thread a token: the last sequence whose first token is
// not behind it (sequences without tokens share their bound with the next), by bisection.
__global__ __launch_bounds__(256) void plan_append_kernel(PlanAppendArgs p) {
    const int64_t token = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (token >= p.tokens) return;
    int position = -1, slot = -1;
    if (token >= p.cu[0] && token < p.cu[p.seqs]) {
        int64_t lo = 0, hi = p.seqs;  // cu[lo] <= token < cu[hi]
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (p.cu[mid] <= token) lo = mid;
            else hi = mid;
        }
        const int64_t at = (int64_t)p.lengths[lo] + token - p.cu[lo];
        if (at >= 0 && at <= 0x7FFFFFFF) {
            position = (int)at;
            const int column = position / p.page_size;
            if (column < p.columns) {
                const int page = p.table[lo * p.table_stride + column];
                const int64_t to = (int64_t)page * p.page_size + position % p.page_size;
                if (page >= 0 && to <= 0x7FFFFFFF) slot = (int)to;
            }
        }
    }
    p.positions[token] = position;
    p.slots[token] = slot;
}

template <int DT, int V, int NC, int HEADS, bool CACHE>
hipError_t launch_heads_pairs(const HeadArgs& a, int units, hipStream_t st) {
    // The units of eight blocks of four tokens one after the other, each block's on one XCD: the few bytes of keys and
    // values are on their way beside the queries (8190 tokens of 32 + 8 + 8 heads into pages 41 us, 45 with all queries
    // first), and a token's cosines come out of that XCD's cache.
    const int64_t blocks = (a.tokens + 31) / 32;
    const dim3 grid((unsigned)(8 * units), (unsigned)(blocks < kBlockRows ? blocks : kBlockRows),
                    (unsigned)((blocks + kBlockRows - 1) / kBlockRows));
    if (a.interleaved) hipLaunchKernelGGL((head_rotary_kernel<DT, V, NC, HEADS, true, CACHE>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((head_rotary_kernel<DT, V, NC, HEADS, false, CACHE>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int DT, int V, int NC, int HEADS>
hipError_t launch_heads_cfg(const HeadArgs& a, int units, hipStream_t st) {
    return a.slots ? launch_heads_pairs<DT, V, NC, HEADS, true>(a, units, st)
                   : launch_heads_pairs<DT, V, NC, HEADS, false>(a, units, st);
}

template <int DT, int V, int NC>
hipError_t launch_heads_vec(HeadArgs a, hipStream_t st) {
    a.inverse_d = 1.0f / (float)a.d;
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes * 2 * V < a.d) a.lanes *= 2;
    const int rows = 64 / a.lanes;
    // Four rows a lane group where that spares waves and leaves the chip more than it holds at once (32 a CU), else one.
    // us, four and one: 18603 tokens of 28 + 28 heads of 128 108 and 123, 8190 of 32 + 8 + 8 into pages 41 and 45; in the
    // caches, 28 + 28 heads of 192: 512 tokens 7.3 and 6.8, 2048 19.7 and 20.3, 4096 32.5 and 34.7; 32 + 8 of 128: 1024 6.9
    // and 5.7, 4096 18.9 and 18.2; 8 + 2 of 64, which one row a group holds: 4096 6.9 and 6.1.
    auto units = [&](int heads) {
        int sum = 0;
        for (int i = 0; i < a.segments; ++i) sum += a.seg[i].units = (a.seg[i].heads + rows * heads - 1) / (rows * heads);
        return sum;
    };
    const int one = units(1), four = units(4);
    if (four < one && a.tokens * four > 8192) return launch_heads_cfg<DT, V, NC, 4>(a, four, st);
    return launch_heads_cfg<DT, V, NC, 1>(a, units(1), st);
}

template <int DT>
hipError_t launch_heads_type(const HeadArgs& a, int vec, hipStream_t st) {
    if constexpr (DT != kInF32) {
        if (vec == 8) return launch_heads_vec<DT, 8, 1>(a, st);
    }
    if (vec >= 4) return launch_heads_vec<DT, 4, 1>(a, st);
    return launch_heads_vec<DT, 1, 4>(a, st);
}

// Whether every vector of V channels of the call is whole and aligned.
bool vectors_fit(const HeadArgs& a, int size, int v) {
    const auto fits = [&](const void* p, int64_t bytes) { return (uintptr_t)p % bytes == 0; };
    if (a.d % (2 * v) || a.half % v) return false;
    if (a.cos && (!fits(a.cos, v >= 4 ? 16 : 4) || !fits(a.sin, v >= 4 ? 16 : 4))) return false;
    for (int i = 0; i < a.segments; ++i) {
        const HeadSegment& s = a.seg[i];
        if (!fits(s.x, v * size) || s.token_stride % v || s.head_stride % v) return false;
        const int wsize = a.weight_f32 ? 4 : size;
        if (s.weight && (!fits(s.weight, v * wsize < 16 ? v * wsize : 16) || s.weight_stride % v)) return false;
        if (s.dest == kDestRows) {
            if (!fits(s.out, v * size) || s.out_token_stride % v || s.out_head_stride % v) return false;
        } else if (!fits(s.cache.pages, v * (s.dest >= kDestStatic ? 1 : size)) || s.cache.page_stride % v ||
                   s.cache.slot_stride % v || s.cache.head_stride % v) {
            return false;
        }
    }
    return true;
}

}  // namespace

hipError_t launch_head_rotary(int dtype, const HeadArgs& a, hipStream_t st) {
    const int size = dtype == kInF32 ? 4 : 2;
    const int vec = dtype != kInF32 && vectors_fit(a, size, 8) ? 8 : vectors_fit(a, size, 4) ? 4 : 1;
    if (dtype == kInBF16) return launch_heads_type<kInBF16>(a, vec, st);
    if (dtype == kInF16) return launch_heads_type<kInF16>(a, vec, st);
    return launch_heads_type<kInF32>(a, vec, st);
}

hipError_t launch_rotary_tables(const void* positions, int type, int64_t n, const double* frequencies, int half,
                                double magnitude, float* cos_out, float* sin_out, hipStream_t st) {
    const int v = half % 4 == 0 && ((uintptr_t)cos_out | (uintptr_t)sin_out) % 16 == 0 ? 4 : 1;
    const unsigned blocks = (unsigned)((n * (half / v) + 255) / 256);
    auto go = [&](auto* at) {
        using P = std::remove_pointer_t<decltype(at)>;
        if (v == 4)
            hipLaunchKernelGGL((rotary_tables_kernel<P, 4>), dim3(blocks), dim3(256), 0, st, (const P*)positions,
                               frequencies, n, half, magnitude, cos_out, sin_out);
        else
            hipLaunchKernelGGL((rotary_tables_kernel<P, 1>), dim3(blocks), dim3(256), 0, st, (const P*)positions,
                               frequencies, n, half, magnitude, cos_out, sin_out);
    };
    if (type == kPositionsI32) go((int32_t*)nullptr);
    else if (type == kPositionsI64) go((int64_t*)nullptr);
    else if (type == kPositionsF32) go((float*)nullptr);
    else go((double*)nullptr);
    return hipGetLastError();
}

hipError_t launch_plan_append(const PlanAppendArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(plan_append_kernel, dim3((unsigned)((a.tokens + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace h3q
