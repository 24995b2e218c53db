// The FFN of a routed-expert layer on quantized weights, gfx950:
//
//   q, s = codes of x per token;   h = bf16(silu(gate) * up) of q against w13[e]
//   qh, sh = codes of h per pair;  y = sh * (s2[e] * (qh . w2[e]))
//   out[t] = bf16(sum_j weights[t, j] * y[t, j])
//
// The quantizers are the dense linears' (int8: the reciprocal form; e4m3: division).
// They take bf16 rows, so h is rounded to bf16 before its codes, as the activations
// between two dense linears are; gate and up are not rounded before that, and y stays
// binary32 up to the sum over the experts, which is rounded once.
//
// A few tokens take two kernels of their own (expert_few.hip).  The rest, here: plan, quantize, grouped gate-up product with SwiGLU (rows gathered from the
// tokens' codes, so no copy of a token per expert is made), quantize, grouped down product,
// weighted sum.
#include "h3q_common.hpp"
#include "h3q_kernels.hpp"

namespace h3q {

namespace {

struct Workspace {
    uint8_t* base;
    int64_t used = 0;
    template <class T>
    T* take(int64_t n) {
        T* const p = (T*)(base + used);
        used += (n * (int64_t)sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

struct Parts {
    int *order, *offsets, *slots, *plan;
    uint8_t* xq;
    float* xs;
    uint16_t* h;
    uint8_t* hq;
    float* hs;
    float* y;
};

Parts carve(Workspace& w, const ExpertFfnArgs& a) {
    const int64_t pairs = a.tokens * a.top_k;
    Parts p;
    p.order = w.take<int>(pairs);
    p.offsets = w.take<int>(a.experts + 1);
    p.slots = w.take<int>(pairs);
    p.plan = w.take<int>(plan_workspace_ints(pairs, a.experts));
    p.xq = w.take<uint8_t>(a.tokens * a.d);
    p.xs = w.take<float>(a.tokens);
    p.h = w.take<uint16_t>(pairs * a.f);
    p.hq = w.take<uint8_t>(pairs * a.f);
    p.hs = w.take<float>(pairs);
    p.y = w.take<float>(pairs * a.d);
    return p;
}

// The two products, over rows sorted by expert.
GroupedArgs gate_up(const ExpertFfnArgs& a, const Parts& p) {
    GroupedArgs g{};
    g.a = p.xq;
    g.lda = a.d;
    g.a_rows = a.tokens;
    g.a_scale = p.xs;
    g.order = p.order;
    g.top_k = a.top_k;
    g.b = a.w13;
    g.b_tiled = a.w13_tiled;
    g.b_scale = a.s13;
    g.offsets = p.offsets;
    g.experts = a.experts;
    g.rows = a.tokens * a.top_k;
    g.n = (int)(2 * a.f);
    g.k = a.d;
    g.swiglu = 1;
    g.wide = 1;  // h is quantized again
    g.out = p.h;
    g.ldo = a.f;
    return g;
}

GroupedArgs down(const ExpertFfnArgs& a, const Parts& p) {
    GroupedArgs g{};
    g.a = p.hq;
    g.lda = a.f;
    g.a_rows = a.tokens * a.top_k;
    g.a_scale = p.hs;
    g.top_k = 1;
    g.b = a.w2;
    g.b_tiled = a.w2_tiled;
    g.b_scale = a.s2;
    g.offsets = p.offsets;
    g.experts = a.experts;
    g.rows = g.a_rows;
    g.n = (int)a.d;
    g.k = a.f;
    g.f32 = 1;
    g.out = p.y;
    g.ldo = a.d;
    return g;
}

}  // namespace

bool expert_ffn_fits(const ExpertFfnArgs& a) {
    const Parts none{};
    return expert_few_supported(a) ||
           (grouped_mm_fits(a.kind, gate_up(a, none)) && grouped_mm_fits(a.kind, down(a, none)));
}

int64_t expert_ffn_workspace_bytes(const ExpertFfnArgs& a) {
    Workspace w{nullptr};
    carve(w, a);
    return w.used;
}

hipError_t launch_expert_ffn(const ExpertFfnArgs& a, void* workspace, hipStream_t st) {
    const int64_t pairs = a.tokens * a.top_k;
    const int fmt = a.kind == kOpInt8 ? kFmtInt8 : kFmtE4M3;
    const int rounding = a.kind == kOpInt8 ? kRoundRcpMul : kRoundDiv;
    Workspace w{(uint8_t*)workspace};
    const Parts p = carve(w, a);
    if (expert_few_supported(a)) return launch_expert_few(a, FewBuffers{p.xq, p.xs, p.h, p.hq, p.hs}, st);

    PlanArgs plan{};
    plan.ids = a.ids;
    plan.pairs = pairs;
    plan.first = a.first;
    plan.experts = a.experts;
    plan.order = p.order;
    plan.offsets = p.offsets;
    plan.slots = p.slots;
    plan.workspace = p.plan;
    hipError_t e;
    if (plan_quant_supported(plan, a.tokens)) {
        e = launch_plan_quant(plan, fmt, a.x, a.ldx, a.tokens, a.d, p.xq, p.xs, st);
    } else {
        e = launch_plan_experts(plan, st);
        if (e == hipSuccess) e = launch_quant_rows(a.x, a.ldx, a.tokens, a.d, fmt, rounding, p.xq, a.d, p.xs, st);
    }
    if (e != hipSuccess) return e;
    e = launch_grouped_mm(a.kind, gate_up(a, p), st);
    if (e != hipSuccess) return e;
    // Rows past the last placed pair hold what the workspace held; their codes are never read.
    e = launch_quant_rows(p.h, a.f, pairs, a.f, fmt, rounding, p.hq, a.f, p.hs, st);
    if (e != hipSuccess) return e;
    e = launch_grouped_mm(a.kind, down(a, p), st);
    if (e != hipSuccess) return e;

    CombineArgs c{};
    c.y = p.y;
    c.ldy = a.d;
    c.rows = pairs;
    c.slots = p.slots;
    c.weights = a.weights;
    c.tokens = a.tokens;
    c.top_k = a.top_k;
    c.cols = a.d;
    c.out = a.out;
    c.ldo = a.ldo;
    return launch_combine_experts(c, true, st);
}

}  // namespace h3q
