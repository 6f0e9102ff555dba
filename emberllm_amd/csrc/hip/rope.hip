// rope.hip — rotary positions of device rows: ehip_rope_plan, ehip_rope_rows.
//
// A pair of dims (a, b) of a head at position p turns by the angle p f_i:
//   a' = a cos - b sin,  b' = a sin + b cos,
// with f_i scaled for contexts beyond the training's (EhipRopeConfig).  The
// plan holds f_i as a fraction of a full turn in 64-bit fixed point, so
// p f_i modulo a turn is one 64-bit multiplication whose overflow is the whole
// turns: exact to 2^-64 p of a turn at any position (an fp32 product p f_i is
// off by 4e-3 rad at position 70000, and a table of cos and sin, as the states'
// default path has it, is 16 MB at 32768 positions).  What is left of the
// fraction after its nearest quarter turn, |x| <= pi/4, goes through the Taylor
// polynomials of sin (to x^9) and cos (to x^10), whose next terms are below
// 2e-9 there.
//
// Bound: memory (4 bytes in and out per value).  A wave takes one token and
// the heads of one part of its row; a lane holds VEC dims and their partners,
// computes their VEC angles once and uses them for all of its heads.  A token of
// 16 + 8 heads of 128 with QK-norm 3.4 us (the launch); 4096 tokens of 9 + 3 heads
// of 64, half of each turning, 7.3 us (25 MB, 3.4 TB/s at this length, start and
// end included).
#include <cmath>

#include "rope.h"

namespace ehip {

template <int VEC, int UPL, bool NORM>
__global__ __launch_bounds__(WG) void k_rope(RopeArgs a, EhipRopePlan p) {
    const int w = blockIdx.x * (WG / 64) + (threadIdx.x >> 6);
    const int tok = w / a.parts, part = w % a.parts, hpw = 64 / a.lg;
    if (tok >= a.n_tok) return;
    const int g0 = part * a.per, g1 = min(g0 + a.per, (a.heads + hpw - 1) / hpw);
    rope_heads<VEC, UPL, NORM>(a, p, tok, g0, g1, 1, a.heads, [](int i) { return i; });
}

template <int VEC, int UPL>
static void rope_go(hipStream_t st, dim3 grid, const RopeArgs &a, const EhipRopePlan &p) {
    if (a.q_norm || a.k_norm) hipLaunchKernelGGL((k_rope<VEC, UPL, true>), grid, dim3(WG), 0, st, a, p);
    else hipLaunchKernelGGL((k_rope<VEC, UPL, false>), grid, dim3(WG), 0, st, a, p);
}

RopeArgs rope_args(const EhipRopePlan &p, const EhipRopeRows &r, bool *vec) {
    RopeArgs a{};
    a.x = r.x; a.out = r.out; a.x_stride = r.x_stride; a.out_stride = r.out_stride;
    a.n_tok = r.n_tok; a.n_q = r.n_q; a.heads = r.n_q + r.n_k; a.pos0 = r.pos0; a.pos = r.pos;
    a.q_norm = r.q_norm; a.k_norm = r.k_norm; a.eps = r.eps;
    const int hd = p.head_dim;
    a.inv_hd = 1.0f / hd;
    *vec = hd % 8 == 0 && p.rotary_dim % 8 == 0 && r.x_stride % 4 == 0 && r.out_stride % 4 == 0 && aligned(r.x, 16) &&
           aligned(r.out, 16) && aligned(r.q_norm, 16) && aligned(r.k_norm, 16);
    const int units = hd / (*vec ? 8 : 2);
    int lg = 1;
    while (lg < units && lg < 64) lg <<= 1;
    a.lg = lg;
    return a;
}

int launch_rope(hipStream_t st, const EhipRopePlan &p, const EhipRopeRows &r) {
    bool vec;
    RopeArgs a = rope_args(p, r, &vec);
    const int lg = a.lg, units = p.head_dim / (vec ? 8 : 2);
    const int groups = (a.heads + 64 / lg - 1) / (64 / lg);
    // A part per head group while the launch has fewer waves than the GPU can
    // hold at once, else the whole row, which computes its angles once.
    a.parts = (int64_t)r.n_tok * groups <= 4096 ? groups : 1;
    a.per = (groups + a.parts - 1) / a.parts;
    const int64_t waves = (int64_t)r.n_tok * a.parts;
    const dim3 grid((unsigned)((waves + WG / 64 - 1) / (WG / 64)));
    if (vec) rope_go<4, 1>(st, grid, a, p);
    else if (units <= 64) rope_go<1, 1>(st, grid, a, p);
    else rope_go<1, 2>(st, grid, a, p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ehip

using namespace ehip;

extern "C" int ehip_rope_plan(const EhipRopeConfig *c, int head_dim, EhipRopePlan *plan) {
    const char *who = "ehip_rope_plan";
    if (!c || !plan) return refuse("%s: null argument", who);
    if (head_dim < 2 || head_dim > 256 || head_dim % 2) return refuse("%s: head_dim %d is not an even number up to 256", who, head_dim);
    const int rd = c->rotary_dim ? c->rotary_dim : head_dim;
    if (rd < 2 || rd > head_dim || rd % 2) return refuse("%s: rotary_dim %d of a head of %d", who, c->rotary_dim, head_dim);
    if (c->style != EMBER_ROPE_INTERLEAVED && c->style != EMBER_ROPE_NEOX) return refuse("%s: unknown rope style %d", who, c->style);
    if (c->scaling < EHIP_ROPE_PLAIN || c->scaling > EHIP_ROPE_BANDS) return refuse("%s: unknown scaling %d", who, c->scaling);
    double theta = c->theta;
    const double factor = c->scaling == EHIP_ROPE_PLAIN ? 1.0 : (double)c->factor;
    if (!(theta > 1.0) || !std::isfinite(theta)) return refuse("%s: theta %g is not above 1", who, theta);
    if (!(factor >= 1.0) || !std::isfinite(factor)) return refuse("%s: factor %g is not at least 1", who, factor);
    if (!std::isfinite(c->magnitude) || c->magnitude < 0.0f) return refuse("%s: magnitude %g", who, (double)c->magnitude);
    double low = c->low, high = c->high;
    const double orig = c->orig_ctx, two_pi = 6.283185307179586;
    if (c->scaling == EHIP_ROPE_YARN || c->scaling == EHIP_ROPE_BANDS) {
        if (low == 0.0 && high == 0.0) { low = 1.0; high = c->scaling == EHIP_ROPE_YARN ? 32.0 : 4.0; }
        if (!(low > 0.0) || !(high > low) || !std::isfinite(high)) return refuse("%s: bounds %g and %g", who, low, high);
        if (c->orig_ctx < 1) return refuse("%s: orig_ctx %d", who, c->orig_ctx);
    }
    if (c->scaling == EHIP_ROPE_NTK) {
        if (rd < 4) return refuse("%s: NTK scaling needs a rotary_dim of at least 4", who);
        theta *= pow(factor, (double)rd / (rd - 2));
    }
    double first = 0.0, last = 0.0;   // YARN: the ramp's pairs
    if (c->scaling == EHIP_ROPE_YARN) {
        const double per = rd / (2.0 * log(theta));
        first = fmax(floor(per * log(orig / (high * two_pi))), 0.0);
        last = fmin(ceil(per * log(orig / (low * two_pi))), rd - 1.0);
    }
    EhipRopePlan p{};
    p.style = c->style;
    p.head_dim = head_dim;
    p.rotary_dim = rd;
    p.magnitude = c->magnitude != 0.0f ? c->magnitude : c->scaling == EHIP_ROPE_YARN ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    for (int i = 0; i < rd / 2; i++) {
        double f = pow(theta, -2.0 * i / rd);
        double keep = c->scaling == EHIP_ROPE_LINEAR ? 0.0 : 1.0;   // the share of f that is not scaled
        if (c->scaling == EHIP_ROPE_YARN) keep = 1.0 - fmin(fmax((i - first) / fmax(last - first, 0.001), 0.0), 1.0);
        if (c->scaling == EHIP_ROPE_BANDS) keep = fmin(fmax((orig * f / two_pi - low) / (high - low), 0.0), 1.0);
        f = f / factor * (1.0 - keep) + f * keep;
        p.turns[i] = (uint64_t)llrint(ldexp(f / two_pi, 62)) << 2;   // f <= 1: below 2^60 before the shift
    }
    *plan = p;
    return 0;
}

extern "C" int ehip_rope_rows(const EhipRopePlan *p, const EhipRopeRows *r, void *stream) {
    const char *who = "ehip_rope_rows";
    if (!p || !r) return refuse("%s: null argument", who);
    if (p->head_dim < 2 || p->head_dim > 256 || p->head_dim % 2 || p->rotary_dim < 2 || p->rotary_dim > p->head_dim || p->rotary_dim % 2 ||
        (p->style != EMBER_ROPE_INTERLEAVED && p->style != EMBER_ROPE_NEOX))
        return refuse("%s: the plan was not made by ehip_rope_plan", who);
    if (r->n_tok < 0 || r->n_q < 0 || r->n_k < 0 || (int64_t)r->n_q + r->n_k > 65536)
        return refuse("%s: %d tokens of %d and %d heads", who, r->n_tok, r->n_q, r->n_k);
    if (!r->n_tok || !(r->n_q + r->n_k)) return 0;
    if (!r->x || !r->out) return refuse("%s: null rows", who);
    const int64_t width = ((int64_t)r->n_q + r->n_k) * p->head_dim;
    if (r->n_tok > 1 && (r->x_stride < width || r->out_stride < width))
        return refuse("%s: strides %lld and %lld for rows of %lld floats", who, (long long)r->x_stride, (long long)r->out_stride, (long long)width);
    if (!r->pos && (int64_t)r->pos0 + r->n_tok - 1 > INT32_MAX) return refuse("%s: positions pass 2^31", who);
    if ((r->q_norm || r->k_norm) && !(r->eps >= 0.0f)) return refuse("%s: eps %g", who, (double)r->eps);
    if (launch_rope(static_cast<hipStream_t>(stream), *p, *r)) return refuse("%s: launch failed", who);
    return 0;
}
