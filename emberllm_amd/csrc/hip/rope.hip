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

#include "session.h"

namespace ehip {

// a pair's (cos, sin) of `turns` per position, times the plan's magnitude
__device__ __forceinline__ float2 turn_by(int pos, uint64_t turns, float magnitude) {
    const uint64_t t = (uint64_t)(int64_t)pos * turns;               // (overflow drops whole turns)
    const int quarter = (int)((t + (1ull << 61)) >> 62);
    const int64_t r = (int64_t)(t - ((uint64_t)quarter << 62));      // [-2^61, 2^61)
    const float x = (float)(int)(r >> 30) * 3.6572952e-10f;          // 2 pi / 2^34
    const float y = x * x;
    const float s = x + x * y * (-1.66666667e-1f + y * (8.33333333e-3f + y * (-1.98412698e-4f + y * 2.75573192e-6f)));
    const float c = 1.0f + y * (-0.5f + y * (4.16666667e-2f + y * (-1.38888889e-3f + y * (2.48015873e-5f - y * 2.75573192e-7f))));
    float cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;        // quarters 1 and 3 swap them
    if (quarter == 1 || quarter == 2) cc = -cc;
    if (quarter >= 2) ss = -ss;
    return make_float2(cc * magnitude, ss * magnitude);
}

struct RopeArgs {
    const float *x;
    float *out;
    int64_t x_stride, out_stride;
    int n_tok, n_q, heads, pos0;
    const int *pos;
    const float *q_norm, *k_norm;
    float eps, inv_hd;
    int parts, per;       // a token's head groups in `parts` parts of `per`
    int lg;               // lanes of a head (a power of two)
};

// A unit is VEC dims and their VEC partners: pairs of turning dims, then plain
// ones.  Lane u of a head's lanes takes the units u, u + lg (UPL of them).
template <int VEC, int UPL, bool NORM>
__global__ __launch_bounds__(WG) void k_rope(RopeArgs a, EhipRopePlan p) {
    typedef float V __attribute__((ext_vector_type(VEC)));
    const int lane = threadIdx.x & 63, w = blockIdx.x * (WG / 64) + (threadIdx.x >> 6);
    const int tok = w / a.parts, part = w % a.parts;
    if (tok >= a.n_tok) return;
    const int hd = p.head_dim, half = p.rotary_dim / 2, units = hd / (2 * VEC), turning = half / VEC;
    const int u0 = lane & (a.lg - 1), hpw = 64 / a.lg;
    const int pos = a.pos ? a.pos[tok] : a.pos0 + tok;
    int da[UPL], db[UPL];        // first dim of each unit, and of its partners
    bool live[UPL], turns[UPL];
    float cs[UPL][VEC], sn[UPL][VEC];
#pragma unroll
    for (int k = 0; k < UPL; k++) {
        const int u = u0 + k * a.lg;
        live[k] = u < units;
        turns[k] = u < turning;
        if (turns[k] && p.style == ROPE_INTERLEAVED) {
            da[k] = 2 * VEC * u;
            db[k] = da[k] + VEC;
        } else if (turns[k]) {
            da[k] = VEC * u;
            db[k] = da[k] + half;
        } else {
            da[k] = 2 * half + 2 * VEC * (u - turning);
            db[k] = da[k] + VEC;
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            // neox: VEC consecutive pairs; interleaved: the pairs (2j, 2j + 1) of the unit's dims
            const float2 t = turns[k] ? turn_by(pos, p.turns[VEC * u + j], p.magnitude) : make_float2(1.0f, 0.0f);
            cs[k][j] = t.x;
            sn[k][j] = t.y;
        }
    }
    const bool inter = p.style == ROPE_INTERLEAVED;
    const float *xr = a.x + (int64_t)tok * a.x_stride;
    float *yr = a.out + (int64_t)tok * a.out_stride;
    const int g0 = part * a.per, g1 = min(g0 + a.per, (a.heads + hpw - 1) / hpw);
    for (int g = g0; g < g1; g++) {
        const int h = g * hpw + lane / a.lg;
        const bool in = h < a.heads;
        const float *xh = xr + (int64_t)min(h, a.heads - 1) * hd;
        V va[UPL], vb[UPL];
#pragma unroll
        for (int k = 0; k < UPL; k++) {
            va[k] = *reinterpret_cast<const V *>(xh + (live[k] ? da[k] : 0));
            vb[k] = *reinterpret_cast<const V *>(xh + (live[k] ? db[k] : 0));
        }
        if (NORM) {
            const float *nw = h < a.n_q ? a.q_norm : a.k_norm;
            if (nw) {   // one of the two may be left out
                float ss = 0.0f;
#pragma unroll
                for (int k = 0; k < UPL; k++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const float x = va[k][j], y = vb[k][j];
                        ss += live[k] ? x * x + y * y : 0.0f;
                    }
                for (int off = 1; off < a.lg; off <<= 1) ss += __shfl_xor(ss, off);
                const float inv = 1.0f / sqrtf(ss * a.inv_hd + a.eps);
#pragma unroll
                for (int k = 0; k < UPL; k++) {
                    V wa = *reinterpret_cast<const V *>(nw + (live[k] ? da[k] : 0)), wb = *reinterpret_cast<const V *>(nw + (live[k] ? db[k] : 0));
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        va[k][j] *= inv * wa[j];
                        vb[k][j] *= inv * wb[j];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < UPL; k++) {
            V ya = va[k], yb = vb[k];
            if (turns[k])
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                if (VEC > 1 && inter) {   // pair j: elements 2j, 2j + 1 of the 2 VEC dims
                    V &src = 2 * j < VEC ? va[k] : vb[k], &dst = 2 * j < VEC ? ya : yb;
                    const float x = src[2 * j % VEC], y = src[(2 * j + 1) % VEC];
                    dst[2 * j % VEC] = x * cs[k][j] - y * sn[k][j];
                    dst[(2 * j + 1) % VEC] = x * sn[k][j] + y * cs[k][j];
                } else {
                    const float x = va[k][j], y = vb[k][j];
                    ya[j] = x * cs[k][j] - y * sn[k][j];
                    yb[j] = x * sn[k][j] + y * cs[k][j];
                }
            }
            if (in && live[k]) {
                *reinterpret_cast<V *>(yr + (int64_t)h * hd + da[k]) = ya;
                *reinterpret_cast<V *>(yr + (int64_t)h * hd + db[k]) = yb;
            }
        }
    }
}

template <int VEC, int UPL>
static void rope_go(hipStream_t st, dim3 grid, const RopeArgs &a, const EhipRopePlan &p) {
    if (a.q_norm || a.k_norm) hipLaunchKernelGGL((k_rope<VEC, UPL, true>), grid, dim3(WG), 0, st, a, p);
    else hipLaunchKernelGGL((k_rope<VEC, UPL, false>), grid, dim3(WG), 0, st, a, p);
}

int launch_rope(hipStream_t st, const EhipRopePlan &p, const EhipRopeRows &r) {
    RopeArgs a{};
    a.x = r.x; a.out = r.out; a.x_stride = r.x_stride; a.out_stride = r.out_stride;
    a.n_tok = r.n_tok; a.n_q = r.n_q; a.heads = r.n_q + r.n_k; a.pos0 = r.pos0; a.pos = r.pos;
    a.q_norm = r.q_norm; a.k_norm = r.k_norm; a.eps = r.eps;
    const int hd = p.head_dim;
    a.inv_hd = 1.0f / hd;
    // 16-byte accesses where every unit's dims are 16-byte aligned, else 4-byte ones
    const bool vec = hd % 8 == 0 && p.rotary_dim % 8 == 0 && r.x_stride % 4 == 0 && r.out_stride % 4 == 0 && aligned(r.x, 16) &&
                     aligned(r.out, 16) && aligned(r.q_norm, 16) && aligned(r.k_norm, 16);
    const int units = hd / (vec ? 8 : 2);
    int lg = 1;
    while (lg < units && lg < 64) lg <<= 1;
    a.lg = lg;
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
