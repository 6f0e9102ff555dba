// rope.h — the rotation of a token's heads, for rope.hip and for the kernel that
// also stores the keys (rope_store.hip).  The mathematics is described in
// rope.hip.
#pragma once
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

// The arguments of rows r by plan p, on 16-byte accesses (*vec) where every
// unit's dims are 16-byte aligned, else 4-byte ones.
RopeArgs rope_args(const EhipRopePlan &p, const EhipRopeRows &r, bool *vec);

// A unit is VEC dims and their VEC partners: pairs of turning dims, then plain
// ones.  Lane u of a head's lanes takes the units u, u + lg (UPL of them).
// A wave's head groups g0, g0 + gs, ... below g1 of token tok; head_of(i): the
// row's i-th head of `count`, 64 / lg of them to a group.
template <int VEC, int UPL, bool NORM, class Heads>
__device__ __forceinline__ void rope_heads(const RopeArgs &a, const EhipRopePlan &p, int tok, int g0, int g1, int gs, int count, Heads head_of) {
    typedef float V __attribute__((ext_vector_type(VEC)));
    const int lane = threadIdx.x & 63;
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
    for (int g = g0; g < g1; g += gs) {
        const int i = g * hpw + lane / a.lg, h = head_of(min(i, count - 1));
        const bool in = i < count;
        const float *xh = xr + (int64_t)h * hd;
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

}  // namespace ehip
