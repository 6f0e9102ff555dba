// attend.hip — attention over a device cache of fp32, fp16 or 4 bits, with a
// sliding window and first positions that stay visible: ehip_attend.
//
// For a row (token at position p, query head) of key head g:
//   s_t = q . k_t * scale,  w_t = exp(s_t - max s),  o = sum w_t v_t / sum w_t
// over t <= p and, with a window W, t > p - W or t < sinks.  One pass over the
// cache with a running maximum and sum.
//
// A wave takes up to 16 CT rows of one key head (rows are (token, head) pairs,
// so a cached row serves all its query heads) and tiles of 32 positions:
//   S^T = K . Q^T  per 16 positions x 16 rows: a lane (l, g) = (lane % 16,
//         lane / 16) supplies position l of K and row l of Q, 8 dims of quarter
//         g of every 32, and receives S[position 4g + i][row l], i < 4;
//   O^T += V^T . P^T  per 16 dims x 16 rows: the contraction runs over the
//         tile's positions in the order 16s + 4g + i in which the lanes hold
//         the scores, so a lane's own probabilities are the operand and never
//         leave its registers, and it receives O[dim 4g + i][row l].
// The 4-bit cache lies in memory as the lanes use it (EhipCache): a lane's
// codes come in 16-byte loads, no LDS is passed, and no wave waits for another
// until the end.
//
// Precision.  The fp16 matrix cores take fp32 operands as hi + lo: x scaled by
// a power of two, hi = fp16(x), lo = fp16(x - hi), |x - hi - lo| <= 2^-23 |x|;
// products and sums are fp32.  q is scaled per row (its largest element into
// [2^13, 2^14)), times scale * log2(e) first, so the scores are in log2 units.
// Codes are exact in fp16; a score is the sum over its blocks of (block's
// product) * d in fp32.  A value (code - 8) d has at most 15 bits, so hi =
// fp16((code - 8) d) and lo = (code - 8) d - hi hold it exactly at any fp16 d.
// Probabilities are split times 2^14 (what a half loses at its smallest is
// 2^-39 of the largest), which the outputs' sums carry until the end; of the
// four products of halves the smallest, lo.lo below 2^-24 of the whole, is
// left out where it is not free.  fp16 caches are one half already; an fp32
// cache goes through the fp32 matrix cores as it is.
//
// What a row does not see cannot reach it: its scores are selected away, its
// probabilities are zero, and where a zero times what the cache holds would be
// NaN (infinite or NaN values, scales of positions never stored) a 4-bit scale
// becomes zero and the scores of the rows that see it NaN, and an fp16 or fp32
// value's products are made one by one for the rows that see it.
#include "session.h"

namespace ehip {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct AttendArgs {
    const float *q;
    float *out;
    int64_t q_stride, out_stride;
    const uint8_t *kc, *vc;
    int64_t head_bytes;          // 4 bits: bytes of a key head's tiles
    int kvd;                     // others: elements of a position
    int n_tok, n_kv, G, pos0, ctx;
    const int *pos;
    int out_vec;                 // out rows take 16-byte stores
    int window, sinks;
    float qscale;                // scale * log2(e)
    int nsplit;                  // workgroups that share a row group's positions
    float *part;                 // [unit][nsplit][rows][HD], then float4 [unit][nsplit][rows]; unit = (row group, key head)
    float4 *part_ml;             // a row's maximum, sum and score scale
    int *count;                  // [unit]: workgroups of the unit that are done; zero between launches
};

constexpr int AT_SPLITS = 64;    // workgroups that a unit's tiles are shared over at most

// maximum / sum over the four lane quarters of a row
__device__ __forceinline__ float quarters_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float quarters_sum(float v) { return xor32_add(xor16_add(v)); }

__device__ __forceinline__ uint32_t pack2(_Float16 a, _Float16 b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, a) | ((uint32_t)__builtin_bit_cast(uint16_t, b) << 16);
}
__device__ __forceinline__ f16x8 as_f16(i32x4 v) { return __builtin_bit_cast(f16x8, v); }
// a dword's two fp16 numbers, and back (by value: __builtin_bit_cast of a
// vector's element takes its first one)
__device__ __forceinline__ f16x2 halves(int w) { return __builtin_bit_cast(f16x2, w); }
__device__ __forceinline__ int dword(f16x2 h) { return __builtin_bit_cast(int, h); }
// number s, widened
__device__ __forceinline__ float half_of(int w, int s) { return (float)halves(w)[s]; }

// The 8 codes of a dword, minus 8, as fp16 pairs (n, n + 4), n = 0 .. 3; the
// pairs of odd n come 16 times too large, which their partner operand makes
// up.  0x6400 is 1024, whose last mantissa bits take a code as it lies (the low
// nibble) or 16 times it.  magic: 0x64006400 in a vector register, so that a
// mask and it make one instruction (v_and_or_b32 takes one scalar).
__device__ __forceinline__ uint32_t code_magic() {
    uint32_t m = 0x64006400u;
    asm volatile("" : "+v"(m));
    return m;
}
__device__ __forceinline__ i32x4 codes_signed(uint32_t w, uint32_t magic) {
    const f16x2 lo = { (_Float16)-1032.0f, (_Float16)-1032.0f }, hi = { (_Float16)-1152.0f, (_Float16)-1152.0f };
    auto one = [](uint32_t bits, f16x2 off) { return dword(halves((int)bits) + off); };
    const uint32_t v = w >> 8;
    return i32x4{ one((w & 0x000f000fu) | magic, lo), one((w & 0x00f000f0u) | magic, hi),
                  one((v & 0x000f000fu) | magic, lo), one((v & 0x00f000f0u) | magic, hi) };
}

// Which tiles of 32 positions the rows r0 .. r1 - 1 of a launch see: the sinks'
// tiles [0, ns), then those from w0 on; n in all, tile of index v.
struct Tiles {
    int ns, w0, n;
    __device__ __forceinline__ int at(int v) const { return v < ns ? v : v - ns + w0; }
};
__device__ __forceinline__ Tiles tiles_seen(int first_pos, int last_pos, int window, int sinks) {
    Tiles t;
    const int last = last_pos / KV_TILE;
    t.ns = 0;
    t.w0 = 0;
    if (window > 0) {
        t.ns = sinks > 0 ? min((sinks - 1) / KV_TILE, last) + 1 : 0;
        t.w0 = max(max(first_pos - window + 1, 0) / KV_TILE, t.ns);
    }
    t.n = t.ns + max(last + 1 - t.w0, 0);
    return t;
}

// The rows of a wave: CT groups of 16 (PACK: one of 8, whose columns 8 .. 15
// hold the low halves of the same rows), their running softmax and output.
template <int HD, int CT> struct Rows {
    float sc[CT];                // score = product * sc
    int p[CT];                   // the row's position
    float m[CT], l[CT];          // maximum (in products), this lane's share of the sum
    f32x4 o[CT][HD / 16];
};

// sum and maximum updates shared by the cache types: S[c][s][i] are products
// (masked ones -inf), which become the probabilities 2^((S - max) sc).  up: what
// the output's sums are multiplied by beside (a new exponent), 1 mostly.
template <int HD, int CT>
__device__ __forceinline__ void softmax_step(Rows<HD, CT> &R, f32x4 (&S)[CT][2], float up) {
#pragma unroll
    for (int c = 0; c < CT; c++) {
        float t = fmaxf(fmaxf(S[c][0][0], S[c][0][1]), fmaxf(S[c][0][2], S[c][0][3]));
        t = fmaxf(t, fmaxf(fmaxf(S[c][1][0], S[c][1][1]), fmaxf(S[c][1][2], S[c][1][3])));
        const float mn = fmaxf(R.m[c], quarters_max(t));
        if (__any(mn > R.m[c]) || up != 1.0f) {
            const float a = R.m[c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((R.m[c] - mn) * R.sc[c]);
            R.l[c] *= a;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) R.o[c][d] *= a * up;
            R.m[c] = mn;
        }
        // (the difference first: the exponential's argument is then off by
        // its own rounding only, at whatever size the scores are)
        const float mu = mn == -INFINITY ? 0.0f : mn;
        float l = 0.0f;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                S[c][s][i] = __builtin_amdgcn_exp2f((S[c][s][i] - mu) * R.sc[c]);
                l += S[c][s][i];
            }
        R.l[c] += l;
    }
}

// the scores of positions that a row does not see become -inf
template <int HD, int CT>
__device__ __forceinline__ bool seen(const AttendArgs &a, const Rows<HD, CT> &R, int c, int t) {
    return t <= R.p[c] && (a.window <= 0 || t > R.p[c] - a.window || t < a.sinks);
}
template <int HD, int CT>
__device__ __forceinline__ void mask_scores(const AttendArgs &a, const Rows<HD, CT> &R, f32x4 (&S)[CT][2], int t0) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!seen(a, R, c, t0 + 16 * s + 4 * g + i)) S[c][s][i] = -INFINITY;
}

// ---- one tile of each cache type ------------------------------------------
// The Q operand of the fp16 matrix cores: q[c][b][0] the high halves, [1] the
// low ones (PACK: [0] alone, high or low by the column).
template <int HD, int CT, bool PACK> struct QHalf {
    static constexpr int NB = (HD + 31) / 32, NH = PACK ? 1 : 2;
    i32x4 q[CT][NB][NH];
};

// Loads a row's dims 32 b + 8 g .. + 7, scales and splits them.  ORDER4: the
// element order of a code dword, (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16.
template <int HD, int CT, bool PACK, bool ORDER4>
__device__ __forceinline__ void load_q16(const AttendArgs &a, const float *row, int c, QHalf<HD, CT, PACK> &Q, float &sc) {
    constexpr int NB = QHalf<HD, CT, PACK>::NB;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    float x[NB][8];
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int d = 32 * b + 8 * g + j;
            x[b][j] = HD % 32 == 0 || d < HD ? row[HD % 32 == 0 ? d : min(d, HD - 1)] * a.qscale : 0.0f;
            top = fmaxf(top, fabsf(x[b][j]));
        }
    top = quarters_max(top);
    const int e = top > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;   // top 2^e in [2^13, 2^14)
    sc = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        _Float16 hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float y = __builtin_amdgcn_ldexpf(x[b][j], ORDER4 && (j & 1) ? e - 4 : e);
            hi[j] = (_Float16)y;
            lo[j] = (_Float16)(y - (float)hi[j]);
        }
        i32x4 h, w;
        if (ORDER4) {
            h = i32x4{ (int)pack2(hi[0], hi[4]), (int)pack2(hi[1], hi[5]), (int)pack2(hi[2], hi[6]), (int)pack2(hi[3], hi[7]) };
            w = i32x4{ (int)pack2(lo[0], lo[4]), (int)pack2(lo[1], lo[5]), (int)pack2(lo[2], lo[6]), (int)pack2(lo[3], lo[7]) };
        } else {
            h = i32x4{ (int)pack2(hi[0], hi[1]), (int)pack2(hi[2], hi[3]), (int)pack2(hi[4], hi[5]), (int)pack2(hi[6], hi[7]) };
            w = i32x4{ (int)pack2(lo[0], lo[1]), (int)pack2(lo[2], lo[3]), (int)pack2(lo[4], lo[5]), (int)pack2(lo[6], lo[7]) };
        }
        if (PACK) Q.q[c][b][0] = (lane & 8) ? w : h;
        else { Q.q[c][b][0] = h; Q.q[c][b][QHalf<HD, CT, PACK>::NH - 1] = w; }
    }
}

__device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16(a), as_f16(b), c, 0, 0, 0);
}

// rows 0 .. 7 and their low halves in columns 8 .. 15, added in both
__device__ __forceinline__ f32x4 add_halves(f32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = xor8_add(v[i]);
    return v;
}

// The hi and lo halves of 8 probabilities, times even / odd by i, as the P
// operand: pairs (s = 0, s = 1) of i.
template <bool PACK>
__device__ __forceinline__ void split_p(const f32x4 (&p)[2], float even, float odd, i32x4 &hi, i32x4 &lo) {
    const bool low = PACK && ((threadIdx.x & 8) != 0);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f32x2 w = f32x2{ p[0][i] * (i & 1 ? odd : even), p[1][i] * (i & 1 ? odd : even) };
        const f16x2 h = __builtin_convertvector(w, f16x2);
        const f32x2 rest = f32x2{ w[0] - (float)h[0], w[1] - (float)h[1] };
        if (PACK) {
            const f32x2 mine = f32x2{ low ? rest[0] : w[0], low ? rest[1] : w[1] };
            hi[i] = dword(__builtin_convertvector(mine, f16x2));
        } else {
            hi[i] = dword(h);
            lo[i] = dword(__builtin_convertvector(rest, f16x2));
        }
    }
}

template <int TYPE, int HD, int CT, bool PACK> struct Tile;

// 4 bits: HD / 16 dwords of codes for keys and for values per lane, and the
// scales of the lane's 8 positions (dword b * 4 + i: positions s = 0, 1)
template <int HD, int CT, bool PACK> struct Tile<EHIP_KV_Q4, HD, CT, PACK> {
    static constexpr int NB = HD / QB, NP = HD / 64;
    i32x4 k[NP], v[NP], ks[NB], vs[NB];
    QHalf<HD, CT, PACK> Q;
    int E = 14;                  // the outputs' sums carry 2^E: 14, or 6 once a value was 4096 and more
    const uint8_t *kb, *vb;
    uint32_t magic;

    __device__ __forceinline__ void init(const AttendArgs &a, int kv) {
        magic = code_magic();
        kb = a.kc + kv * a.head_bytes;
        vb = a.vc + kv * a.head_bytes;
    }
    __device__ __forceinline__ void load_q(const AttendArgs &a, const float *row, int c, float &sc) {
        load_q16<HD, CT, PACK, true>(a, row, c, Q, sc);
    }
    __device__ __forceinline__ void load_k(const AttendArgs &, int tile, int) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const uint8_t *t = kb + (int64_t)tile * kv_tile_bytes(HD);
#pragma unroll
        for (int i = 0; i < NP; i++) k[i] = *reinterpret_cast<const i32x4 *>(t + i * 1024 + lane * 16);
#pragma unroll
        for (int b = 0; b < NB; b++) ks[b] = *reinterpret_cast<const i32x4 *>(t + kv_scale_at(HD, g, b, 0, 0));
    }
    __device__ __forceinline__ void load_v(const AttendArgs &, int tile, int) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const uint8_t *t = vb + (int64_t)tile * kv_tile_bytes(HD);
#pragma unroll
        for (int i = 0; i < NP; i++) v[i] = *reinterpret_cast<const i32x4 *>(t + i * 1024 + lane * 16);
#pragma unroll
        for (int b = 0; b < NB; b++) vs[b] = *reinterpret_cast<const i32x4 *>(t + kv_scale_at(HD, g, b, 0, 0));
    }
    __device__ __forceinline__ void scores(f32x4 (&S)[CT][2]) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int c = 0; c < CT; c++) S[c][s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int e = s * NB + b;
                const i32x4 codes = codes_signed((uint32_t)k[e >> 2][e & 3], magic);
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    f32x4 x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int h = 0; h < QHalf<HD, CT, PACK>::NH; h++) x = mfma16(codes, Q.q[c][b][h], x);
#pragma unroll
                    for (int i = 0; i < 4; i++) S[c][s][i] = __builtin_fmaf(x[i], half_of(ks[b][i], s), S[c][s][i]);
                }
            }
            if (PACK) S[0][s] = add_halves(S[0][s]);
        }
    }
    // whether a value's 16 times too large codes can leave fp16: |d| of 512 and more (not NaN)
    __device__ __forceinline__ bool large() const {
        int any = 0;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) any |= vs[b][i];
        if (!__any((any & 0x6000) == 0x6000 || (any & 0x60000000) == 0x60000000)) return false;   // (no |d| has both exponent bits)
        bool big = false;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                int w = vs[b][i];
                asm volatile("" : "+v"(w));   // (stays in this branch: the exact test is rare)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const int d = w >> (16 * s) & 0x7fff;
                    big |= d >= 0x6000 && d < 0x7c00;
                }
            }
        return __any(big);
    }
    template <bool MASKED>
    __device__ __forceinline__ void values(const AttendArgs &, Rows<HD, CT> &R, f32x4 (&S)[CT][2], int, int, int) {
        if (MASKED) {   // scales that are not finite: their rows' scores are not, and the values zero
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int expo = 0x7c00 << (16 * s);
                    bool bad = false;
#pragma unroll
                    for (int b = 0; b < NB; b++) bad |= (vs[b][i] & expo) == expo;
#pragma unroll
                    for (int b = 0; b < NB; b++) vs[b][i] = bad ? vs[b][i] & (s ? 0xffff : (int)0xffff0000) : vs[b][i];
#pragma unroll
                    for (int c = 0; c < CT; c++) S[c][s][i] = bad && S[c][s][i] != -INFINITY ? __builtin_nanf("") : S[c][s][i];
                }
        }
        const bool big = large();
        softmax_step(R, S, big && E == 14 ? 0x1p-8f : 1.0f);
        if (big) {
            E = 6;
            const f16x2 down = { (_Float16)0x1p-8f, (_Float16)0x1p-8f };
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) vs[b][i] = dword(halves(vs[b][i]) * down);
        }
        const float even = big || E == 14 ? 0x1p14f : 0x1p6f, odd = even * 0.0625f;   // (the codes of odd i are 16 times too large)
        i32x4 hi[CT], lo[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) split_p<PACK>(S[c], even, odd, hi[c], lo[c]);
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            const i32x4 code = codes_signed((uint32_t)v[d >> 2][d & 3], magic);
            i32x4 vh, vl;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f16x2 x = halves(code[i]), y = halves(vs[d >> 1][i]), h = x * y;
                vh[i] = dword(h);
                vl[i] = dword(__builtin_elementwise_fma(x, y, -h));
            }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                R.o[c][d] = mfma16(vl, hi[c], R.o[c][d]);
                if (!PACK) R.o[c][d] = mfma16(vh, lo[c], R.o[c][d]);
                R.o[c][d] = mfma16(vh, hi[c], R.o[c][d]);
            }
        }
    }
    __device__ __forceinline__ int exponent() const { return E; }
};

// The values of a masked tile that are not finite, for the rows that see
// them, one position at a time: o[dim][row] += p v (the tile's products took
// them as zero).  P: the probabilities.
template <int HD, int CT, bool F16, bool PACK>
__device__ __forceinline__ void odd_values(const AttendArgs &a, Rows<HD, CT> &R, f32x4 (&P)[CT][2], int t0, int kv, int last_pos) {
    const int lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    const bool low = PACK && (lane & 8);
#pragma unroll 1
    for (int h = 0; h < 4; h++)
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = t0 + 16 * s + 4 * h + i;
                const int64_t at = (int64_t)min(t, last_pos) * a.kvd + kv * HD;
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    const float p = __shfl(P[c][s][i], h * 16 + l);
                    const bool in = seen(a, R, c, t) && !low;
#pragma unroll
                    for (int d = 0; d < HD / 16; d++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int64_t e = at + 16 * d + 4 * g + r;
                            const float v = F16 ? (float)reinterpret_cast<const _Float16 *>(a.vc)[e] : reinterpret_cast<const float *>(a.vc)[e];
                            if (in && !(fabsf(v) < INFINITY)) R.o[c][d][r] += p * v;   // (not finite: 2^E does not matter)
                        }
                }
            }
}

// fp16: the lanes' pieces of K are 16-byte loads; a V operand is gathered from
// 8 positions (64 bytes of a position to 16 lanes).  Positions past last_pos
// repeat it.
template <int HD, int CT, bool PACK> struct Tile<EHIP_KV_F16, HD, CT, PACK> {
    static constexpr int NB = (HD + 31) / 32;
    i32x4 k[2][NB], v[HD / 16];
    QHalf<HD, CT, PACK> Q;
    const _Float16 *kb, *vb;

    __device__ __forceinline__ void init(const AttendArgs &a, int kv) {
        kb = reinterpret_cast<const _Float16 *>(a.kc) + kv * HD;
        vb = reinterpret_cast<const _Float16 *>(a.vc) + kv * HD;
    }
    __device__ __forceinline__ void load_q(const AttendArgs &a, const float *row, int c, float &sc) {
        load_q16<HD, CT, PACK, false>(a, row, c, Q, sc);
    }
    __device__ __forceinline__ void load_k(const AttendArgs &a, int tile, int last_pos) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const _Float16 *r = kb + (int64_t)min(tile * KV_TILE + 16 * s + (lane & 15), last_pos) * a.kvd;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const bool in = HD % 32 == 0 || 32 * b + 8 * g < HD;   // (HD 48: the last piece's upper half is zero)
                k[s][b] = *reinterpret_cast<const i32x4 *>(r + (in ? 32 * b + 8 * g : 0));
                if (!in) k[s][b] = i32x4{0, 0, 0, 0};
            }
        }
    }
    __device__ __forceinline__ void load_v(const AttendArgs &a, int tile, int last_pos) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const uint16_t *base = reinterpret_cast<const uint16_t *>(vb) + (lane & 15);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = tile * KV_TILE + 4 * g + i;
            const uint16_t *r0 = base + (int64_t)min(t, last_pos) * a.kvd, *r1 = base + (int64_t)min(t + 16, last_pos) * a.kvd;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) v[d][i] = (int)((uint32_t)r0[16 * d] | ((uint32_t)r1[16 * d] << 16));
        }
    }
    __device__ __forceinline__ void scores(f32x4 (&S)[CT][2]) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int c = 0; c < CT; c++) {
                S[c][s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int h = 0; h < QHalf<HD, CT, PACK>::NH; h++) S[c][s] = mfma16(k[s][b], Q.q[c][b][h], S[c][s]);
                if (PACK) S[c][s] = add_halves(S[c][s]);
            }
    }
    template <bool MASKED>
    __device__ __forceinline__ void values(const AttendArgs &a, Rows<HD, CT> &R, f32x4 (&S)[CT][2], int t0, int kv, int last_pos) {
        bool odd = false;
        if (MASKED) {   // what is not finite goes to its own rows only
#pragma unroll
            for (int d = 0; d < HD / 16; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool a0 = (v[d][i] & 0x7c00) == 0x7c00, a1 = (v[d][i] & 0x7c000000) == 0x7c000000;
                    odd |= a0 | a1;
                    if (a0) v[d][i] &= (int)0xffff0000;
                    if (a1) v[d][i] &= 0x0000ffff;
                }
        }
        softmax_step(R, S, 1.0f);
#pragma unroll
        for (int c = 0; c < CT; c++) {
            i32x4 hi, lo;
            split_p<PACK>(S[c], 0x1p14f, 0x1p14f, hi, lo);
#pragma unroll
            for (int d = 0; d < HD / 16; d++) {
                R.o[c][d] = mfma16(v[d], hi, R.o[c][d]);
                if (!PACK) R.o[c][d] = mfma16(v[d], lo, R.o[c][d]);
            }
        }
        if (MASKED && __any(odd)) odd_values<HD, CT, true, PACK>(a, R, S, t0, kv, last_pos);
    }
    __device__ __forceinline__ int exponent() const { return 14; }
};

// fp32, on the fp32 matrix cores (16x16x4): lane quarter g supplies dims
// g HD / 4 .. of K and Q, so its pieces are contiguous; a P.V step contracts
// one position per quarter.
template <int HD, int CT, bool PACK> struct Tile<EHIP_KV_F32, HD, CT, PACK> {
    static_assert(!PACK, "fp32 rows have no low halves");
    static constexpr int NQ = HD / 16;   // 16-byte pieces of a quarter
    f32x4 k[2][NQ], q[CT][NQ];
    float v[HD / 16][2][4];
    const float *kb, *vb;

    __device__ __forceinline__ void init(const AttendArgs &a, int kv) {
        kb = reinterpret_cast<const float *>(a.kc) + kv * HD;
        vb = reinterpret_cast<const float *>(a.vc) + kv * HD;
    }
    __device__ __forceinline__ void load_q(const AttendArgs &a, const float *row, int c, float &sc) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int j = 0; j < NQ; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) q[c][j][r] = row[g * (HD / 4) + 4 * j + r] * a.qscale;
        sc = 1.0f;
    }
    __device__ __forceinline__ void load_k(const AttendArgs &a, int tile, int last_pos) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const float *r = kb + (int64_t)min(tile * KV_TILE + 16 * s + (lane & 15), last_pos) * a.kvd + g * (HD / 4);
#pragma unroll
            for (int j = 0; j < NQ; j++) k[s][j] = *reinterpret_cast<const f32x4 *>(r + 4 * j);
        }
    }
    __device__ __forceinline__ void load_v(const AttendArgs &a, int tile, int last_pos) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float *r = vb + (int64_t)min(tile * KV_TILE + 16 * s + 4 * g + i, last_pos) * a.kvd + (lane & 15);
#pragma unroll
                for (int d = 0; d < HD / 16; d++) v[d][s][i] = r[16 * d];
            }
    }
    __device__ __forceinline__ void scores(f32x4 (&S)[CT][2]) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int c = 0; c < CT; c++) {
                S[c][s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < NQ; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) S[c][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][j][r], q[c][j][r], S[c][s], 0, 0, 0);
            }
    }
    template <bool MASKED>
    __device__ __forceinline__ void values(const AttendArgs &a, Rows<HD, CT> &R, f32x4 (&S)[CT][2], int t0, int kv, int last_pos) {
        bool odd = false;
        if (MASKED) {
#pragma unroll
            for (int d = 0; d < HD / 16; d++)
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool bad = !(fabsf(v[d][s][i]) < INFINITY);
                        odd |= bad;
                        if (bad) v[d][s][i] = 0.0f;
                    }
        }
        softmax_step(R, S, 1.0f);
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int d = 0; d < HD / 16; d++)
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int i = 0; i < 4; i++) R.o[c][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[d][s][i], S[c][s][i], R.o[c][d], 0, 0, 0);
        if (MASKED && __any(odd)) odd_values<HD, CT, false, PACK>(a, R, S, t0, kv, last_pos);
    }
    __device__ __forceinline__ int exponent() const { return 0; }
};

// dims d .. d + 3 of row r of key head kv: o / l
template <int HD>
__device__ __forceinline__ void store_out(const AttendArgs &a, int pos0, int kv, int r, int d, f32x4 o, float l) {
    const int b = r / a.G;
    const float inv = 1.0f / l;
    o *= inv;
    if (pos0 + b < 0 || pos0 + b >= a.ctx) o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float *dst = a.out + (int64_t)b * a.out_stride + (kv * a.G + r % a.G) * HD + d;
    if (a.out_vec) {
        *reinterpret_cast<f32x4 *>(dst) = o;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) dst[j] = o[j];
    }
}

// 16 bytes that workgroups of other XCDs read or have written: agent scope,
// so they pass the XCD's L2 both ways (a release and acquire per workgroup
// instead writes back and drops a whole L2 each time: 512 workgroups 17 us
// where 264 take 12)
__device__ __forceinline__ void put_part(float *p, f32x4 v) {
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    const u64x2 w = __builtin_bit_cast(u64x2, v);
    unsigned long long *q = reinterpret_cast<unsigned long long *>(p);
    __hip_atomic_store(q, w[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(q + 1, w[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 get_part(const float *p) {
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    const unsigned long long *q = reinterpret_cast<const unsigned long long *>(p);
    const u64x2 w = u64x2{ __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), __hip_atomic_load(q + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) };
    return __builtin_bit_cast(f32x4, w);
}

// ---- the kernel ------------------------------------------------------------
// Workgroup (unit, split): unit = (row group, key head), key heads fastest so
// that a key head's workgroups share an XCD's L2; row groups from the last, so
// that the longest start first.  The unit's nsplit workgroups take equal runs
// of its tiles (those without one leave), and the wave w of a workgroup's NW
// the tiles w, w + NW, ... of the run.  The last workgroup of a unit to arrive puts
// the runs together.
template <int TYPE, int HD, int CT, bool PACK, int NW>
__global__ __launch_bounds__(64 * NW) void k_attend(AttendArgs a) {
    constexpr int BR = PACK ? 8 : 16 * CT;        // rows of a unit
    constexpr int LD = HD + 4;                    // floats between rows in LDS
    __shared__ __align__(16) float so[NW][BR][LD];
    __shared__ float sm[NW][BR], sl[NW][BR], ssc[BR], se[NW];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int nunits = gridDim.x / a.nsplit;
    const int unit = blockIdx.x % nunits, split = blockIdx.x / nunits;
    const int kv = unit % a.n_kv, groups = nunits / a.n_kv;
    const int nrows = a.n_tok * a.G, r0 = (groups - 1 - unit / a.n_kv) * BR, r1 = min(r0 + BR, nrows);
    const int pos0 = a.pos ? max(min(*a.pos, a.ctx), -a.n_tok) : a.pos0;
    // rows whose position lies outside the cache (a device position only) give zeros
    const int first_pos = max(pos0 + r0 / a.G, 0), last_pos = min(pos0 + (r1 - 1) / a.G, a.ctx - 1);
    const Tiles T = tiles_seen(first_pos, last_pos, a.window, a.sinks);
    const int ntiles = last_pos < first_pos ? 0 : T.n;
    const int run = max((ntiles + a.nsplit - 1) / a.nsplit, 1), nact = max((ntiles + run - 1) / run, 1);
    if (split >= nact) return;
    const int v1 = min((split + 1) * run, ntiles);

    Rows<HD, CT> R;
    Tile<TYPE, HD, CT, PACK> X;
    X.init(a, kv);
    int vi = split * run + wave;
    if (vi < v1) {
        X.load_k(a, T.at(vi), last_pos);
        X.load_v(a, T.at(vi), last_pos);
    }
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int r = min(r0 + 16 * c + (lane & (PACK ? 7 : 15)), nrows - 1), b = r / a.G;
        R.p[c] = pos0 + b;
        R.m[c] = -INFINITY;
        R.l[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) R.o[c][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        X.load_q(a, a.q + (int64_t)b * a.q_stride + (kv * a.G + r % a.G) * HD, c, R.sc[c]);
    }
    // positions that every row sees: up to that of the first row, and from the last row's window on (or a sink)
    const int all_to = pos0 + r0 / a.G, all_from = a.window > 0 ? pos0 + (r1 - 1) / a.G - a.window + 1 : 0;
    while (vi < v1) {
        const int tile = T.at(vi), t0 = tile * KV_TILE;
        const bool whole = t0 + KV_TILE - 1 <= all_to && (t0 >= all_from || t0 + KV_TILE <= a.sinks);
        f32x4 S[CT][2];
        X.scores(S);
        vi += NW;
        if (vi < v1) X.load_k(a, T.at(vi), last_pos);
        if (whole) {
            X.template values<false>(a, R, S, t0, kv, last_pos);
        } else {
            mask_scores(a, R, S, t0);
            X.template values<true>(a, R, S, t0, kv, last_pos);
        }
        if (vi < v1) X.load_v(a, T.at(vi), last_pos);
    }

    // ---- the workgroup's waves: a row's sums weigh 2^((m - M) sc), M the largest of its m, the output's 2^-E of it
    const int E = X.exponent();
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int r = 16 * c + (lane & (PACK ? 7 : 15));
        const float l = quarters_sum(R.l[c]);
        if (g == 0 && !(PACK && (lane & 8))) {
            sm[wave][r] = R.m[c];
            sl[wave][r] = l;
            ssc[r] = R.sc[c];   // every wave's is the same
        }
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            f32x4 o = R.o[c][d];
            if (PACK) o = add_halves(o);
            if (!(PACK && (lane & 8))) *reinterpret_cast<f32x4 *>(&so[wave][r][16 * d + 4 * g]) = o;
        }
    }
    if (lane == 0) se[wave] = __builtin_amdgcn_ldexpf(1.0f, -E);
    __syncthreads();
    const bool alone = nact == 1;
    const int64_t slot = (int64_t)unit * a.nsplit + split;
    for (int i = tid; i < BR * (HD / 4); i += 64 * NW) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        float M = sm[0][r];
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, sm[w][r]);
        f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = sm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((sm[w][r] - M) * ssc[r]);
            o += *reinterpret_cast<const f32x4 *>(&so[w][r][d]) * (f * se[w]);
            l += sl[w][r] * f;
        }
        if (r0 + r >= nrows) continue;
        if (alone) {
            store_out<HD>(a, pos0, kv, r0 + r, d, o, l);
        } else {
            put_part(a.part + (slot * BR + r) * HD + d, o);
            if (d == 0) put_part(reinterpret_cast<float *>(a.part_ml + slot * BR + r), f32x4{M, l, ssc[r], 0.0f});
        }
    }
    if (alone) return;

    // ---- the unit's workgroups: the last one to arrive joins the runs.  Every
    // wave's partial stores have completed, past its XCD's L2, before the
    // workgroup counts itself, and the last one's loads go past its own.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) s_last = __hip_atomic_fetch_add(a.count + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nact - 1;
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) __hip_atomic_store(a.count + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int64_t base = (int64_t)unit * a.nsplit;
    float *sf = &so[0][0][0];                       // [row][AT_SPLITS]: the runs' weights over the row's sum
    f32x4 *red = reinterpret_cast<f32x4 *>(sf + BR * AT_SPLITS);
    static_assert(BR * AT_SPLITS * 4 + 64 * NW * 16 <= sizeof(so), "the join fits the waves' outputs");
    const int nr = r1 - r0;
    for (int r = wave; r < nr; r += NW) {     // a wave a row, a lane a run: one round trip
        const f32x4 ml = get_part(reinterpret_cast<const float *>(a.part_ml + (base + min(lane, nact - 1)) * BR + r));
        const float m = lane < nact ? ml[0] : -INFINITY, M = wave_max(m);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - M) * ml[2]);
        const float l = wave_sum(lane < nact ? f * ml[1] : 0.0f);
        sf[r * AT_SPLITS + lane] = f;
        if (lane == 0) sl[0][r] = l;
    }
    __syncthreads();
    // an item is four dims of a row; with fewer items than threads they share the runs
    const int items = nr * (HD / 4), parts = max(64 * NW / items, 1);
    for (int i0 = 0; i0 < items; i0 += 64 * NW) {
        const int part = parts > 1 ? tid / items : 0, i = parts > 1 ? tid % items : i0 + tid;
        const int r = min(i, items - 1) / (HD / 4), d = i % (HD / 4) * 4;
        f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (i < items && part < parts) {
            const float *p = a.part + (base * BR + r) * HD + d;
            for (int z = part; z < nact; z += 8 * parts) {
                f32x4 x[8];
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = get_part(p + (int64_t)min(z + j * parts, nact - 1) * (BR * HD));
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float f = z + j * parts < nact ? sf[r * AT_SPLITS + z + j * parts] : 0.0f;
                    o += x[j] * f;
                }
            }
        }
        if (parts > 1) {
            red[tid] = o;
            __syncthreads();
            if (tid >= items) return;
            for (int q = 1; q < parts; q++) o += red[q * items + tid];
        }
        if (i < items) store_out<HD>(a, pos0, kv, r0 + r, d, o, sl[0][r]);
    }
}

// ---- shapes of a launch ------------------------------------------------------
// Rows of a unit: 8 (PACK) or 16 while they hold all the rows of a key head,
// else 32.  Waves of a workgroup: 4; for few rows of a 4-bit cache 8 where 4
// would make more workgroups than CUs, as half the ranges are then joined
// (16 heads of 128 over 8192 positions 15.0 -> 13.4 us; over 2048, which 4
// waves spread over more CUs, 10.0 -> 10.9; an fp32 cache, whose products are
// longer, 54 -> 58 over 32,768).
struct Shape { int br, waves; int64_t units; int nsplit; };
static Shape shape_of(const EhipCache &c, int n_heads, int n_tok, int64_t tiles) {
    Shape s;
    const int64_t rows = (int64_t)n_tok * (n_heads / c.n_kv);
    s.br = c.type != EHIP_KV_F32 && rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    s.units = (rows + s.br - 1) / s.br * c.n_kv;
    s.waves = c.type == EHIP_KV_Q4 && s.br <= 16 && s.units * ((tiles + 3) / 4) > 256 ? 8 : 4;
    // 2048 waves (two to each SIMD), each with at least a tile
    const int64_t all = 2048 / s.waves, want = s.units >= all ? 1 : (all + s.units - 1) / s.units, most = (tiles + s.waves - 1) / s.waves;
    s.nsplit = (int)(want < most ? want : most);
    if (s.nsplit > AT_SPLITS) s.nsplit = AT_SPLITS;
    if (s.nsplit < 1) s.nsplit = 1;
    return s;
}

// Workspace: the units' counters (units that split are fewer than 512), then
// the partial rows and their (maximum, sum).
constexpr int COUNT_BYTES = 2048;
static uint64_t space_bytes(int64_t rows, int hd) { return rows ? COUNT_BYTES + (uint64_t)rows * (4 * hd + 16) : 0; }
static int64_t space_rows(const Shape &s) { return s.nsplit > 1 ? s.units * s.nsplit * s.br : 0; }

template <int TYPE, int HD>
static int attend_go(hipStream_t st, const AttendArgs &a, const Shape &s) {
    const dim3 grid((unsigned)(s.units * s.nsplit)), wg(64 * s.waves);
    if constexpr (TYPE != EHIP_KV_F32) {
        if (s.br == 8 && s.waves == 4) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, true, 4>), grid, wg, 0, st, a);
    }
    if constexpr (TYPE == EHIP_KV_Q4) {
        if (s.br == 8 && s.waves == 8) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, true, 8>), grid, wg, 0, st, a);
        if (s.br == 16 && s.waves == 8) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, false, 8>), grid, wg, 0, st, a);
    }
    if (s.br == 16 && s.waves == 4) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, false, 4>), grid, wg, 0, st, a);
    else if (s.br == 32) hipLaunchKernelGGL((k_attend<TYPE, HD, 2, false, 4>), grid, wg, 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : refuse("ehip_attend: launch: %s", hipGetErrorString(e));
}

// How a call is shared over workgroups; -1 where its workspace does not do.
static int shape_call(const EhipCache &c, const EhipAttend &q, Shape *s) {
    // a host position says how many tiles there are to share
    int64_t tiles = (c.ctx + KV_TILE - 1) / KV_TILE;
    if (!q.pos) tiles = ((int64_t)q.pos0 + q.n_tok + KV_TILE - 1) / KV_TILE;
    if (q.window > 0) {
        const int64_t in = ((int64_t)q.window + q.n_tok + 2 * KV_TILE) / KV_TILE + ((int64_t)q.sinks + KV_TILE - 1) / KV_TILE;
        if (in < tiles) tiles = in;
    }
    *s = shape_of(c, q.n_heads, q.n_tok, tiles);
    const uint64_t need = space_bytes(space_rows(*s), c.head_dim);
    if (need && (!q.workspace || !aligned(q.workspace, 16) || q.workspace_bytes < need))
        return refuse("ehip_attend: the workspace is null, not 16-byte aligned, or smaller than this call's %llu bytes", (unsigned long long)need);
    return 0;
}

int launch_attend(hipStream_t st, const EhipCache &c, const EhipAttend &q) {
    Shape s;
    if (shape_call(c, q, &s)) return -1;
    AttendArgs a{};
    a.q = q.q; a.out = q.out; a.q_stride = q.q_stride; a.out_stride = q.out_stride;
    a.kc = static_cast<const uint8_t *>(c.k); a.vc = static_cast<const uint8_t *>(c.v);
    a.head_bytes = (c.ctx + KV_TILE - 1) / KV_TILE * kv_tile_bytes(c.head_dim);
    a.kvd = c.n_kv * c.head_dim;
    a.n_tok = q.n_tok; a.n_kv = c.n_kv; a.G = q.n_heads / c.n_kv; a.pos0 = q.pos0; a.ctx = (int)c.ctx; a.pos = q.pos;
    a.window = q.window; a.sinks = q.sinks;
    a.qscale = (q.scale != 0.0f ? q.scale : 1.0f / sqrtf((float)c.head_dim)) * 1.4426950408889634f;
    a.nsplit = s.nsplit;
    a.out_vec = aligned(q.out, 16) && q.out_stride % 4 == 0;
    if (s.nsplit > 1) {
        a.count = static_cast<int *>(q.workspace);
        a.part = reinterpret_cast<float *>(static_cast<uint8_t *>(q.workspace) + COUNT_BYTES);
        a.part_ml = reinterpret_cast<float4 *>(a.part + space_rows(s) * c.head_dim);
    }
    switch (c.type * 1000 + c.head_dim) {
        case EHIP_KV_F32 * 1000 + 48: return attend_go<EHIP_KV_F32, 48>(st, a, s);
        case EHIP_KV_F32 * 1000 + 64: return attend_go<EHIP_KV_F32, 64>(st, a, s);
        case EHIP_KV_F32 * 1000 + 128: return attend_go<EHIP_KV_F32, 128>(st, a, s);
        case EHIP_KV_F16 * 1000 + 48: return attend_go<EHIP_KV_F16, 48>(st, a, s);
        case EHIP_KV_F16 * 1000 + 64: return attend_go<EHIP_KV_F16, 64>(st, a, s);
        case EHIP_KV_F16 * 1000 + 128: return attend_go<EHIP_KV_F16, 128>(st, a, s);
        case EHIP_KV_Q4 * 1000 + 64: return attend_go<EHIP_KV_Q4, 64>(st, a, s);
        case EHIP_KV_Q4 * 1000 + 128: return attend_go<EHIP_KV_Q4, 128>(st, a, s);
    }
    return refuse("ehip_attend: head_dim %d", c.head_dim);
}

}  // namespace ehip

using namespace ehip;

static int check_heads(const char *who, const EhipCache *c, int n_heads, int n_tok) {
    if (n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv) return refuse("%s: %d query heads over %d key heads", who, n_heads, c->n_kv);
    if (n_tok < 0 || n_tok > c->ctx || (int64_t)n_tok * (n_heads / c->n_kv) > INT32_MAX / 2)
        return refuse("%s: %d tokens over a cache of %lld", who, n_tok, (long long)c->ctx);
    return 0;
}

extern "C" uint64_t ehip_attend_workspace(const EhipCache *c, int n_heads, int n_tok) {
    const char *who = "ehip_attend_workspace";
    if (check_cache(who, c, false) || check_heads(who, c, n_heads, n_tok)) return 0;
    const int G = n_heads / c->n_kv;
    const int64_t tiles = (c->ctx + KV_TILE - 1) / KV_TILE;
    uint64_t most = 0;
    // on the way to n_tok tokens a unit's rows go through at most three sizes:
    // the largest counts of tokens of each, with either count of waves
    for (int64_t n : { (int64_t)1, (int64_t)8 / G, (int64_t)16 / G, (int64_t)n_tok }) {
        if (n < 1 || n > n_tok) continue;
        const Shape s = shape_of(*c, n_heads, (int)n, tiles);
        const int64_t all = 512, units = s.units < all - 1 ? s.units : all - 1, by_tiles = units * ((tiles + 3) / 4);
        const int64_t wgs = all - 1 + units < by_tiles ? all - 1 + units : by_tiles;
        const uint64_t b = wgs > units ? space_bytes(wgs * s.br, c->head_dim) : 0;
        if (b > most) most = b;
    }
    return most;
}

extern "C" int ehip_attend(const EhipCache *c, const EhipAttend *q, void *stream) {
    const char *who = "ehip_attend";
    if (!q) return refuse("%s: null argument", who);
    if (check_cache(who, c, true) || check_heads(who, c, q->n_heads, q->n_tok)) return -1;
    if (!q->n_tok) return 0;
    const int64_t width = (int64_t)q->n_heads * c->head_dim;
    if (q->n_tok > 1 && (q->q_stride < width || q->out_stride < width))
        return refuse("%s: strides %lld and %lld for rows of %lld floats", who, (long long)q->q_stride, (long long)q->out_stride, (long long)width);
    if (q->window < 0 || q->sinks < 0) return refuse("%s: a window of %d and %d sinks", who, q->window, q->sinks);
    if (!(q->scale - q->scale == 0.0f)) return refuse("%s: scale %g", who, (double)q->scale);
    if (!q->pos && (q->pos0 < 0 || (int64_t)q->pos0 + q->n_tok > c->ctx))
        return refuse("%s: positions %d..%lld exceed the cache of %lld", who, q->pos0, (long long)q->pos0 + q->n_tok - 1, (long long)c->ctx);
    Shape s;
    if (shape_call(*c, *q, &s)) return -1;
    if (!q->q || !q->out) return refuse("%s: null rows", who);
    return launch_attend(static_cast<hipStream_t>(stream), *c, *q);
}
