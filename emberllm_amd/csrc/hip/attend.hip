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
// Probabilities, 4 at most, are split times 2^13 (what a half loses at its
// smallest is 2^-38), which the outputs' sums carry until the end; of the
// four products of halves the smallest, lo.lo below 2^-24 of the whole, is
// left out where it is not free.  fp16 caches are one half already; an fp32
// cache goes through the fp32 matrix cores as it is.
//
// What a row does not see cannot reach it: its scores are selected away, its
// probabilities are zero, and where a zero times what the cache holds would be
// NaN (infinite or NaN values, scales of positions never stored) a 4-bit scale
// becomes zero and the scores of the rows that see it NaN, and an fp16 or fp32
// value's products are made one by one for the rows that see it.
//
// Bound.  A token: the launch, its loads' latencies and, where ranges are joined,
// a round trip past the L2 each for the partial rows, the count and the join (16
// heads of 128 over 4 bits: 60 to 128 positions 5 us, 4096 10.4, 40,000 20.2 for
// 46 MB).  A prompt: the vector units, which make codes into operands, halves
// and exponentials (4 bits, 4096 tokens: 617 instructions a tile and wave, 73% of
// the time; matrix cores 37%, 880 TFLOP/s of fp16 products) and, for fp16, the
// loads' latencies (without them 186 us would be 135).  16 heads of 128 over 4
// bits: 128 tokens 9 us, 512 16, 1024 27, 2048 70, 4096 196; fp16 4096 186.
#include "attend.h"

namespace ehip {

// ---- one tile of each cache type ------------------------------------------
// QL: the rows' Q operands lie in LDS (at ql), where the workgroup's waves share
// them, instead of in registers
template <int TYPE, int HD, int CT, bool PACK, bool QL> struct Tile;

// 4 bits: HD / 16 dwords of codes for keys and for values per lane, and the
// scales of the lane's 8 positions (dword b * 4 + i: positions s = 0, 1)
template <int HD, int CT, bool PACK, bool QL> struct Tile<EHIP_KV_Q4, HD, CT, PACK, QL> {
    static constexpr int NB = HD / QB, NP = HD / 64;
    static constexpr int NH = PACK ? 1 : 2, QN = NB * NH;
    i32x4 k[NP], v[NP], ks[NB], vs[NB];
    i32x4 Q[QL ? 1 : CT][QN];
    const i32x4 *ql;
    int E = 13;                  // the outputs' sums carry 2^E: 13, or 5 once a value was 4096 and more
    const uint8_t *kb, *vb;
    uint32_t magic;

    __device__ __forceinline__ void init(const AttendArgs &a, int kv) {
        magic = code_magic();
        kb = a.kc + kv * a.head_bytes;
        vb = a.vc + kv * a.head_bytes;
    }
    __device__ __forceinline__ void load_q(const AttendArgs &a, const float *row, int c, float &sc, i32x4 *lds) {
        QHalf<HD, PACK> x;
        load_q16<HD, PACK, true>(a, row, x, sc);
#pragma unroll
        for (int b = 0; b < QN / NH; b++)
#pragma unroll
            for (int h = 0; h < NH; h++) {
                if (QL) lds[((c * QN) + b * NH + h) * 64 + (threadIdx.x & 63)] = x.q[b][h];
                else Q[c][b * NH + h] = x.q[b][h];
            }
    }
    __device__ __forceinline__ i32x4 q_at(int c, int b, int h) const {
        return QL ? ql[(c * QN + b * NH + h) * 64 + (threadIdx.x & 63)] : Q[QL ? 0 : c][b * NH + h];
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
                    for (int h = 0; h < NH; h++) x = mfma16(codes, q_at(c, b, h), x);
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
        softmax_step(R, S, big && E == 13 ? 0x1p-8f : 1.0f);
        if (big) {
            E = 5;
            const f16x2 down = { (_Float16)0x1p-8f, (_Float16)0x1p-8f };
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) vs[b][i] = dword(halves(vs[b][i]) * down);
        }
        const float even = big || E == 13 ? 0x1p13f : 0x1p5f, odd = even * 0.0625f;   // (the codes of odd i are 16 times too large)
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
                            const int64_t e = at + HD / 16 * (4 * g + r) + d;
                            const float v = F16 ? (float)reinterpret_cast<const _Float16 *>(a.vc)[e] : reinterpret_cast<const float *>(a.vc)[e];
                            if (in && !(fabsf(v) < INFINITY)) R.o[c][d][r] += p * v;   // (not finite: 2^E does not matter)
                        }
                }
            }
}

// fp16: the lanes' pieces of K and V are 16-byte loads (HD 128): lane l holds the
// dims HD/16 l .. of its quarter's 8 positions, so that the d-th of each make
// the V operand of the dims d, HD/16 + d, ... (one byte permutation a dword;
// gathering 16 dims of a position by 2-byte loads took 205 us where this takes
// 192, 16 heads of 128 and 4096 tokens).  Positions past last_pos repeat it.
template <int HD, int CT, bool PACK, bool QL> struct Tile<EHIP_KV_F16, HD, CT, PACK, QL> {
    static constexpr int NB = (HD + 31) / 32;
    static constexpr int NH = PACK ? 1 : 2, QN = NB * NH;
    static constexpr int ND = HD / 16, NW2 = (ND + 1) / 2;   // dims of a lane, and their dwords
    i32x4 k[2][NB];
    int v[2][4][NW2];
    i32x4 Q[QL ? 1 : CT][QN];
    const i32x4 *ql;
    const _Float16 *kb, *vb;

    __device__ __forceinline__ void init(const AttendArgs &a, int kv) {
        kb = reinterpret_cast<const _Float16 *>(a.kc) + kv * HD;
        vb = reinterpret_cast<const _Float16 *>(a.vc) + kv * HD;
    }
    __device__ __forceinline__ void load_q(const AttendArgs &a, const float *row, int c, float &sc, i32x4 *lds) {
        QHalf<HD, PACK> x;
        load_q16<HD, PACK, false>(a, row, x, sc);
#pragma unroll
        for (int b = 0; b < QN / NH; b++)
#pragma unroll
            for (int h = 0; h < NH; h++) {
                if (QL) lds[((c * QN) + b * NH + h) * 64 + (threadIdx.x & 63)] = x.q[b][h];
                else Q[c][b * NH + h] = x.q[b][h];
            }
    }
    __device__ __forceinline__ i32x4 q_at(int c, int b, int h) const {
        return QL ? ql[(c * QN + b * NH + h) * 64 + (threadIdx.x & 63)] : Q[QL ? 0 : c][b * NH + h];
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
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const _Float16 *r = vb + (int64_t)min(tile * KV_TILE + 16 * s + 4 * g + i, last_pos) * a.kvd + ND * (lane & 15);
                if constexpr (ND == 8) {
                    const i32x4 x = *reinterpret_cast<const i32x4 *>(r);
#pragma unroll
                    for (int n = 0; n < 4; n++) v[s][i][n] = x[n];
                } else if constexpr (ND == 4) {
                    const int2 x = *reinterpret_cast<const int2 *>(r);
                    v[s][i][0] = x.x;
                    v[s][i][1] = x.y;
                } else {
                    static_assert(ND == 3, "three dims: 2-byte aligned");
                    typedef int Int2 __attribute__((aligned(2)));
                    v[s][i][0] = *reinterpret_cast<const Int2 *>(r);
                    v[s][i][1] = reinterpret_cast<const uint16_t *>(r)[2];
                }
            }
    }
    // the V operand of the dims d, ND + d, ...: dword i holds d of positions 4g + i and 16 + 4g + i
    __device__ __forceinline__ i32x4 v_at(int d) const {
        i32x4 x;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (int)__builtin_amdgcn_perm((uint32_t)v[1][i][d / 2], (uint32_t)v[0][i][d / 2], d & 1 ? 0x07060302 : 0x05040100);
        return x;
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
                    for (int h = 0; h < NH; h++) S[c][s] = mfma16(k[s][b], q_at(c, b, h), S[c][s]);
                if (PACK) S[c][s] = add_halves(S[c][s]);
            }
    }
    template <bool MASKED>
    __device__ __forceinline__ void values(const AttendArgs &a, Rows<HD, CT> &R, f32x4 (&S)[CT][2], int t0, int kv, int last_pos) {
        bool odd = false;
        if (MASKED) {   // what is not finite goes to its own rows only
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int n = 0; n < NW2; n++) {
                        int &w = v[s][i][n];
                        const bool a0 = (w & 0x7c00) == 0x7c00, a1 = (w & 0x7c000000) == 0x7c000000;
                        odd |= a0 | a1;
                        w &= (a0 ? 0 : 0xffff) | (a1 ? 0 : (int)0xffff0000);
                    }
        }
        softmax_step(R, S);
        i32x4 hi[CT], lo[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) split_p<PACK>(S[c], 0x1p13f, 0x1p13f, hi[c], lo[c]);
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const i32x4 x = v_at(d);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                if (!PACK) R.o[c][d] = mfma16(x, lo[c], R.o[c][d]);
                R.o[c][d] = mfma16(x, hi[c], R.o[c][d]);
            }
        }
        if (MASKED && __any(odd)) odd_values<HD, CT, true, PACK>(a, R, S, t0, kv, last_pos);
    }
    __device__ __forceinline__ int exponent() const { return 13; }
};

// fp32, on the fp32 matrix cores (16x16x4): lane quarter g supplies dims
// g HD / 4 .. of K and Q, so its pieces are contiguous; a P.V step contracts
// one position per quarter.  Lane l holds the dims HD/16 l .. of V, as for fp16.
template <int HD, int CT, bool PACK, bool QL> struct Tile<EHIP_KV_F32, HD, CT, PACK, QL> {
    static_assert(!PACK, "fp32 rows have no low halves");
    static constexpr int NQ = HD / 16;   // 16-byte pieces of a quarter
    f32x4 k[2][NQ], q[QL ? 1 : CT][NQ];
    float v[HD / 16][2][4];
    const i32x4 *ql;
    const float *kb, *vb;

    __device__ __forceinline__ void init(const AttendArgs &a, int kv) {
        kb = reinterpret_cast<const float *>(a.kc) + kv * HD;
        vb = reinterpret_cast<const float *>(a.vc) + kv * HD;
    }
    static constexpr int QN = NQ;
    __device__ __forceinline__ void load_q(const AttendArgs &a, const float *row, int c, float &sc, i32x4 *lds) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int j = 0; j < NQ; j++) {
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; r++) x[r] = row[g * (HD / 4) + 4 * j + r] * a.qscale;
            if (QL) reinterpret_cast<f32x4 *>(lds)[(c * NQ + j) * 64 + (threadIdx.x & 63)] = x;
            else q[QL ? 0 : c][j] = x;
        }
        sc = 1.0f;
    }
    __device__ __forceinline__ f32x4 q_at(int c, int j) const {
        return QL ? reinterpret_cast<const f32x4 *>(ql)[(c * NQ + j) * 64 + (threadIdx.x & 63)] : q[QL ? 0 : c][j];
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
                const float *r = vb + (int64_t)min(tile * KV_TILE + 16 * s + 4 * g + i, last_pos) * a.kvd + HD / 16 * (lane & 15);
#pragma unroll
                for (int d = 0; d < HD / 16; d++) v[d][s][i] = r[d];
            }
    }
    __device__ __forceinline__ void scores(f32x4 (&S)[CT][2]) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int c = 0; c < CT; c++) {
                S[c][s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < NQ; j++) {
                    const f32x4 x = q_at(c, j);
#pragma unroll
                    for (int r = 0; r < 4; r++) S[c][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][j][r], x[r], S[c][s], 0, 0, 0);
                }
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
        softmax_step(R, S);
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

// ---- the kernel ------------------------------------------------------------
// Q in LDS, where the outputs go at the end, instead of in 64 registers: 32 rows
// of 128 dims then leave room for two waves on a SIMD (16 heads of 128, 4096
// tokens: 4 bits 305 -> 223 us, fp16 270 -> 205).  64 dims have two waves in
// any case (4 bits, 14 heads and 4096 tokens 115 -> 129), and an fp32 tile
// would spill (1024 tokens 61 -> 105).
constexpr bool q_in_lds(int type, int hd, int ct) { return type != EHIP_KV_F32 && hd == 128 && ct == 2; }

// Workgroup (unit, split): unit = (row group, key head), key heads fastest so
// that a key head's workgroups share an XCD's L2; row groups from the last, so
// that the longest start first.  The unit's nsplit workgroups take equal runs
// of its tiles (those without one leave), and the wave w of a workgroup's NW
// the tiles w, w + NW, ... of the run.  The last workgroup of a unit to arrive puts
// the runs together.
template <int TYPE, int HD, int CT, bool PACK, int NW>
__device__ __forceinline__ void attend_body(const AttendArgs &a) {
    constexpr int BR = PACK ? 8 : 16 * CT;        // rows of a unit
    constexpr int LD = HD + 4;                    // floats between rows in LDS
    __shared__ __align__(16) float so[NW][BR][LD];
    __shared__ float sm[NW][BR], sl[NW][BR], ssc[BR], se[NW];
    static_assert(join_floats(BR, 64 * NW) * 4 <= sizeof(so), "the join fits the waves' outputs");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int unit = blockIdx.x, split = blockIdx.y, group = a.n_kv(unit), kv = unit - group * a.n_kv.d;
    const int nrows = a.n_tok * a.G.d, r0 = (a.groups - 1 - group) * BR, r1 = min(r0 + BR, nrows);
    const int pos0 = a.pos ? max(min(*a.pos, a.ctx), -a.n_tok) : a.pos0;
    // rows whose position lies outside the cache (a device position only) give zeros
    const int first_pos = max(pos0 + a.G(r0), 0), last_pos = min(pos0 + a.G(r1 - 1), a.ctx - 1);
    const Tiles T = tiles_seen(first_pos, last_pos, a.window, a.sinks);
    const int ntiles = last_pos < first_pos ? 0 : T.n;
    const int run = max(a.nsplit(ntiles + a.nsplit.d - 1), 1);
    if (split && split * run >= ntiles) return;
    const int v1 = min((split + 1) * run, ntiles);

    Rows<HD, CT> R;
    constexpr bool QL = q_in_lds(TYPE, HD, CT);
    Tile<TYPE, HD, CT, PACK, QL> X;
    static_assert(CT * Tile<TYPE, HD, CT, PACK, QL>::QN * 1024 <= sizeof(so) && CT <= NW, "Q fits the outputs' place");
    i32x4 *ql = reinterpret_cast<i32x4 *>(&so[0][0][0]);
    X.ql = ql;
    X.init(a, kv);
    int vi = split * run + wave;
    if (vi < v1) {
        X.load_k(a, T.at(vi), last_pos);
        X.load_v(a, T.at(vi), last_pos);
    }
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int r = min(r0 + 16 * c + (lane & (PACK ? 7 : 15)), nrows - 1), b = a.G(r);
        R.p[c] = pos0 + b;
        R.m[c] = -INFINITY;
        R.l[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) R.o[c][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (QL && wave != c) continue;
        X.load_q(a, a.q + (int64_t)b * a.q_stride + ((kv - b) * a.G.d + r) * HD, c, R.sc[c], ql);
        if (QL && g == 0) ssc[16 * c + lane] = R.sc[c];
    }
    if (QL) {
        lds_barrier();
#pragma unroll
        for (int c = 0; c < CT; c++) R.sc[c] = ssc[16 * c + (lane & 15)];
    }
    // positions that every row sees: up to that of the first row, and from the last row's window on (or a sink)
    const int all_to = pos0 + a.G(r0), all_from = a.window > 0 ? pos0 + a.G(r1 - 1) - a.window + 1 : 0;
    while (vi < v1) {
        if (QL) asm volatile("" ::: "memory");   // (Q stays in LDS: the compiler would keep it in registers over the loop)
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
    if (QL) lds_barrier();   // (every wave is past its last reads of Q)

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
            if (PACK && (lane & 8)) continue;
            if (TYPE == EHIP_KV_Q4) {
                *reinterpret_cast<f32x4 *>(&so[wave][r][16 * d + 4 * g]) = o;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) so[wave][r][HD / 16 * (4 * g + i) + d] = o[i];
            }
        }
    }
    if (lane == 0) se[wave] = __builtin_amdgcn_ldexpf(1.0f, -E);
    __syncthreads();
    const bool alone = ntiles <= run;
    const Parts<HD, BR> mine(a, (int64_t)unit * a.nsplit.d + split, 1);
#pragma unroll
    for (int i0 = 0; i0 < BR * (HD / 4); i0 += 64 * NW) {
        const int i = i0 + tid, r = i / (HD / 4), d = i % (HD / 4) * 4;
        if (BR * (HD / 4) % (64 * NW) && r >= BR) break;
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
            mine.rows.put((r * HD + d) * 4, o);
            if (d == 0) mine.ml.put(r * 16, f32x4{M, l, ssc[r], 0.0f});
        }
    }
    if (alone) return;

    join_runs<HD, BR, 64 * NW>(a, unit, (ntiles + run - 1) / run, r0, r1, pos0, kv, &so[0][0][0]);
}

template <int TYPE, int HD, int CT, bool PACK, int NW>
__global__ __launch_bounds__(64 * NW) void k_attend(AttendArgs a) { attend_body<TYPE, HD, CT, PACK, NW>(a); }
// the same held to the registers of two waves on a SIMD
template <int TYPE, int HD, int CT, bool PACK, int NW>
__global__ __launch_bounds__(64 * NW, 2) void k_attend_two(AttendArgs a) { attend_body<TYPE, HD, CT, PACK, NW>(a); }

// ---- shapes of a launch ------------------------------------------------------
// Rows of a unit: 8 (PACK) or 16 while they hold all the rows of a key head,
// then 32; over an fp32 cache ATTEND_ROWS (attend_rows.hip), if that makes four
// tiles and more for each workgroup that the GPU holds: 16 heads of 128, whole
// prompts, 512 tokens 27 us (48 there), 1024 61 (57), 2048 183 (120).  Waves of
// a workgroup: 4; for few rows of a 4-bit cache 8 where 4 would make more
// workgroups than CUs, as half the ranges are then joined (16 heads of 128 over
// 8192 positions 15.0 -> 13.4 us; over 2048, which 4 waves spread over more
// CUs, 10.0 -> 10.9; an fp32 cache, whose products are longer, 54 -> 58 over
// 32,768).
struct Shape { int br, waves; int64_t units; int nsplit, run; };
constexpr int SLOTS = 512;       // workgroups of four waves that the GPU holds, two waves to each SIMD
constexpr int MAX_UNITS = 2 * SLOTS;   // units from which on none is split

static int tiles_of_rows(int64_t pos0, int64_t r0, int64_t r1, int G, int window, int sinks) {
    return tiles_seen((int)(pos0 + r0 / G), (int)(pos0 + (r1 - 1) / G), window, sinks).n;
}

// Into how many ranges a unit's tiles are cut, each for a workgroup: the least
// time, counted in fifths of what a wave takes for a tile by itself (7 beside a
// second wave on its SIMD).  A workgroup's start and end take three tiles, a join
// two (16 heads of 128 over 4 bits: a range of one tile per wave 8.5 us, of two
// 10.6, of five 16.3, one tile and a join 12.9).  23 tokens at 517, 17 tiles of
// 16 units: 5 ranges 13.4 us, one 16.3; a prompt of 700, up to 22 tiles of 352
// units: one range 19.4, two 26.4; 300 tokens at 4000, 135 of 152: three 46.5,
// four, which do not run at once, 54.6.
// slots: workgroups that the GPU holds at a time.
static int ranges(int64_t units, int tiles, int waves, int64_t slots) {
    int64_t best = 0;
    int n = 1;
    for (int z = 1; z <= AT_SPLITS; z++) {
        const int64_t wgs = units * z, k = ((tiles + z - 1) / z + waves - 1) / waves;
        if (z > 1 && (wgs > 2 * slots || tiles <= (z - 1) * waves)) break;
        const int64_t cost = (wgs + slots - 1) / slots * (15 + k * (2 * wgs > slots ? 7 : 5)) + (z > 1 ? 10 : 0);
        if (z == 1 || cost < best) {
            best = cost;
            n = z;
        }
    }
    return n;
}

static int few_rows(int type, int64_t rows) { return type != EHIP_KV_F32 && rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }

// q: its n_tok, n_heads, window and sinks; positions: q.pos0, or any (q.pos)
static Shape shape_of(const EhipCache &c, const EhipAttend &q) {
    Shape s{};
    const int G = q.n_heads / c.n_kv;
    const int64_t rows = (int64_t)q.n_tok * G;
    const int64_t pos0 = q.pos ? c.ctx - q.n_tok : q.pos0;
    s.br = few_rows(c.type, rows);
    int tiles = 0;
    int64_t all = 0;             // many rows: tiles of all units
    if (c.type == EHIP_KV_F32 && rows >= ATTEND_ROWS) {
        for (int64_t r = 0; r < rows; r += ATTEND_ROWS) {   // (behind a window a last group of few rows sees less than one before)
            const int n = tiles_of_rows(pos0, r, r + ATTEND_ROWS < rows ? r + ATTEND_ROWS : rows, G, q.window, q.sinks);
            all += (int64_t)n * c.n_kv;
            if (n > tiles) tiles = n;
        }
        if (all >= 4 * SLOTS) s.br = ATTEND_ROWS;
    }
    const int64_t groups = (rows + s.br - 1) / s.br;
    s.units = groups * c.n_kv;
    s.waves = 4;
    if (s.br == ATTEND_ROWS) {
        // ranges of a slot's average, of at least 8 tiles (a range's start and
        // its join take the time of about four)
        int64_t run = (all + SLOTS - 1) / SLOTS;
        if (run < 8) run = 8;
        // many units fill the slots by themselves, and a rest of less than a
        // quarter is not worth a join
        if (s.units >= MAX_UNITS || tiles <= run + run / 4) run = tiles;
        s.nsplit = (int)((tiles + run - 1) / run);
        s.run = q.pos ? 0 : (int)run;
    } else {
        tiles = tiles_of_rows(pos0, (groups - 1) * s.br, rows, G, q.window, q.sinks);
        if (c.type == EHIP_KV_Q4 && s.br <= 16 && s.units * ((tiles + 3) / 4) > 256) s.waves = 8;
        // (32 rows of 128 dims over fp32 take more than half of a SIMD's registers)
        const int simd_waves = c.type == EHIP_KV_F32 && c.head_dim == 128 && s.br == 32 ? 1 : 2;
        s.nsplit = ranges(s.units, tiles, s.waves, SLOTS / 2 * simd_waves * 4 / s.waves);
    }
    if (s.nsplit > AT_SPLITS) {
        s.nsplit = AT_SPLITS;
        if (s.run) s.run = (tiles + AT_SPLITS - 1) / AT_SPLITS;
    }
    if (s.nsplit < 1) s.nsplit = 1;
    return s;
}

// Workspace: the units' counters (units that split are fewer than MAX_UNITS),
// then the partial rows and their (maximum, sum, scale).
constexpr int COUNT_BYTES = 4 * MAX_UNITS;
static uint64_t space_bytes(int64_t rows, int hd) { return rows ? COUNT_BYTES + (uint64_t)rows * (4 * hd + 16) : 0; }
static int64_t space_rows(const Shape &s) { return s.nsplit > 1 ? s.units * s.nsplit * s.br : 0; }

template <int TYPE, int HD>
static int attend_go(hipStream_t st, const AttendArgs &a, const Shape &s) {
    const dim3 grid((unsigned)s.units, (unsigned)s.nsplit), wg(64 * s.waves);
    if constexpr (TYPE != EHIP_KV_F32) {
        if (s.br == 8 && s.waves == 4) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, true, 4>), grid, wg, 0, st, a);
    }
    if constexpr (TYPE == EHIP_KV_Q4) {
        if (s.br == 8 && s.waves == 8) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, true, 8>), grid, wg, 0, st, a);
        if (s.br == 16 && s.waves == 8) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, false, 8>), grid, wg, 0, st, a);
    }
    if (s.br == 16 && s.waves == 4) hipLaunchKernelGGL((k_attend<TYPE, HD, 1, false, 4>), grid, wg, 0, st, a);
    if (s.br == 32) {
        if constexpr (q_in_lds(TYPE, HD, 2)) hipLaunchKernelGGL((k_attend_two<TYPE, HD, 2, false, 4>), grid, wg, 0, st, a);
        else hipLaunchKernelGGL((k_attend<TYPE, HD, 2, false, 4>), grid, wg, 0, st, a);
    }
    if (TYPE == EHIP_KV_F32 && s.br == ATTEND_ROWS) launch_attend_rows(st, HD, grid, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : refuse("ehip_attend: launch: %s", hipGetErrorString(e));
}

// How a call is shared over workgroups; -1 where its workspace does not do.
static int shape_call(const EhipCache &c, const EhipAttend &q, Shape *s) {
    *s = shape_of(c, q);
    if (s->units * 64 * s->waves > UINT32_MAX) return refuse("ehip_attend: %d tokens of %d heads are more than a launch's threads", q.n_tok, q.n_heads);
    const uint64_t need = space_bytes(space_rows(*s), c.head_dim);
    if (need && (!q.workspace || !aligned(q.workspace, 16) || q.workspace_bytes < need))
        return refuse("ehip_attend: the workspace is null, not 16-byte aligned, or smaller than this call's %llu bytes", (unsigned long long)need);
    return 0;
}

int launch_attend(hipStream_t st, const EhipCache &c, const EhipAttend &q) {
    Shape s;
    if (shape_call(c, q, &s)) return -1;
    if (!q.q || !q.out) return refuse("ehip_attend: null rows");
    AttendArgs a{};
    a.q = q.q; a.out = q.out; a.q_stride = q.q_stride; a.out_stride = q.out_stride;
    a.kc = static_cast<const uint8_t *>(c.k); a.vc = static_cast<const uint8_t *>(c.v);
    a.head_bytes = (c.ctx + KV_TILE - 1) / KV_TILE * kv_tile_bytes(c.head_dim);
    a.kvd = c.n_kv * c.head_dim;
    a.n_tok = q.n_tok; a.groups = (int)(s.units / c.n_kv); a.pos0 = q.pos0; a.ctx = (int)c.ctx; a.pos = q.pos;
    a.window = q.window; a.sinks = q.sinks;
    a.qscale = (q.scale != 0.0f ? q.scale : 1.0f / sqrtf((float)c.head_dim)) * 1.4426950408889634f;
    a.n_kv.set(c.n_kv); a.G.set(q.n_heads / c.n_kv); a.nsplit.set(s.nsplit);
    a.run = s.run;
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
    // On the way to n_tok tokens a unit's rows go through at most four sizes;
    // the largest count of tokens of each, U units of it and T tiles at most.
    // Few rows: at most 2 SLOTS workgroups, of at least a tile to each of four
    // waves.  Many: tiles per unit grow along a prompt ever more slowly, so the
    // average is at least half of the most, and with it a range: U (2 SLOTS / U +
    // 1), and U more for rounding.
    auto bound = [&](int64_t rows, int br) {
        const bool many = br == ATTEND_ROWS;
        const int64_t units = (rows + br - 1) / br * c->n_kv, U = units < MAX_UNITS ? units : MAX_UNITS;
        const int64_t wgs = many ? 2 * SLOTS + 2 * U : 2 * SLOTS, by_tiles = U * ((tiles + (many ? 7 : 3)) / (many ? 8 : 4));
        const uint64_t b = by_tiles > U ? space_bytes((wgs < by_tiles ? wgs : by_tiles) * br, c->head_dim) : 0;
        if (b > most) most = b;
    };
    const int64_t all = (int64_t)n_tok * G;
    for (int64_t rows : { (int64_t)G, (int64_t)8 / G * G, (int64_t)16 / G * G, all })
        if (rows > 0 && rows <= all) bound(rows, few_rows(c->type, rows));
    if (c->type == EHIP_KV_F32 && all >= ATTEND_ROWS) bound(all, ATTEND_ROWS);
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
    return launch_attend(static_cast<hipStream_t>(stream), *c, *q);
}
