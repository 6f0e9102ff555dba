// attend_rows.hip — attention of many rows over an fp32 cache (prompts): the
// mathematics of attend.hip with the cache, too, as fp16 halves, a tile of 32
// positions made ready once per workgroup.
//
// A workgroup takes 128 rows of one key head, 32 for each of its four waves,
// and a run of their tiles.  The waves split a tile together, each a quarter
// of it, into LDS fragments that lie as the matrix cores' operands (64 lanes x
// 16 bytes, so every read and write of a wave is 1 KB without bank conflicts):
//   K   [hi, lo][half s][32 dims b]: lane (l, g) holds position 16 s + l, dims
//       32 b + 8 g .. + 7 (in the place of lane l ^ (g + 4 (b & 1)): eight lanes of
//       a staging wave hold one position, whose pieces would share their banks)
//   V   [hi, lo][16 dims d]: lane (l, g) holds dim 16 d + l, positions
//       16 s + 4 g + i in the order (i, s) of the probabilities
// while the next tile's rows are on their way to registers, and the tile after a
// barrier is used by all four.
//
// Halves.  x 2^e as hi + lo like q's: e per key (its largest element into [2^13,
// 2^14), undone in the scores), and for V per wave's dims (by the largest element
// so far, carried by the outputs' sums).  Of the four products of halves lo.lo,
// below 2^-22 of the largest terms, is left out: scores and outputs are three
// products on the fp16 matrix cores, which take sixteen times the fp32 ones' rate.
//
// Bound: the latencies of a wave's chain of products, maximum, exponentials and
// halves, which two waves on a SIMD hide in part; the vector units issue 56% of
// the time, the matrix cores work 32% of it.  Whole prompts, 16 heads over 8 of
// 128 dims: 1024 tokens 57 us (attend.hip 61), 2048 120 (183), 4096 281 (637: 245
// TFLOP/s of fp32 work, 734 of fp16 products); behind a window of 1024 with 4 sinks
// 139; 9 over 3 of 64: 2048 62 (78), 4096 138 (221).  A cache of 16 bits or 4 needs
// no splitting that is worth a barrier: attend.hip was as fast with them (4096
// tokens 211 and 223 us at 128 dims, this kernel's form for them 212 and 228).
#include "attend.h"

namespace ehip {

// waves; row tiles and rows of a wave; rows
constexpr int AR_NW = 4, AR_CT = 2, AR_WR = 16 * AR_CT, AR_BR = AR_NW * AR_WR;
static_assert(AR_BR == ATTEND_ROWS, "rows of a unit");

// One staged tile in LDS
template <int HD> struct Staged {
    static constexpr int NB = (HD + 31) / 32, ND = HD / 16;
    i32x4 k[2][2 * NB][64];
    i32x4 v[2][ND][64];
    float ks[4][4][2];   // a key's power of two, undone: [g][i][s]
    i32x4 bad;           // positions (bits) whose values are not all finite, by staging wave
    i32x4 vexp;          // V's power of two, by staging wave
};

// bits 16 s + 4 g + i of the positions where bad[s][i] holds in any lane of quarter g
__device__ __forceinline__ uint32_t position_bits(const bool (&bad)[2][4]) {
    uint32_t bits = 0;
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint64_t m = __ballot(bad[s][i]);
#pragma unroll
            for (int g = 0; g < 4; g++) bits |= (m >> (16 * g) & 0xffff) ? 1u << (16 * s + 4 * g + i) : 0u;
        }
    return bits;
}

template <int HD> struct Stager {
    using S = Staged<HD>;
    static constexpr int NB = S::NB, NP = (HD / 8 + 7) / 8, NV = (S::ND + AR_NW - 1) / AR_NW;
    const float *kb, *vb;
    f32x4 kr[NP][2];             // lane (key 8 wave + lane / 8, pieces of 8 dims lane % 8, + 8)
    float vr[NV][2][4];
    float vtop = 0.0f;           // the largest finite |V| of this wave's dims so far

    __device__ __forceinline__ void init(const AttendArgs &a, int kv) {
        kb = reinterpret_cast<const float *>(a.kc) + kv * HD;
        vb = reinterpret_cast<const float *>(a.vc) + kv * HD;
    }
    __device__ __forceinline__ void load(const AttendArgs &a, int tile, int last_pos) {
        const int lane = threadIdx.x & 63, wave = wave_id(), g = lane >> 4, l = lane & 15;
        const float *kp = kb + (int64_t)min(tile * KV_TILE + 8 * wave + (lane >> 3), last_pos) * a.kvd;
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const int p = (lane & 7) + 8 * j;
            const float *src = kp + 8 * (HD % 64 == 0 ? p : min(p, HD / 8 - 1));
            kr[j][0] = *reinterpret_cast<const f32x4 *>(src);
            kr[j][1] = *reinterpret_cast<const f32x4 *>(src + 4);
        }
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float *r = vb + (int64_t)min(tile * KV_TILE + 16 * s + 4 * g + i, last_pos) * a.kvd + l;
#pragma unroll
                for (int j = 0; j < NV; j++) vr[j][s][i] = r[16 * (S::ND % AR_NW == 0 ? wave * NV + j : min(wave * NV + j, S::ND - 1))];
            }
    }
    __device__ __forceinline__ void put(S &o, bool masked) {
        const int lane = threadIdx.x & 63, wave = wave_id();
        // ---- keys: hi and lo of the row times 2^e
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < NP; j++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < 4; r++) top = fmaxf(top, fabsf(kr[j][h][r]));
        top = max8(top);
        const int e = top > 0.0f && top < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
        const int key = 8 * wave + (lane >> 3), s = key / 16, l = key % 16;
        if ((lane & 7) == 0) o.ks[l / 4][l % 4][s] = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
        for (int j = 0; j < NP; j++) {
            const int p = (lane & 7) + 8 * j;
            i32x4 hi, lo;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const f32x2 x = f32x2{ __builtin_amdgcn_ldexpf(kr[j][r / 2][2 * (r % 2)], e), __builtin_amdgcn_ldexpf(kr[j][r / 2][2 * (r % 2) + 1], e) };
                const f16x2 h = __builtin_convertvector(x, f16x2);
                hi[r] = dword(h);
                lo[r] = dword(__builtin_convertvector(f32x2{ x[0] - (float)h[0], x[1] - (float)h[1] }, f16x2));
            }
            if (HD % 32 != 0 && 8 * p >= HD) hi = lo = i32x4{0, 0, 0, 0};   // (HD 48: the last fragment's upper half)
            if (HD % 64 == 0 || p < 4 * NB) {
                o.k[0][s * NB + p / 4][(p % 4) * 16 + (l ^ (p & 7))] = hi;
                o.k[1][s * NB + p / 4][(p % 4) * 16 + (l ^ (p & 7))] = lo;
            }
        }
        // ---- values
        uint32_t bits = 0;
        bool bad[2][4], any = false;
        float big = 0.0f;
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                bad[s2][i] = false;
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    const bool b = !(fabsf(vr[j][s2][i]) < INFINITY);
                    bad[s2][i] |= b;
                    if (masked && b) vr[j][s2][i] = 0.0f;
                    big = fmaxf(big, b ? 0.0f : fabsf(vr[j][s2][i]));
                }
                any |= bad[s2][i];
            }
        if (masked && __any(any)) bits = position_bits(bad);
        vtop = fmaxf(vtop, wave_max(big));
        const int x = vtop > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(vtop) : 0;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            i32x4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f32x2 y = f32x2{ __builtin_amdgcn_ldexpf(vr[j][0][i], x), __builtin_amdgcn_ldexpf(vr[j][1][i], x) };
                const f16x2 h = __builtin_convertvector(y, f16x2);
                hi[i] = dword(h);
                lo[i] = dword(__builtin_convertvector(f32x2{ y[0] - (float)h[0], y[1] - (float)h[1] }, f16x2));
            }
            if (S::ND % AR_NW == 0 || wave * NV + j < S::ND) {
                o.v[0][wave * NV + j][lane] = hi;
                o.v[1][wave * NV + j][lane] = lo;
            }
        }
        if (lane == 0) {
            reinterpret_cast<int *>(&o.bad)[wave] = (int)bits;
            reinterpret_cast<int *>(&o.vexp)[wave] = x;
        }
    }
};

// Workgroup (unit, split) as in attend.hip, with ranges of a.run tiles where the
// host knows the positions: a range is then about the average of what a slot of
// the GPU (two workgroups to a CU) has to do, units of more tiles are cut, and
// the order (first ranges, longest first, then the rests of the cut units) puts
// the longest rests behind the shortest units (16 heads of 128, 4096 tokens:
// whole units, whose last ones take twice the average, kept 1.2 waves on a SIMD).
template <int HD>
__global__ __launch_bounds__(64 * AR_NW, 2) void k_attend_rows(AttendArgs a) {
    using S = Staged<HD>;
    constexpr int NB = S::NB, ND = S::ND, CT = AR_CT, NV = (ND + AR_NW - 1) / AR_NW;
    constexpr size_t JOIN = join_floats(AR_BR, 64 * AR_NW) * 4, BYTES = 2 * sizeof(S) > JOIN ? 2 * sizeof(S) : JOIN;
    __shared__ __align__(16) uint8_t lds[BYTES];
    S *buf = reinterpret_cast<S *>(lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), g = lane >> 4, l = lane & 15;
    const int unit = blockIdx.x, split = blockIdx.y, group = a.n_kv(unit), kv = unit - group * a.n_kv.d;
    const int nrows = a.n_tok * a.G.d, r0 = (a.groups - 1 - group) * AR_BR, r1 = min(r0 + AR_BR, nrows);
    const int pos0 = a.pos ? max(min(*a.pos, a.ctx), -a.n_tok) : a.pos0;
    const int first_pos = max(pos0 + a.G(r0), 0), last_pos = min(pos0 + a.G(r1 - 1), a.ctx - 1);
    const Tiles T = tiles_seen(first_pos, last_pos, a.window, a.sinks);
    const int ntiles = last_pos < first_pos ? 0 : T.n;
    const int run = max(max(a.nsplit(ntiles + a.nsplit.d - 1), a.run), 1);
    if (split && split * run >= ntiles) return;
    const int v0 = split * run, v1 = min(v0 + run, ntiles);

    Stager<HD> X;
    X.init(a, kv);
    if (v0 < v1) X.load(a, T.at(v0), last_pos);

    // ---- this wave's rows
    const int w0 = r0 + AR_WR * wave, w1 = min(w0 + AR_WR, nrows);
    Rows<HD, CT> R;
    QHalf<HD, false> Q[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int r = min(w0 + 16 * c + l, nrows - 1), b = a.G(r);
        R.p[c] = pos0 + b;
        R.m[c] = -INFINITY;
        R.l[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++) R.o[c][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        load_q16<HD, false, false>(a, a.q + (int64_t)b * a.q_stride + ((kv - b) * a.G.d + r) * HD, Q[c], R.sc[c]);
    }
    // positions that all rows of the workgroup, and of the wave, see (or a sink's), and that any of the wave sees
    const int all_to = pos0 + a.G(r0), all_from = a.window > 0 ? pos0 + a.G(r1 - 1) - a.window + 1 : 0;
    const int mine_to = pos0 + a.G(w0), mine_last = w0 < nrows ? pos0 + a.G(w1 - 1) : -1;
    const int mine_from = a.window > 0 ? mine_last - a.window + 1 : 0, mine_first = a.window > 0 ? mine_to - a.window + 1 : 0;
    auto masked = [&](int t0) { return !(t0 + KV_TILE - 1 <= all_to && (t0 >= all_from || t0 + KV_TILE <= a.sinks)); };
    i32x4 vexp = { 0, 0, 0, 0 };   // the power of two of V that the output's sums carry, by staging wave's dims

    if (v0 < v1) {
        X.put(buf[0], masked(T.at(v0) * KV_TILE));
        if (v0 + 1 < v1) X.load(a, T.at(v0 + 1), last_pos);
    }
    lds_barrier();
    for (int vi = v0; vi < v1; vi++) {
        const int t0 = T.at(vi) * KV_TILE;
        const S &t = buf[(vi - v0) & 1];
        const bool use = t0 <= mine_last && (t0 + KV_TILE > mine_first || t0 < a.sinks);   // (uniform in the wave)
        f32x4 P[CT][2];
        i32x4 bad, x;
        if (use) {
            bad = t.bad;
            x = t.vexp;
#pragma unroll
            for (int s = 0; s < 2; s++) {
#pragma unroll
                for (int c = 0; c < CT; c++) P[c][s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const int at = lane ^ (g + 4 * (b & 1));
                    const i32x4 kh = t.k[0][s * NB + b][at];
                    const i32x4 kl = t.k[1][s * NB + b][at];
#pragma unroll
                    for (int c = 0; c < CT; c++) {
                        P[c][s] = mfma16(kh, Q[c].q[b][1], P[c][s]);
                        P[c][s] = mfma16(kl, Q[c].q[b][0], P[c][s]);
                        P[c][s] = mfma16(kh, Q[c].q[b][0], P[c][s]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int c = 0; c < CT; c++) P[c][s][i] *= t.ks[g][i][s];
            }
        }
        if (vi + 1 < v1) {   // the next tile, into the buffer that every wave has left
            X.put(buf[(vi + 1 - v0) & 1], masked(T.at(vi + 1) * KV_TILE));
            if (vi + 2 < v1) X.load(a, T.at(vi + 2), last_pos);
        }
        if (use) {
            if (!(t0 + KV_TILE - 1 <= mine_to && (t0 >= mine_from || t0 + KV_TILE <= a.sinks))) mask_scores(a, R, P, t0);
            const int odd = bad[0] | bad[1] | bad[2] | bad[3] | (x[0] ^ vexp[0]) | (x[1] ^ vexp[1]) | (x[2] ^ vexp[2]) | (x[3] ^ vexp[3]);
            if (__builtin_amdgcn_readfirstlane(odd)) {   // (the same in all lanes)
                // positions with values that are not finite, in a tile that some rows do not see wholly
                const int bits = bad[0] | bad[1] | bad[2] | bad[3];
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if ((bits >> (16 * s + 4 * g + i) & 1) && P[c][s][i] != -INFINITY) P[c][s][i] = __builtin_nanf("");
                // and V's powers of two that have changed
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int r = 0; r < 4; r++) R.o[c][d][r] = __builtin_amdgcn_ldexpf(R.o[c][d][r], x[d / NV] - vexp[d / NV]);
                vexp = x;
            }
            softmax_step(R, P);
            i32x4 hi[CT], lo[CT];
#pragma unroll
            for (int c = 0; c < CT; c++) split_p<false>(P[c], 0x1p13f, 0x1p13f, hi[c], lo[c]);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const i32x4 vh = t.v[0][d][lane], vl = t.v[1][d][lane];
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    R.o[c][d] = mfma16(vl, hi[c], R.o[c][d]);
                    R.o[c][d] = mfma16(vh, lo[c], R.o[c][d]);
                    R.o[c][d] = mfma16(vh, hi[c], R.o[c][d]);
                }
            }
        }
        lds_barrier();
    }

    const bool alone = ntiles <= run;
    const Parts<HD, AR_BR> mine_parts(a, (int64_t)unit * a.nsplit.d + split, 1);
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const float sum = quarters_sum(R.l[c]);
        const int r = w0 + 16 * c + l;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            f32x4 o;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = __builtin_amdgcn_ldexpf(R.o[c][d][i], -13 - vexp[d / NV]);
            if (r >= nrows) continue;
            if (alone) store_out<HD>(a, pos0, kv, r, 16 * d + 4 * g, o, sum);
            else mine_parts.rows.put(((r - r0) * HD + 16 * d + 4 * g) * 4, o);
        }
        if (!alone && g == 0 && r < nrows) mine_parts.ml.put((r - r0) * 16, f32x4{R.m[c], sum, R.sc[c], 0.0f});
    }
    if (!alone) join_runs<HD, AR_BR, 64 * AR_NW>(a, unit, (ntiles + run - 1) / run, r0, r1, pos0, kv, reinterpret_cast<float *>(lds));
}

void launch_attend_rows(hipStream_t st, int hd, dim3 grid, const AttendArgs &a) {
    const dim3 wg(64 * AR_NW);
    if (hd == 48) hipLaunchKernelGGL((k_attend_rows<48>), grid, wg, 0, st, a);
    if (hd == 64) hipLaunchKernelGGL((k_attend_rows<64>), grid, wg, 0, st, a);
    if (hd == 128) hipLaunchKernelGGL((k_attend_rows<128>), grid, wg, 0, st, a);
}

}  // namespace ehip
