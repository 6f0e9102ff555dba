// attend.h — what the two attention kernels share (attend.hip, and
// attend_rows.hip for many rows over an fp32 cache): their arguments, the
// running softmax, fp16 halves, the joining of ranges.  The mathematics is
// described in attend.hip.
#pragma once
#include "session.h"

namespace ehip {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// x / d for 0 <= x < 2^31, as x * m >> shift with m = ceil(2^(31 + l) / d), l =
// ceil(log2 d): m d exceeds 2^(31 + l) by less than d <= 2^l, so x of that less
// than 1 / d.  (A division by a number that is not constant takes 25
// instructions, and a short launch is mostly its first and last microseconds.)
struct Div {
    uint32_t d, m, shift;
    void set(uint32_t by) {
        uint32_t l = 0;
        while ((1ull << l) < by) l++;
        d = by;
        shift = 31 + l;
        m = (uint32_t)(((1ull << shift) + by - 1) / by);
    }
    __device__ __forceinline__ int operator()(int x) const { return (int)((uint64_t)(uint32_t)x * m >> shift); }
};

struct AttendArgs {
    const float *q;
    float *out;
    int64_t q_stride, out_stride;
    const uint8_t *kc, *vc;
    int64_t head_bytes;          // 4 bits: bytes of a key head's tiles
    int kvd;                     // others: elements of a position
    int n_tok, groups, pos0, ctx; // groups: of rows
    Div n_kv, G, nsplit;          // key heads; query heads of each; workgroups that share a row group's positions
    const int *pos;
    int out_vec;                 // out rows take 16-byte stores
    int window, sinks;
    float qscale;                // scale * log2(e)
    int run;                     // tiles of a range (0: a unit's tiles over nsplit)
    float *part;                 // [unit][nsplit][rows][HD], then float4 [unit][nsplit][rows]; unit = (row group, key head)
    float4 *part_ml;             // a row's maximum, sum and score scale
    int *count;                  // [unit]: workgroups of the unit that are done; zero between launches
};

constexpr int AT_SPLITS = 64;    // workgroups that a unit's tiles are shared over at most

// Workgroup barrier after LDS accesses alone: loads of the next tile stay in
// flight (a workgroup fence would wait for them).
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));   // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// the wave's number, in a scalar register
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// the larger of two, NaN if either is (which spares the quieting that fmaxf
// puts before each operand)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// maximum / sum over the four lane quarters of a row
__device__ __forceinline__ float quarters_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return larger(__uint_as_float(t[0]), __uint_as_float(t[1]));
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
__host__ __device__ inline Tiles tiles_seen(int first_pos, int last_pos, int window, int sinks) {
    Tiles t;
    const int last = last_pos / KV_TILE;
    t.ns = t.w0 = 0;
    if (window > 0) {
        if (sinks > 0) t.ns = ((sinks - 1) / KV_TILE < last ? (sinks - 1) / KV_TILE : last) + 1;
        t.w0 = first_pos >= window ? (first_pos - window + 1) / KV_TILE : 0;
        if (t.w0 < t.ns) t.w0 = t.ns;
    }
    t.n = t.ns + (last + 1 > t.w0 ? last + 1 - t.w0 : 0);
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
// (masked ones -inf), which become the probabilities 2^((S - m) sc).  m follows
// the maximum when that is past it by 2 and more (a probability is then 4 at
// most): a prompt's rows seldom move it after their first tiles, where every
// third tile has a new maximum in some row and 32 products to make.  up: what
// the output's sums are multiplied by beside (a new power of two of V).
template <int HD, int CT>
__device__ __forceinline__ void softmax_step(Rows<HD, CT> &R, f32x4 (&S)[CT][2], float up = 1.0f) {
#pragma unroll
    for (int c = 0; c < CT; c++) {
        float t = larger(larger(S[c][0][0], S[c][0][1]), S[c][0][2]);
        t = larger(larger(t, S[c][0][3]), S[c][1][0]);
        t = larger(larger(t, S[c][1][1]), S[c][1][2]);
        t = larger(t, S[c][1][3]);
        const float mn = larger(R.m[c], quarters_max(t));
        if (__any((mn - R.m[c]) * R.sc[c] > 2.0f) || up != 1.0f) {
            const float a = R.m[c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((R.m[c] - mn) * R.sc[c]);
            R.l[c] *= a;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) R.o[c][d] *= a * up;
            R.m[c] = mn;
        }
        // (sc is a power of two, so the argument is the difference rounded
        // once, at whatever size the scores are)
        const float mu = R.m[c] == -INFINITY ? 0.0f : -R.m[c] * R.sc[c];
        float l = 0.0f;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                S[c][s][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[c][s][i], R.sc[c], mu));
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

// The Q operand of the fp16 matrix cores: q[b][0] the high halves, [1] the low
// ones (PACK: [0] alone, high or low by the column).
template <int HD, bool PACK> struct QHalf {
    static constexpr int NB = (HD + 31) / 32, NH = PACK ? 1 : 2;
    i32x4 q[NB][NH];
};

// Loads a row's dims 32 b + 8 g .. + 7, scales and splits them.  ORDER4: the
// element order of a code dword, (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16.
template <int HD, bool PACK, bool ORDER4>
__device__ __forceinline__ void load_q16(const AttendArgs &a, const float *row, QHalf<HD, PACK> &Q, float &sc) {
    constexpr int NB = QHalf<HD, PACK>::NB;
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
        if (PACK) Q.q[b][0] = (lane & 8) ? w : h;
        else { Q.q[b][0] = h; Q.q[b][QHalf<HD, PACK>::NH - 1] = w; }
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
// operand: pairs (s = 0, s = 1) of i.  (The conversions of pairs are faster than
// v_fma_mixlo_f16, which would save a third of the instructions: 14 heads of 64,
// 4096 tokens 101 us, 108 with it.)
template <bool PACK>
__device__ __forceinline__ void split_p(const f32x4 (&p)[2], float even, float odd, i32x4 &hi, i32x4 &lo) {
    const bool low = PACK && ((threadIdx.x & 8) != 0);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float f = i & 1 ? odd : even;
        const f32x2 w = f32x2{ p[0][i] * f, p[1][i] * f };
        const f16x2 h = __builtin_convertvector(w, f16x2);
        const f32x2 rest = f32x2{ __builtin_fmaf(p[0][i], f, -(float)h[0]), __builtin_fmaf(p[1][i], f, -(float)h[1]) };   // (exact: f is a power of two)
        if (PACK) {
            const f32x2 mine = f32x2{ low ? rest[0] : w[0], low ? rest[1] : w[1] };
            hi[i] = dword(__builtin_convertvector(mine, f16x2));
        } else {
            hi[i] = dword(h);
            lo[i] = dword(__builtin_convertvector(rest, f16x2));
        }
    }
}

// dims d .. d + 3 of row r of key head kv: o / l
template <int HD>
__device__ __forceinline__ void store_out(const AttendArgs &a, int pos0, int kv, int r, int d, f32x4 o, float l) {
    const int b = a.G(r);
    const float inv = 1.0f / l;
    o *= inv;
    if (pos0 + b < 0 || pos0 + b >= a.ctx) o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float *dst = a.out + (int64_t)b * a.out_stride + ((kv - b) * a.G.d + r) * HD + d;
    if (a.out_vec) {
        *reinterpret_cast<f32x4 *>(dst) = o;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) dst[j] = o[j];
    }
}

// 16 bytes that workgroups of other XCDs read or have written: agent scope
// (sc1), so they pass the XCD's L2 both ways.  A release and acquire per
// workgroup instead writes back and drops a whole L2 each time (512 workgroups
// 17 us where 264 take 12); 8-byte atomics, the widest that the language has,
// make two requests a lane.  p: the start of `bytes` bytes, at: the offset of
// these in them (uniform p).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int AT_SC1 = 16;       // the buffer instructions' bit
struct Shared16 {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ Shared16(void *p, int bytes) : rsrc(__builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, 0x00027000)) {}
    __device__ __forceinline__ void put(int at, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rsrc, at, 0, AT_SC1);
    }
    __device__ __forceinline__ f32x4 get(int at) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, AT_SC1));
    }
};
// one workgroup's partial rows, and their (maximum, sum, scale); those of all
// of a unit's workgroups (at most AT_SPLITS of 128 rows of 128: 4 MB)
template <int HD, int BR> struct Parts {
    Shared16 rows, ml;
    __device__ __forceinline__ Parts(const AttendArgs &a, int64_t slot, int slots)
        : rows(a.part + slot * BR * HD, slots * BR * HD * 4), ml(a.part_ml + slot * BR, slots * BR * 16) {}
};

// The unit's workgroups have put their partial rows away: the last one to
// arrive joins the runs.  Every wave's partial stores have completed, past its
// XCD's L2, before the workgroup counts itself, and the last one's loads go
// past its own.  Called by all NT threads; lds: join_floats(BR, NT) floats.
constexpr size_t join_floats(int br, int nt) { return (size_t)br * (AT_SPLITS + 1) + 4 * nt + 4; }
template <int HD, int BR, int NT>
__device__ __forceinline__ void join_runs(const AttendArgs &a, int unit, int nact, int r0, int r1, int pos0, int kv, float *lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    f32x4 *red = reinterpret_cast<f32x4 *>(lds);    // [NT]
    float *sf = lds + 4 * NT, *sl = sf + BR * AT_SPLITS;   // the runs' weights [row][AT_SPLITS], the rows' sums
    int *last = reinterpret_cast<int *>(sl + BR);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) *last = __hip_atomic_fetch_add(a.count + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nact - 1;
    __syncthreads();
    if (!*last) return;
    if (tid == 0) __hip_atomic_store(a.count + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const Parts<HD, BR> P(a, (int64_t)unit * a.nsplit.d, nact);
    // an item is four dims of a row.  A thread has U of them for Z runs at a time;
    // where there are fewer items than threads, one for Z U runs, and `parts`
    // threads share an item's runs.  The first loads are on their way before the
    // weights are known (a round trip past the L2 is some 1.5 us).
    constexpr int all = (BR * HD / 4 + NT - 1) / NT, U = all < 8 ? all : 8, Z = (BR == 32 && HD == 128 ? 24 : 16) / U;
    const int nr = r1 - r0, items = nr * (HD / 4), parts = items <= NT / 2 ? NT / items : 1;
    const int part = parts > 1 ? tid / items : 0, item = parts > 1 ? tid % items : tid;
    f32x4 x[Z][U];
    auto fetch = [&](int z0, int i0) {   // (z0: the same in all threads)
#pragma unroll
        for (int j = 0; j < Z; j++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (z0 + (parts > 1 ? (j * U + u) * parts : j) >= nact) continue;
                const int z = parts > 1 ? z0 + (j * U + u) * parts + part : z0 + j, i = parts > 1 ? item : min(i0 + u * NT, items - 1);
                x[j][u] = P.rows.get((min(z, nact - 1) * BR * (HD / 4) + i) * 16);
            }
    };
    // a wave a row, a lane a run
    constexpr int NW = NT / 64, RW = (BR + NW - 1) / NW < 8 ? (BR + NW - 1) / NW : 8;
    f32x4 ml[RW];
    auto fetch_ml = [&](int r) {
#pragma unroll
        for (int k = 0; k < RW; k++) ml[k] = P.ml.get((min(lane, nact - 1) * BR + min(r + k * NW, nr - 1)) * 16);
    };
    fetch_ml(wave);
    fetch(0, item);
    for (int r = wave; r < nr; r += RW * NW) {
        if (r != wave) fetch_ml(r);
#pragma unroll
        for (int k = 0; k < RW; k++) {
            const float m = lane < nact ? ml[k][0] : -INFINITY, M = wave_max(m);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - M) * ml[k][2]);
            const float l = wave_sum(lane < nact ? f * ml[k][1] : 0.0f);
            if (r + k * NW >= nr) break;
            sf[(r + k * NW) * AT_SPLITS + lane] = f;
            if (lane == 0) sl[r + k * NW] = l;
        }
    }
    __syncthreads();
    if (parts > 1) {
        const int r = item / (HD / 4);
        f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int z0 = 0; z0 < nact; z0 += Z * U * parts) {
            if (z0) fetch(z0, item);
#pragma unroll
            for (int j = 0; j < Z * U; j++) {
                if (z0 + j * parts >= nact) continue;
                const int z = z0 + j * parts + part;
                const float f = sf[r * AT_SPLITS + min(z, nact - 1)];
                o += x[j / U][j % U] * (part < parts && z < nact ? f : 0.0f);
            }
        }
        red[tid] = o;
        __syncthreads();
        if (tid >= items) return;
#pragma unroll 8
        for (int q = 1; q < parts; q++) o += red[q * items + tid];
        store_out<HD>(a, pos0, kv, r0 + r, item % (HD / 4) * 4, o, sl[r]);
        return;
    }
    for (int i0 = tid; i0 < items; i0 += U * NT) {
        f32x4 o[U];
#pragma unroll
        for (int u = 0; u < U; u++) o[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int z = 0; z < nact; z += Z) {
            if (z || i0 != tid) fetch(z, i0);
#pragma unroll
            for (int j = 0; j < Z; j++) {
                if (z + j >= nact) continue;
#pragma unroll
                for (int u = 0; u < U; u++) o[u] += x[j][u] * sf[min(i0 + u * NT, items - 1) / (HD / 4) * AT_SPLITS + z + j];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * NT, r = i / (HD / 4);
            if (i < items) store_out<HD>(a, pos0, kv, r0 + r, i % (HD / 4) * 4, o[u], sl[r]);
        }
    }
}

// attend_rows.hip: units of ATTEND_ROWS rows
constexpr int ATTEND_ROWS = 128;
void launch_attend_rows(hipStream_t st, int hd, dim3 grid, const AttendArgs &a);

}  // namespace ehip
