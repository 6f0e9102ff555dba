// kvcache.hip — rows of keys and values into a device cache of fp32, fp16 or
// 4 bits and back: ehip_cache_bytes, ehip_cache_store, ehip_cache_load.
//
// 4 bits: blocks of 32 dims as ember_quant_q4_row makes them: v the element of
// largest magnitude (the first of equal ones), d = v / -8, code = (int)(x / d
// + 8.5) by the reciprocal of d, clamped to 0 .. 15; the value is (code - 8)
// times d rounded to fp16.  The tile layout (EhipCache) is the one in which the
// attention's lanes feed the matrix cores: a code dword is 8 dims of a key, or
// 8 positions of a value's dim.  A value's dword therefore belongs to up to 8
// stored tokens: the workgroup that stores them keeps the nibbles of the
// positions it does not store.
//
// Bound: memory.  A workgroup takes one tile of one key head: a thread's piece
// of a row is 8 consecutive dims (its block's maximum over the 4 threads of the
// block, a quad of lanes); values' codes then cross over through LDS, 8
// positions of 8 dims at a time.  8 heads of 128: a token 3.5 us (the launch and
// three trips to memory), 4001 tokens 8.8 us (42 MB, 4.8 TB/s; a copy reaches
// 4.9); the keys back as fp32 6.0 us, the values 6.9 (21 MB).
#include "kv4.h"

namespace ehip {

// nibble j of r[n] <-> nibble n of r[j]
__device__ __forceinline__ void transpose_nibbles(uint32_t (&r)[8]) {
#pragma unroll
    for (int n = 0; n < 4; n++) {
        const uint32_t a = r[n], b = r[n + 4];
        r[n] = __builtin_amdgcn_perm(b, a, 0x05040100);
        r[n + 4] = __builtin_amdgcn_perm(b, a, 0x07060302);
    }
#pragma unroll
    for (int n = 0; n < 8; n += 1 + (n & 1) * 2) {   // 0, 1, 4, 5
        const uint32_t a = r[n], b = r[n + 2];
        r[n] = __builtin_amdgcn_perm(b, a, 0x06020400);
        r[n + 2] = __builtin_amdgcn_perm(b, a, 0x07030501);
    }
#pragma unroll
    for (int n = 0; n < 8; n += 2) {
        const uint32_t a = r[n], b = r[n + 1];
        r[n] = (a & 0x0f0f0f0fu) | (b & 0x0f0f0f0fu) << 4;
        r[n + 1] = (a >> 4 & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u);
    }
}

// grid (tiles the tokens touch, n_kv)
template <int HD>
__global__ __launch_bounds__(WG) void k_kv4_store(KvArgs a) {
    constexpr int NB = HD / QB, KP = HD / 8, KU = KV_TILE * KP / WG;
    __shared__ uint32_t vc[KV_TILE][KP];
    const int tid = threadIdx.x, kv = blockIdx.y;
    const int64_t p0 = a.pos ? (int64_t)*a.pos : a.pos0;
    const int64_t first = p0 < 0 ? 0 : p0, end = min(p0 + a.n_tok, a.ctx);   // positions that are stored
    const int64_t tile = first / KV_TILE + blockIdx.x, t0 = tile * KV_TILE;
    if (max(first, t0) >= end) return;
    const int k0 = (int)max(first - t0, (int64_t)0), k1 = (int)min(end - t0, (int64_t)KV_TILE);   // those of this tile
    uint8_t *kt = a.kc + ((int64_t)kv * a.tiles + tile) * kv_tile_bytes(HD), *vt = a.vc + ((int64_t)kv * a.tiles + tile) * kv_tile_bytes(HD);
    const float *kr = a.k + (t0 - p0) * a.k_stride + (int64_t)kv * HD, *vr = a.v + (t0 - p0) * a.v_stride + (int64_t)kv * HD;

    // thread (position, piece of 8 dims), pieces fastest; all of its rows' loads
    // are on their way before the first is used
    RowV x[KU][2], y[KU][2];
#pragma unroll
    for (int u = 0; u < KU; u++) {
        const int i = tid + u * WG, t = min(max(i / KP, k0), k1 - 1), c = i % KP;   // (a stored position in any case)
        const RowV *xs = reinterpret_cast<const RowV *>(kr + t * a.k_stride + 8 * c), *ys = reinterpret_cast<const RowV *>(vr + t * a.v_stride + 8 * c);
        x[u][0] = xs[0]; x[u][1] = xs[1];
        y[u][0] = ys[0]; y[u][1] = ys[1];
    }
#pragma unroll
    for (int u = 0; u < KU; u++) {
        const int i = tid + u * WG, t = i / KP, c = i % KP, b = c / 4, g = c % 4, half = t / 16, l = t % 16;
        const bool in = t >= k0 && t < k1;
        uint16_t kd, vd;
        const uint32_t kw = q4_piece(x[u], kd);
        vc[t][c] = q4_piece(y[u], vd);
        if (!in) continue;
        *reinterpret_cast<uint32_t *>(kt + kv_code_at(g * 16 + l, half * NB + b)) = kw;
        if (g == 0) {
            *reinterpret_cast<uint16_t *>(kt + kv_scale_at(HD, l / 4, b, l % 4, half)) = kd;
            *reinterpret_cast<uint16_t *>(vt + kv_scale_at(HD, l / 4, b, l % 4, half)) = vd;
        }
    }
    __syncthreads();

    // values: thread (quarter g, piece of 8 dims): positions 16 s + 4 g + i
    if (tid >= 4 * KP) return;
    const int g = tid / KP, c = tid % KP;
    uint32_t keep = 0, r[8];
#pragma unroll
    for (int n = 0; n < 8; n++) {
        const int t = 16 * (n / 4) + 4 * g + n % 4;
        if (t < k0 || t >= k1) keep |= 15u << (4 * n);
        r[n] = vc[t][c];
    }
    if (keep == 0xffffffffu) return;
    transpose_nibbles(r);
    uint8_t *dst = vt + kv_code_at(g * 16 + 8 * c % 16, c / 2);
    if (keep) {
        uint32_t old[8];
#pragma unroll
        for (int j = 0; j < 8; j++) old[j] = *reinterpret_cast<const uint32_t *>(dst + 16 * j);
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = (r[j] & ~keep) | (old[j] & keep);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) *reinterpret_cast<uint32_t *>(dst + 16 * j) = r[j];
}

// fp32 and fp16: grid-stride over the rows' pieces of four
template <bool F16>
__global__ __launch_bounds__(WG) void k_kv_store(KvArgs a, int kvd) {
    const int64_t p0 = a.pos ? (int64_t)*a.pos : a.pos0;
    const int per = kvd / 4;
    const int64_t n = (int64_t)a.n_tok * per;
    for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < n; i += (int64_t)gridDim.x * WG) {
        const int64_t b = i / per, t = p0 + b;
        const int c = (int)(i % per) * 4;
        if (t < 0 || t >= a.ctx) continue;
        const f32x4 x = *reinterpret_cast<const RowV *>(a.k + b * a.k_stride + c), y = *reinterpret_cast<const RowV *>(a.v + b * a.v_stride + c);
        if (F16) {
            typedef _Float16 H __attribute__((ext_vector_type(4)));
            *reinterpret_cast<H *>(reinterpret_cast<_Float16 *>(a.kc) + t * kvd + c) = __builtin_convertvector(x, H);
            *reinterpret_cast<H *>(reinterpret_cast<_Float16 *>(a.vc) + t * kvd + c) = __builtin_convertvector(y, H);
        } else {
            *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(a.kc) + t * kvd + c) = x;
            *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(a.vc) + t * kvd + c) = y;
        }
    }
}

// ---- back to fp32 rows (positions pos0 .. pos0 + n_tok - 1, in range) -----
template <int HD>
__global__ __launch_bounds__(WG) void k_kv4_load(KvArgs a) {
    const int tid = threadIdx.x, kv = blockIdx.y;
    const int64_t tile = a.pos0 / KV_TILE + blockIdx.x, t0 = tile * KV_TILE, end = a.pos0 + a.n_tok;
    const uint8_t *ct = (a.which ? a.vc : a.kc) + ((int64_t)kv * a.tiles + tile) * kv_tile_bytes(HD);
    float *out = a.out + (int64_t)kv * HD;
    constexpr int NB = HD / QB;
    if (!a.which) {
        constexpr int KP = HD / 8;
#pragma unroll
        for (int u = 0; u < KV_TILE * KP / WG; u++) {
            const int i = tid + u * WG, key = i / KP, c = i % KP, b = c / 4, g = c % 4, half = key / 16, l = key % 16;
            const int64_t t = t0 + key;
            if (t < a.pos0 || t >= end) continue;
            const uint32_t w = *reinterpret_cast<const uint32_t *>(ct + kv_code_at(g * 16 + l, half * NB + b));
            const float d = h2f(*reinterpret_cast<const uint16_t *>(ct + kv_scale_at(HD, l / 4, b, l % 4, half)));
            RowV *dst = reinterpret_cast<RowV *>(out + (t - a.pos0) * a.k_stride + 8 * c);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                RowV x;
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = (float)((int)(w >> (16 * h + 4 * j) & 15) - 8) * d;
                dst[h] = x;
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < 4 * HD / WG; u++) {
            const int j = tid + u * WG, dim = j % HD, g = j / HD, b = dim / QB;
            const uint32_t w = *reinterpret_cast<const uint32_t *>(ct + kv_code_at(g * 16 + dim % 16, dim / 16));
            const i32x4 ds = *reinterpret_cast<const i32x4 *>(ct + kv_scale_at(HD, g, b, 0, 0));   // [i][s]
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const int64_t t = t0 + 16 * (n / 4) + 4 * g + n % 4;
                if (t < a.pos0 || t >= end) continue;
                const float d = h2f((uint16_t)(ds[n % 4] >> (16 * (n / 4))));
                out[(t - a.pos0) * a.k_stride + dim] = (float)((int)(w >> (4 * n) & 15) - 8) * d;
            }
        }
    }
}

template <bool F16>
__global__ __launch_bounds__(WG) void k_kv_load(KvArgs a, int kvd) {
    const int per = kvd / 4;
    const int64_t n = (int64_t)a.n_tok * per;
    const uint8_t *src = a.which ? a.vc : a.kc;
    for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < n; i += (int64_t)gridDim.x * WG) {
        const int64_t b = i / per, t = a.pos0 + b;
        const int c = (int)(i % per) * 4;
        f32x4 x;
        if (F16) {
            typedef _Float16 H __attribute__((ext_vector_type(4)));
            x = __builtin_convertvector(*reinterpret_cast<const H *>(reinterpret_cast<const _Float16 *>(src) + t * kvd + c), f32x4);
        } else {
            x = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(src) + t * kvd + c);
        }
        *reinterpret_cast<RowV *>(a.out + b * a.k_stride + c) = x;
    }
}

int check_cache(const char *who, const EhipCache *c, bool pointers) {
    if (!c) return refuse("%s: null cache", who);
    if (c->type < EHIP_KV_F32 || c->type > EHIP_KV_Q4) return refuse("%s: unknown cache type %d", who, c->type);
    if (c->head_dim != 64 && c->head_dim != 128 && !(c->head_dim == 48 && c->type != EHIP_KV_Q4))
        return refuse("%s: head_dim %d is not supported by a cache of type %d", who, c->head_dim, c->type);
    if (c->n_kv < 1 || c->n_kv > 65535) return refuse("%s: %d key heads", who, c->n_kv);
    if (c->ctx < 1 || c->ctx > 1 << 30) return refuse("%s: a cache of %lld positions", who, (long long)c->ctx);
    if (c->reserved) return refuse("%s: the reserved field is not zero", who);
    if (pointers && (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)))
        return refuse("%s: the cache's pointers are null or not 16-byte aligned", who);
    return 0;
}

KvArgs kv_args(const EhipCache &c) {
    KvArgs a{};
    a.kc = static_cast<uint8_t *>(c.k);
    a.vc = static_cast<uint8_t *>(c.v);
    a.ctx = c.ctx;
    a.n_kv = c.n_kv;
    a.tiles = (int)((c.ctx + KV_TILE - 1) / KV_TILE);
    return a;
}

// tiles that n positions from any first one, or from pos0, can touch
static unsigned tiles_of(const int *pos, int64_t pos0, int n) {
    const int64_t off = pos ? KV_TILE - 1 : pos0 % KV_TILE;
    return (unsigned)((off + n + KV_TILE - 1) / KV_TILE);
}

static dim3 row_grid(int64_t pieces) {
    const int64_t wgs = (pieces + WG - 1) / WG;
    return dim3((unsigned)(wgs < 8192 ? wgs : 8192));
}

int launch_cache_store(hipStream_t st, const EhipCache &c, const EhipCacheRows &r) {
    KvArgs a = kv_args(c);
    a.k = r.k; a.v = r.v; a.k_stride = r.k_stride; a.v_stride = r.v_stride;
    a.n_tok = r.n_tok; a.pos0 = r.pos0; a.pos = r.pos;
    const int kvd = c.n_kv * c.head_dim;
    if (c.type == EHIP_KV_Q4) {
        const dim3 grid(tiles_of(r.pos, r.pos0, r.n_tok), c.n_kv);
        if (c.head_dim == 128) hipLaunchKernelGGL(k_kv4_store<128>, grid, dim3(WG), 0, st, a);
        else hipLaunchKernelGGL(k_kv4_store<64>, grid, dim3(WG), 0, st, a);
    } else {
        const dim3 grid = row_grid((int64_t)r.n_tok * kvd / 4);
        if (c.type == EHIP_KV_F16) hipLaunchKernelGGL(k_kv_store<true>, grid, dim3(WG), 0, st, a, kvd);
        else hipLaunchKernelGGL(k_kv_store<false>, grid, dim3(WG), 0, st, a, kvd);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ehip

using namespace ehip;

extern "C" uint64_t ehip_cache_bytes(const EhipCache *c) {
    if (check_cache("ehip_cache_bytes", c, false)) return 0;
    const uint64_t kvd = (uint64_t)c->n_kv * c->head_dim;
    if (c->type == EHIP_KV_Q4) return (uint64_t)(c->ctx + KV_TILE - 1) / KV_TILE * c->n_kv * kv_tile_bytes(c->head_dim);
    return (uint64_t)c->ctx * kvd * (c->type == EHIP_KV_F16 ? 2 : 4);
}

extern "C" int ehip_cache_store(const EhipCache *c, const EhipCacheRows *r, void *stream) {
    const char *who = "ehip_cache_store";
    if (!r) return refuse("%s: null argument", who);
    if (check_cache(who, c, true)) return -1;
    if (r->n_tok < 0 || r->n_tok > c->ctx) return refuse("%s: %d tokens into a cache of %lld", who, r->n_tok, (long long)c->ctx);
    if (!r->n_tok) return 0;
    if (!r->k || !r->v) return refuse("%s: null rows", who);
    const int64_t kvd = (int64_t)c->n_kv * c->head_dim;
    if (r->n_tok > 1 && (r->k_stride < kvd || r->v_stride < kvd))
        return refuse("%s: strides %lld and %lld for rows of %lld floats", who, (long long)r->k_stride, (long long)r->v_stride, (long long)kvd);
    if (!r->pos && (r->pos0 < 0 || (int64_t)r->pos0 + r->n_tok > c->ctx))
        return refuse("%s: positions %d..%lld exceed the cache of %lld", who, r->pos0, (long long)r->pos0 + r->n_tok - 1, (long long)c->ctx);
    if (launch_cache_store(static_cast<hipStream_t>(stream), *c, *r)) return refuse("%s: launch failed", who);
    return 0;
}

extern "C" int ehip_cache_load(const EhipCache *c, int which, int64_t pos0, int n_pos, float *out, int64_t out_stride, void *stream) {
    const char *who = "ehip_cache_load";
    if (check_cache(who, c, true)) return -1;
    if (which != 0 && which != 1) return refuse("%s: %d is neither keys (0) nor values (1)", who, which);
    if (n_pos < 0 || pos0 < 0 || pos0 > c->ctx || n_pos > c->ctx - pos0)
        return refuse("%s: positions %lld.. (%d) exceed the cache of %lld", who, (long long)pos0, n_pos, (long long)c->ctx);
    if (!n_pos) return 0;
    if (!out) return refuse("%s: null rows", who);
    const int kvd = c->n_kv * c->head_dim;
    if (n_pos > 1 && out_stride < kvd) return refuse("%s: stride %lld for rows of %d floats", who, (long long)out_stride, kvd);
    hipStream_t st = static_cast<hipStream_t>(stream);
    KvArgs a = kv_args(*c);
    a.out = out; a.k_stride = out_stride; a.pos0 = pos0; a.n_tok = n_pos; a.which = which;
    if (c->type == EHIP_KV_Q4) {
        const dim3 grid(tiles_of(nullptr, pos0, n_pos), c->n_kv);
        if (c->head_dim == 128) hipLaunchKernelGGL(k_kv4_load<128>, grid, dim3(WG), 0, st, a);
        else hipLaunchKernelGGL(k_kv4_load<64>, grid, dim3(WG), 0, st, a);
    } else {
        const dim3 grid = row_grid((int64_t)n_pos * kvd / 4);
        if (c->type == EHIP_KV_F16) hipLaunchKernelGGL(k_kv_load<true>, grid, dim3(WG), 0, st, a, kvd);
        else hipLaunchKernelGGL(k_kv_load<false>, grid, dim3(WG), 0, st, a, kvd);
    }
    if (hipGetLastError() != hipSuccess) return refuse("%s: launch failed", who);
    return 0;
}
