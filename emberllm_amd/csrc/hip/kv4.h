// kv4.h — the 4-bit blocks of a row's dims and the caches' arguments, for
// kvcache.hip and for the kernel that rotates and stores (rope_store.hip).
#pragma once
#include "session.h"

namespace ehip {

struct KvArgs {
    const float *k, *v;          // store: rows; load: unused
    float *out;                  // load
    int64_t k_stride, v_stride;
    uint8_t *kc, *vc;
    int64_t ctx, pos0;
    const int *pos;
    int n_tok, n_kv, tiles, which;
};

// the element of larger magnitude as fp32 bits: NaN above infinity above all
// numbers; the first of equal ones (`o` comes before `m` where before)
__device__ __forceinline__ uint32_t q4_top(uint32_t m, uint32_t o, bool before) {
    const uint32_t a = m & 0x7fffffffu, b = o & 0x7fffffffu;
    return b > a || (b == a && before) ? o : m;
}

struct Q4Scale { float inv; uint16_t d; };
__device__ __forceinline__ Q4Scale q4_scale(uint32_t top) {
    const float d = __uint_as_float(top) / -8.0f;
    Q4Scale s;
    s.inv = d != 0.0f ? 1.0f / d : 0.0f;
    s.d = f2h(d);
    if ((s.d & 0x7c00) == 0x7c00) s.d = 0x7e00;   // NaN, infinite, or past fp16: the block reads back as NaN
    return s;
}
__device__ __forceinline__ uint32_t q4_code(float x, float inv) {
    const int c = (int)(x * inv + 8.5f);
    return (uint32_t)min(max(c, 0), 15);
}

// four floats of a row (rows of any alignment)
typedef float RowV __attribute__((ext_vector_type(4), aligned(4)));

// The codes of 8 dims of a row (nibble j: dim j) and their block's scale, the
// block's other dims in the quad's other lanes.
__device__ __forceinline__ uint32_t q4_piece(const RowV (&x)[2], uint16_t &d) {
    uint32_t m = __float_as_uint(x[0][0]);
#pragma unroll
    for (int j = 1; j < 8; j++) m = q4_top(m, __float_as_uint(x[j / 4][j % 4]), false);
    m = q4_top(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, false), (threadIdx.x & 1) != 0);
    m = q4_top(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, false), (threadIdx.x & 2) != 0);
    const Q4Scale s = q4_scale(m);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) w |= q4_code(x[j / 4][j % 4], s.inv) << (4 * j);
    d = s.d;
    return w;
}

KvArgs kv_args(const EhipCache &c);

}  // namespace ehip
