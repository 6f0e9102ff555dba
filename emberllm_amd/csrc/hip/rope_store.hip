// rope_store.hip — the rotation of one token's heads and the store of its key and
// value in one launch, for the decode steps of states with options: the
// arithmetic of rope.hip and kvcache.hip, so a step's rows are what those two
// launches make of them.
//
// Bound: the launch.  A workgroup takes a key head: its waves turn the query
// heads that share it and the key, then its first wave stores the key and its
// second the value.  A step of the 28-layer Qwen3-0.6B shape with a 4-bit cache
// and a window takes 0.853 ms, with the two launches 0.927.
#include "kv4.h"
#include "rope.h"

namespace ehip {

template <int TYPE, int HD, int VEC, bool NORM>
__global__ __launch_bounds__(WG) void k_rope_store(RopeArgs a, EhipRopePlan p, KvArgs c) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kv = blockIdx.x;
    const int G = a.n_q / c.n_kv, hpw = 64 / a.lg;
    rope_heads<VEC, 1, NORM>(a, p, 0, wave, (G + hpw) / hpw, WG / 64, G + 1, [&](int i) { return i < G ? kv * G + i : a.n_q + kv; });
    __syncthreads();   // (the key's row is read back below)
    const int64_t t = c.pos ? (int64_t)*c.pos : c.pos0;
    if (wave > 1 || t < 0 || t >= c.ctx) return;
    const float *row = (wave ? c.v : c.k) + (int64_t)kv * HD;
    if constexpr (TYPE == EHIP_KV_Q4) {
        constexpr int NB = HD / QB, KP = HD / 8;
        const int pc = lane % KP, s = (int)(t % KV_TILE) / 16, l = (int)(t % 16), b = pc / 4, g = pc % 4;
        uint8_t *tile = (wave ? c.vc : c.kc) + ((int64_t)kv * c.tiles + t / KV_TILE) * kv_tile_bytes(HD);
        const RowV *src = reinterpret_cast<const RowV *>(row + 8 * pc);
        const RowV x[2] = { src[0], src[1] };
        uint16_t d;
        const uint32_t w = q4_piece(x, d);
        if (lane >= KP) return;
        if (g == 0) *reinterpret_cast<uint16_t *>(tile + kv_scale_at(HD, l / 4, b, l % 4, s)) = d;
        if (wave == 0) {
            *reinterpret_cast<uint32_t *>(tile + kv_code_at(g * 16 + l, s * NB + b)) = w;
        } else {   // nibble n of eight dims' dwords, which this thread alone writes
            const int n = 4 * (4 * s + l % 4);
            uint8_t *dst = tile + kv_code_at(l / 4 * 16 + 8 * pc % 16, pc / 2);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                uint32_t *o = reinterpret_cast<uint32_t *>(dst + 16 * j);
                *o = (*o & ~(15u << n)) | (w >> (4 * j) & 15) << n;
            }
        }
    } else {
        if (lane >= HD / 4) return;
        const f32x4 x = reinterpret_cast<const RowV *>(row)[lane];
        const int64_t at = t * c.n_kv * HD + kv * HD + 4 * lane;
        if constexpr (TYPE == EHIP_KV_F16) {
            typedef _Float16 H __attribute__((ext_vector_type(4)));
            *reinterpret_cast<H *>(reinterpret_cast<_Float16 *>(wave ? c.vc : c.kc) + at) = __builtin_convertvector(x, H);
        } else {
            *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(wave ? c.vc : c.kc) + at) = x;
        }
    }
}

// One token: r's rows, whose key heads are w's keys (w.k lies in r.out).
int launch_rope_store(hipStream_t st, const EhipRopePlan &p, const EhipRopeRows &r, const EhipCache &c, const EhipCacheRows &w) {
    bool vec;
    const RopeArgs a = rope_args(p, r, &vec);
    KvArgs k = kv_args(c);
    k.k = w.k; k.v = w.v; k.pos0 = w.pos0; k.pos = w.pos;
    const bool norm = r.q_norm || r.k_norm;
    const dim3 grid(c.n_kv), wg(WG);
#define RS_GO(T, H)                                                                                                      \
    if (c.type == T && c.head_dim == H) {                                                                                \
        if (vec && norm) hipLaunchKernelGGL((k_rope_store<T, H, 4, true>), grid, wg, 0, st, a, p, k);                    \
        else if (vec) hipLaunchKernelGGL((k_rope_store<T, H, 4, false>), grid, wg, 0, st, a, p, k);                      \
        else if (norm) hipLaunchKernelGGL((k_rope_store<T, H, 1, true>), grid, wg, 0, st, a, p, k);                      \
        else hipLaunchKernelGGL((k_rope_store<T, H, 1, false>), grid, wg, 0, st, a, p, k);                               \
    }
    RS_GO(EHIP_KV_F32, 48) RS_GO(EHIP_KV_F32, 64) RS_GO(EHIP_KV_F32, 128)
    RS_GO(EHIP_KV_F16, 48) RS_GO(EHIP_KV_F16, 64) RS_GO(EHIP_KV_F16, 128)
    RS_GO(EHIP_KV_Q4, 64) RS_GO(EHIP_KV_Q4, 128)
#undef RS_GO
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ehip
