// session.h — rotary positions, key/value caches and attention on device rows
// (rope.hip, kvcache.hip, attend.hip): what the three share, and their launches
// for the states' schedules.
#pragma once
#include <cstdarg>
#include <cstdio>

#include "../../../include/ehip.h"
#include "kernels.h"

namespace ehip {

// ehip_last_error()'s text for an entry point that refuses its call
__attribute__((format(printf, 1, 2))) inline int refuse(const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_error_text(buf);
    return -1;
}

inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The 4-bit cache (the layout is described at EhipCache): positions and dims
// of a tile, its bytes, and the bytes of its codes.
constexpr int KV_TILE = 32;
__host__ __device__ constexpr int kv_tile_codes(int hd) { return hd * KV_TILE / 2; }
__host__ __device__ constexpr int kv_tile_bytes(int hd) { return kv_tile_codes(hd) + hd / QB * KV_TILE * 2; }
// byte of lane `lane`'s code dword e, and of the scale of (g, b, i, s)
__host__ __device__ constexpr int kv_code_at(int lane, int e) { return (e >> 2) * 1024 + lane * 16 + (e & 3) * 4; }
__host__ __device__ constexpr int kv_scale_at(int hd, int g, int b, int i, int s) {
    return kv_tile_codes(hd) + (((g * (hd / QB) + b) * 4 + i) * 2 + s) * 2;
}

int launch_rope(hipStream_t st, const EhipRopePlan &p, const EhipRopeRows &r);
int launch_cache_store(hipStream_t st, const EhipCache &c, const EhipCacheRows &r);
int launch_rope_store(hipStream_t st, const EhipRopePlan &p, const EhipRopeRows &r, const EhipCache &c, const EhipCacheRows &w);   // one token
int launch_attend(hipStream_t st, const EhipCache &c, const EhipAttend &q);   // sets ehip_last_error() itself

// 0, or -1 with ehip_last_error() set: a cache that the kernels support
int check_cache(const char *who, const EhipCache *c, bool pointers);

}  // namespace ehip
