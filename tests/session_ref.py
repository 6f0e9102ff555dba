"""64-bit references of the device-row operators (rope.hip, kvcache.hip,
attend.hip) in numpy, and device buffers on the HIP runtime that libember.so
has loaded."""
import ctypes
import math

import numpy as np

from emberllm_amd import _native

TILE, QB = 32, 32
EPS = 2.0 ** -24          # half a step of fp32, relative


class Hip:
    """The few runtime calls that the tests make; loaded once."""

    def __init__(self):
        _native.lib()
        with open("/proc/self/maps") as f:
            paths = {ln.split()[-1] for ln in f if "libamdhip64.so" in ln}
        assert paths, "libamdhip64 is not loaded"
        self.h = h = ctypes.CDLL(sorted(paths)[0])
        P, Z = ctypes.c_void_p, ctypes.c_size_t
        h.hipMalloc.argtypes = [ctypes.POINTER(P), Z]
        h.hipFree.argtypes = [P]
        h.hipMemcpy.argtypes = [P, P, Z, ctypes.c_int]
        h.hipMemset.argtypes = [P, ctypes.c_int, Z]
        h.hipStreamCreate.argtypes = [ctypes.POINTER(P)]
        h.hipStreamSynchronize.argtypes = [P]
        h.hipStreamDestroy.argtypes = [P]
        h.hipStreamBeginCapture.argtypes = [P, ctypes.c_int]
        h.hipStreamEndCapture.argtypes = [P, ctypes.POINTER(P)]
        h.hipGraphInstantiate.argtypes = [ctypes.POINTER(P), P, P, P, Z]
        h.hipGraphLaunch.argtypes = [P, P]
        h.hipGraphExecDestroy.argtypes = [P]
        h.hipGraphDestroy.argtypes = [P]

    def sync(self):
        assert self.h.hipDeviceSynchronize() == 0

    def stream(self):
        s = ctypes.c_void_p()
        assert self.h.hipStreamCreate(ctypes.byref(s)) == 0
        return s

    def capture(self, stream, enqueue):
        g, x = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.h.hipStreamBeginCapture(stream, 0) == 0
        enqueue()
        assert self.h.hipStreamEndCapture(stream, ctypes.byref(g)) == 0
        assert self.h.hipGraphInstantiate(ctypes.byref(x), g, None, None, 0) == 0
        return g, x


_hip = None


def hip():
    global _hip
    if _hip is None:
        _hip = Hip()
    return _hip


class Buf:
    """A device buffer holding a copy of a numpy array."""

    def __init__(self, host):
        self.h, a = hip().h, np.ascontiguousarray(host)
        self.shape, self.dtype, self.nbytes = a.shape, a.dtype, a.nbytes
        p = ctypes.c_void_p()
        assert self.h.hipMalloc(ctypes.byref(p), max(16, a.nbytes)) == 0
        self.ptr = p.value
        self.write(a)

    def write(self, a):
        a = np.ascontiguousarray(a, dtype=self.dtype)
        assert a.nbytes == self.nbytes and self.h.hipMemcpy(self.ptr, a.ctypes.data, a.nbytes, 1) == 0

    def read(self):
        out = np.empty(self.shape, self.dtype)
        assert self.h.hipMemcpy(out.ctypes.data, self.ptr, out.nbytes, 2) == 0
        return out

    def __del__(self):
        try:
            self.h.hipFree(self.ptr)
        except Exception:
            pass


# ------------------------------------------------------------------ rope ----
def frequencies(c, rd):
    theta, s = float(np.float32(c.theta)), float(np.float32(c.factor))
    low, high = float(c.low), float(c.high)
    if c.scaling == _native.ROPE_NTK:
        theta *= s ** (rd / (rd - 2))
    f = np.array([theta ** (-2.0 * i / rd) for i in range(rd // 2)])
    if low == 0 and high == 0:
        low, high = 1.0, 32.0 if c.scaling == _native.ROPE_YARN else 4.0
    if c.scaling == _native.ROPE_LINEAR:
        return f / s
    if c.scaling == _native.ROPE_YARN:
        where = [rd * math.log(c.orig_ctx / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (high, low)]
        first, last = max(math.floor(where[0]), 0), min(math.ceil(where[1]), rd - 1)
        ramp = np.clip((np.arange(rd // 2) - first) / max(last - first, 0.001), 0, 1)
        return f / s * ramp + f * (1 - ramp)
    if c.scaling == _native.ROPE_BANDS:
        keep = np.clip((c.orig_ctx * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f / s * (1 - keep) + f * keep
    return f


def magnitude(c):
    if c.magnitude:
        return float(np.float32(c.magnitude))
    return 0.1 * math.log(float(np.float32(c.factor))) + 1 if c.scaling == _native.ROPE_YARN else 1.0


def turned(c, hd, x, pos, norms=None, eps=0.0):
    """x [n][heads][hd] turned to pos [n]; the second result is |a| + |b| of
    each element's pair (what rounding errors go by; 0 where nothing turns)."""
    x = x.astype(np.float64)
    if norms is not None:
        x = np.where(np.isnan(norms), x, x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * norms)
    rd = c.rotary_dim or hd
    ang = np.asarray(pos, np.float64)[:, None] * frequencies(c, rd)
    cos, sin = (t[:, None, :] * magnitude(c) for t in (np.cos(ang), np.sin(ang)))
    a, b = (slice(0, rd // 2), slice(rd // 2, rd)) if c.style == _native.ROPE_NEOX else (slice(0, rd, 2), slice(1, rd, 2))
    y, size = x.copy(), np.abs(x) if norms is not None else np.zeros_like(x)
    u, v = x[..., a], x[..., b]
    y[..., a], y[..., b] = u * cos - v * sin, u * sin + v * cos
    size[..., a] = size[..., b] = (np.abs(u) + np.abs(v)) * magnitude(c)
    return y, size


# ----------------------------------------------------------------- cache ----
def q4_encode(x):
    """[..., hd] fp32 -> codes [..., hd / 32, 32] and fp16 scales, by
    ember_quant_q4_row's steps; blocks without a finite fp16 scale are NaN."""
    b = np.asarray(x, np.float32).reshape(x.shape[:-1] + (-1, QB))
    m = np.abs(b)
    top = np.take_along_axis(b, np.where(np.isnan(m), np.inf, m).argmax(-1)[..., None], -1)
    with np.errstate(all="ignore"):
        d = (top / np.float32(-8)).astype(np.float32)
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        h = d[..., 0].astype(np.float16)
        bad = ~np.isfinite(h) | ~np.isfinite(b).all(-1)
        codes = np.clip(np.trunc(np.where(bad[..., None], 0, b * inv + np.float32(8.5))), 0, 15).astype(np.uint8)
    h[bad] = np.nan
    return codes, h


def q4_values(x):
    c, d = q4_encode(x)
    return ((c.astype(np.float64) - 8) * d.astype(np.float64)[..., None]).reshape(x.shape)


def cache_values(kind, x):
    """What a cache of this type holds of fp32 rows, in 64 bits."""
    if kind == _native.KV_Q4:
        return q4_values(x)
    with np.errstate(over="ignore"):
        return x.astype(np.float16 if kind == _native.KV_F16 else np.float32).astype(np.float64)


def q4_bytes(x, values, before, have=None):
    """`before`, the bytes [n_kv][tiles][18 * hd] of a 4-bit cache, with the
    positions `have` (default: all) of the rows x [ctx][n_kv][hd] stored:
    element by element of the layout that ehip.h describes."""
    ctx, nkv, hd = x.shape
    nb = hd // QB
    codes, d = q4_encode(x)
    out = before.copy()
    pos = np.arange(ctx) if have is None else np.flatnonzero(have)
    p, dim = np.meshgrid(pos, np.arange(hd), indexing="ij")
    s = p % TILE // 16
    if values:
        g, l, e, n = p % 16 // 4, dim % 16, dim // 16, 4 * s + p % 4
    else:
        g, l, e, n = dim % 32 // 8, p % 16, s * nb + dim // 32, dim % 8
    byte, up = e // 4 * 1024 + (g * 16 + l) * 16 + e % 4 * 4 + n // 2, (4 * (n & 1)).astype(np.uint8)
    sp, sb = np.meshgrid(pos, np.arange(nb), indexing="ij")
    scale_at = 16 * hd + ((((sp % 16 // 4) * nb + sb) * 4 + sp % 4) * 2 + sp % TILE // 16) * 2
    for kv in range(nkv):
        np.bitwise_and.at(out[kv], (p // TILE, byte), ~(np.uint8(15) << up))
        np.bitwise_or.at(out[kv], (p // TILE, byte), codes[pos, kv].reshape(-1, hd) << up)
        raw = d[pos, kv].copy().view(np.uint8).reshape(-1, nb, 2)
        for i in range(2):
            out[kv][sp // TILE, scale_at + i] = raw[..., i]
    return out


# ---------------------------------------------------------------- attend ----
def attended(q, k, v, pos0, window=0, sinks=0, scale=0.0):
    """q [n][nh][hd], cached k, v [ctx][nkv][hd] -> out [n][nh][hd] in 64 bits
    and a bound of |device - out|.

    A score is a product of hd terms: q times scale and log2(e) is rounded
    twice, its two halves leave 2^-23 of it, and the products' sum (in the
    matrix cores, over blocks, and of the two halves) rounds some 12 times:
    20 half steps of sum |q k|.  An error e of the scores (twice: the maximum's
    too) moves a weight by e, the exponential and its argument add 8 half
    steps and half a step of each unit of distance to the maximum; the halves
    of a weight, its sums and the merges of ranges add 24 more.  A row is off by
    at most twice its weights' relative error times sum p |v|.

    fp16 halves also lose what lies below half their smallest step, 2^-25.  A
    weight reaches them relative to a score within 2 (in powers of two) below
    the row's largest so far, so it is 4 at most and goes in times 2^13 without
    leaving fp16; each of the N positions loses at most 2^-25 2^-13 of 1:
    2^-38 N max |v|, before a division by a sum of at least 1 (the largest
    score's own weight is 1 or more)."""
    n, nh, hd = q.shape
    ctx, nkv = k.shape[:2]
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    sc = scale or 1.0 / math.sqrt(hd)
    p = pos0 + np.arange(n)[:, None]
    t = np.arange(ctx)[None, :]
    seen = t <= p
    if window:
        seen &= (t > p - window) | (t < sinks)
    out, bound = np.empty_like(q), np.empty_like(q)
    for h in range(nh):
        kk, vv = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
        use = seen.any(0)
        kk, vv = np.where(use[:, None], kk, 0), np.where(use[:, None], vv, 0)
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(seen, q[:, h] @ kk.T * sc, -np.inf)
            size = np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T * abs(sc), 0)
            m = s.max(1, keepdims=True)
            w = np.exp(s - m)
            w /= w.sum(1, keepdims=True)
            far = np.where(w > 2.0 ** -30, m - s, 0)
            rel = EPS * (40 * size.max(1) + 2 * far.max(1) + 32)
            if np.isfinite(vv).all():   # (an unseen one adds 0)
                if h % (nh // nkv) == 0:
                    top = np.array([np.abs(vv[j]).max(initial=0) for j in seen])
                out[:, h] = w @ vv
                bound[:, h] = 2 * rel[:, None] * (w @ np.abs(vv)) + 2.0 ** -38 * (seen.sum(1) * top)[:, None] + 1e-38
                continue
            for i in range(n):
                j = seen[i]
                out[i, h] = w[i, j] @ vv[j]
                bound[i, h] = 2 * rel[i] * (w[i, j] @ np.abs(vv[j])) + 2.0 ** -38 * j.sum() * np.abs(vv[j]).max(initial=0) + 1e-38
    return out, bound
