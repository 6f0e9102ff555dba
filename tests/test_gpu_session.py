"""The operators of a long session on device rows: scaled rotary positions
(ehip_rope_rows), rows in a cache (ehip_cache_store, ehip_cache_load) and
attention over it (ehip_attend), each against 64-bit references (session_ref),
and a run of them together."""
import ctypes
import math
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import session_ref as R  # noqa: E402

from emberllm_amd import _native  # noqa: E402

pytestmark = pytest.mark.gpu
I, N = _native.ROPE_INTERLEAVED, _native.ROPE_NEOX
F32, F16, Q4 = _native.KV_F32, _native.KV_F16, _native.KV_Q4
GUARD = 64   # floats of padding behind the last row of an output, which stay as they were


def ok(rc):
    assert rc == 0, _native.last_error()


def within(err, bound):
    """Every error within its bound (NaN is not)."""
    if not (err <= bound).all():
        at = np.unravel_index(np.argmax(np.where(err <= bound, 0, np.nan_to_num(err, nan=np.inf))), err.shape)
        pytest.fail(f"{np.count_nonzero(~(err <= bound))} of {err.size} off, worst at {at}: {err[at]:.3g}, bound {bound[at]:.3g}")


def rows_buf(n, width, stride, fill=np.nan):
    return R.Buf(np.full(max(0, n - 1) * stride + width + GUARD, fill, np.float32))


def as_rows(flat, n, width, stride):
    return np.stack([flat[i * stride:i * stride + width] for i in range(n)]) if n else np.empty((0, width), np.float32)


def untouched(flat, n, width, stride):
    keep = np.ones(len(flat), bool)
    for i in range(n):
        keep[i * stride:i * stride + width] = False
    return np.isnan(flat[keep]).all()


# ------------------------------------------------------------------ rope ----
def config(style=N, rd=0, scaling=0, theta=1e4, factor=1.0, orig=2048, low=0.0, high=0.0, magnitude=0.0):
    return _native.EhipRopeConfig(style=style, rotary_dim=rd, scaling=scaling, theta=theta, factor=factor, orig_ctx=orig, low=low, high=high,
                                  magnitude=magnitude)


def rope(cfg, hd, x, n_q, n_k, pos0=0, pos=None, norms=None, eps=1e-6, stride=None, in_place=False, shift=0):
    """x [n][width >= (n_q + n_k) hd] on the device; the turned rows."""
    lib, n, w = _native.lib(), len(x), (n_q + n_k) * hd
    plan = _native.EhipRopePlan()
    ok(lib.ehip_rope_plan(cfg, hd, plan))
    stride = stride or w
    flat = np.concatenate([np.full(shift, 7, np.float32), x.ravel()])
    xb = R.Buf(flat)
    out = rows_buf(n, w, stride)
    r = _native.EhipRopeRows(x=xb.ptr + 4 * shift, out=xb.ptr + 4 * shift if in_place else out.ptr, x_stride=x.shape[1],
                             out_stride=x.shape[1] if in_place else stride, n_tok=n, n_q=n_q, n_k=n_k, pos0=pos0, eps=eps)
    pb = R.Buf(np.asarray(pos, np.int32)) if pos is not None else None
    if pb:
        r.pos = pb.ptr
    nb = [R.Buf(t) if t is not None else None for t in norms or (None, None)]
    r.q_norm, r.k_norm = (b.ptr if b else None for b in nb)
    ok(lib.ehip_rope_rows(plan, r, None))
    R.hip().sync()
    if in_place:
        got = xb.read()[shift:].reshape(x.shape)
        np.testing.assert_array_equal(got[:, w:], x[:, w:])
        return got[:, :w]
    flat = out.read()
    assert untouched(flat, n, w, stride)
    return as_rows(flat, n, w, stride)


def check_rope(got, cfg, hd, x, n_q, n_k, pos, norms=None, eps=1e-6):
    n = len(x)
    xx = x[:, :(n_q + n_k) * hd].reshape(n, n_q + n_k, hd)
    w = None
    if norms is not None:
        w = np.full((n_q + n_k, hd), np.nan)
        for part, t in ((slice(0, n_q), norms[0]), (slice(n_q, None), norms[1])):
            if t is not None:
                w[part] = t
    want, size = R.turned(cfg, hd, xx, pos, w, eps)
    # cos and sin: the angle's conversion and constant (2 half steps of an
    # angle below 0.8), the polynomial's last two roundings and the magnitude;
    # then two products and a sum: at most 8 half steps of |a| + |b|.  A norm
    # adds its sum of squares over lanes (at most 10), root, reciprocal and two
    # products.
    bound = R.EPS * size * (8 if norms is None else 24)
    err = np.abs(got.reshape(want.shape) - want)
    within(err, bound)


SCALED = [dict(), dict(scaling=1, factor=4.0), dict(scaling=2, factor=3.0), dict(scaling=3, factor=8.0, theta=1e6, orig=4096),
          dict(scaling=3, factor=16.0, theta=5e5, orig=300, low=2.0, high=20.0), dict(scaling=4, factor=8.0, theta=5e5, orig=8192),
          dict(magnitude=1.25), dict(scaling=3, factor=1.0)]


@pytest.mark.parametrize("style", [I, N])
@pytest.mark.parametrize("k", range(len(SCALED)))
def test_rope_scalings(style, k):
    rng = np.random.default_rng(k)
    cfg = config(style, **SCALED[k])
    x = rng.standard_normal((33, 6 * 64)).astype(np.float32)
    for pos0 in (0, 131000, 2 ** 31 - 40):
        got = rope(cfg, 64, x, 4, 2, pos0)
        check_rope(got, cfg, 64, x, 4, 2, pos0 + np.arange(33, dtype=np.int64))


# (head_dim, rotary_dim, query heads, key heads, tokens): whole heads and
# parts, sizes that take the 4-byte path, one head, many rows (angles shared)
SIZES = [(128, 128, 16, 8, 1), (128, 32, 3, 1, 7), (64, 48, 9, 3, 65), (48, 48, 2, 1, 5), (48, 12, 2, 0, 3), (80, 20, 0, 5, 9), (2, 2, 3, 2, 4),
         (6, 4, 5, 1, 11), (256, 256, 2, 1, 3), (256, 62, 1, 1, 2), (250, 250, 2, 1, 3), (64, 64, 14, 2, 700), (64, 32, 14, 2, 2100), (72, 72, 1, 0, 1), (128, 128, 1, 1, 4100)]


@pytest.mark.parametrize("style", [I, N])
@pytest.mark.parametrize("hd,rd,n_q,n_k,n", SIZES)
def test_rope_sizes(style, hd, rd, n_q, n_k, n):
    rng = np.random.default_rng(hd + n)
    cfg = config(style, rd=rd, theta=1e5)
    x = rng.standard_normal((n, (n_q + n_k) * hd)).astype(np.float32)
    got = rope(cfg, hd, x, n_q, n_k, 1000)
    check_rope(got, cfg, hd, x, n_q, n_k, 1000 + np.arange(n))
    norms = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    for pair in (norms, (norms[0], None), (None, norms[1])):
        got = rope(cfg, hd, x, n_q, n_k, 5, norms=pair)
        check_rope(got, cfg, hd, x, n_q, n_k, 5 + np.arange(n), pair)


@pytest.mark.parametrize("style", [I, N])
def test_rope_rows_in_place_strided_unaligned_and_at_any_position(style):
    rng = np.random.default_rng(3)
    cfg = config(style, rd=64, scaling=4, factor=4.0)
    x = rng.standard_normal((10, 8 * 128 + 20)).astype(np.float32)   # q | k | (other)
    pos = np.array([0, 5, 5, 1, -7, 2 ** 31 - 1, -2 ** 31, 123456789, 40000, 2], np.int64)
    want = rope(cfg, 128, x, 6, 2, pos=pos)
    check_rope(want, cfg, 128, x, 6, 2, pos)
    np.testing.assert_array_equal(rope(cfg, 128, x, 6, 2, pos=pos, in_place=True), want)
    for shift, stride in ((1, None), (0, 1031), (4, 1040)):   # 4-byte accesses, and 16-byte ones
        np.testing.assert_array_equal(rope(cfg, 128, x, 6, 2, pos=pos, shift=shift, stride=stride), want)


@pytest.mark.parametrize("style", [I, N])
def test_rope_keeps_what_does_not_turn(style):
    """Infinities and NaN in dims that do not turn stay there."""
    x = np.ones((3, 2 * 64), np.float32)
    x[:, 40], x[:, 41], x[:, 63], x[:, 64 + 60] = np.inf, np.nan, -np.inf, np.nan
    cfg = config(style, rd=40)
    got = rope(cfg, 64, x, 1, 1, 9).reshape(3, 2, 64)
    np.testing.assert_array_equal(got[..., 40:], x.reshape(3, 2, 64)[..., 40:])
    assert np.isfinite(got[..., :40]).all()


# ----------------------------------------------------------------- cache ----
class Cache:
    def __init__(self, kind, n_kv, hd, ctx, fill=None):
        self.c = _native.EhipCache(type=kind, n_kv=n_kv, head_dim=hd, ctx=ctx)
        self.lib, self.kind, self.n_kv, self.hd, self.ctx = _native.lib(), kind, n_kv, hd, ctx
        n = self.lib.ehip_cache_bytes(self.c)
        assert n > 0, _native.last_error()
        self.k, self.v = (R.Buf(np.full(n, 0xA5 if fill is None else fill, np.uint8)) for _ in range(2))
        self.c.k, self.c.v = self.k.ptr, self.v.ptr

    def store(self, k, v, pos0, pos=None, stream=None, pad=0):
        n, w = len(k), self.n_kv * self.hd
        kb, vb = (R.Buf(np.pad(t.reshape(n, w), ((0, 0), (0, p)))) for t, p in ((k, pad), (v, 2 * pad)))
        r = _native.EhipCacheRows(k=kb.ptr, v=vb.ptr, k_stride=w + pad, v_stride=w + 2 * pad, n_tok=n, pos0=pos0, pos=pos)
        ok(self.lib.ehip_cache_store(self.c, r, stream))
        R.hip().sync()

    def load(self, which, pos0, n, pad=0):
        w = self.n_kv * self.hd
        out = rows_buf(n, w, w + pad)
        ok(self.lib.ehip_cache_load(self.c, which, pos0, n, out.ptr, w + pad, None))
        R.hip().sync()
        flat = out.read()
        assert untouched(flat, n, w, w + pad)
        return as_rows(flat, n, w, w + pad).reshape(n, self.n_kv, self.hd)


def kv_rows(rng, n, n_kv, hd):
    k = rng.standard_normal((n, n_kv, hd)) * np.where(rng.random(hd) < 0.05, 6, 1)
    v = rng.standard_normal((n, n_kv, hd)) * 0.4
    return k.astype(np.float32), v.astype(np.float32)


KINDS = [(F32, 48), (F32, 64), (F32, 128), (F16, 48), (F16, 64), (F16, 128), (Q4, 64), (Q4, 128)]


@pytest.mark.parametrize("kind,hd", KINDS)
@pytest.mark.parametrize("n_kv", [1, 3])
def test_cache_stores_and_loads(kind, hd, n_kv):
    """Rows come back as the type holds them, exactly, from any first position
    and in any order of stores; positions not stored keep their bytes."""
    rng = np.random.default_rng(hd + n_kv)
    ctx = 150
    c = Cache(kind, n_kv, hd, ctx)
    before = [b.read() for b in (c.k, c.v)]
    k, v = kv_rows(rng, ctx, n_kv, hd)
    have = np.zeros(ctx, bool)
    for pos0, n, pad in ((33, 1, 0), (0, 5, 0), (34, 30, 3), (70, 70, 4), (40, 8, 0), (149, 1, 0), (31, 1, 1)):
        if pos0 == 40:   # again, with other rows
            k[40:48], v[40:48] = kv_rows(rng, 8, n_kv, hd)
        c.store(k[pos0:pos0 + n], v[pos0:pos0 + n], pos0, pad=pad)
        have[pos0:pos0 + n] = True
        for a, b in ((pos0, n), (max(0, pos0 - 1) if have[max(0, pos0 - 1)] else pos0, 1)):
            for which, x in ((0, k), (1, v)):
                np.testing.assert_array_equal(c.load(which, a, b, pad), R.cache_values(kind, x[a:a + b]).astype(np.float32))
    for which, (x, buf) in enumerate(((k, c.k), (v, c.v))):
        got = buf.read()
        if kind == Q4:
            was = before[which].reshape(n_kv, -(-ctx // 32), 18 * hd)
            np.testing.assert_array_equal(got.reshape(was.shape), R.q4_bytes(x, which == 1, was, have))
        else:
            width = n_kv * hd * (2 if kind == F16 else 4)
            np.testing.assert_array_equal(got.reshape(ctx, width)[~have], before[which].reshape(ctx, width)[~have])


@pytest.mark.parametrize("hd", [64, 128])
def test_q4_bytes_are_the_described_layout(hd):
    rng = np.random.default_rng(hd)
    k, v = kv_rows(rng, 70, 2, hd)
    c = Cache(Q4, 2, hd, 70, fill=0)
    c.store(k, v, 0)
    for buf, x, values in ((c.k, k, False), (c.v, v, True)):
        np.testing.assert_array_equal(buf.read().reshape(2, 3, 18 * hd), R.q4_bytes(x, values, np.zeros((2, 3, 18 * hd), np.uint8)))


@pytest.mark.parametrize("hd", [64, 128])
def test_q4_blocks_at_the_format_edges(hd):
    """Zeros, equal magnitudes of both signs, one element, the smallest and
    largest scales, infinities and NaN: the host quantizer's values, NaN where
    a block has no finite fp16 scale."""
    lib = _native.lib()
    x = np.zeros((40, 1, hd), np.float32)
    rng = np.random.default_rng(1)
    x[1], x[2] = 1.0, -1.0
    x[3, 0, ::2], x[3, 0, 1::2] = 2.0, -2.0
    x[4, 0, 1::2], x[4, 0, ::2] = 2.0, -2.0
    x[5, 0, 31] = 3e-5
    x[6] = rng.standard_normal(hd) * 1e-7
    x[7] = rng.standard_normal(hd) * 1e-40
    x[8] = rng.standard_normal(hd) * 1e5
    x[9, 0, 3] = 6e5
    x[10, 0, 7] = np.inf
    x[11, 0, 40] = -np.inf
    x[12, 0, 63] = np.nan
    x[13, 0, 0], x[13, 0, 1] = np.nan, np.inf
    x[14] = np.arange(hd) - hd / 2
    x[15:] = rng.standard_normal((25, 1, hd))
    c = Cache(Q4, 1, hd, 40)
    c.store(x, x[::-1].copy(), 0)
    got = c.load(0, 0, 40)
    np.testing.assert_array_equal(got, R.q4_values(x).astype(np.float32))
    np.testing.assert_array_equal(c.load(1, 0, 40), R.q4_values(x[::-1]).astype(np.float32))
    for i in [0, 1, 2, 3, 4, 5, 6, 8, 14, 20]:   # ember_quant_q4_row's blocks
        raw = np.zeros(hd // 32 * 18, np.uint8)
        row = x[i, 0].copy()
        lib.ember_quant_q4_row(row.ctypes.data_as(ctypes.POINTER(ctypes.c_float)), raw.ctypes.data, hd)
        b = raw.reshape(-1, 18)
        d = b[:, :2].copy().view(np.float16).astype(np.float32)
        codes = np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1).astype(np.float32)
        np.testing.assert_array_equal(got[i, 0], ((codes - 8) * d).reshape(-1))


@pytest.mark.parametrize("kind,hd", KINDS)
def test_cache_store_at_device_positions(kind, hd):
    """A position read on the device; tokens outside the cache store nothing."""
    rng = np.random.default_rng(5)
    ctx = 45
    k, v = kv_rows(rng, 10, 2, hd)
    for p in (0, 7, 40, 44, 45, 1000, -4, -10, -2 ** 31, 2 ** 31 - 1):
        c = Cache(kind, 2, hd, ctx, fill=0)
        pos = R.Buf(np.array([p], np.int32))
        c.store(k, v, 0, pos=pos.ptr)
        for which, x in ((0, k), (1, v)):
            want = np.zeros((ctx, 2, hd), np.float32)
            for i in range(10):
                if 0 <= p + i < ctx:
                    want[p + i] = R.cache_values(kind, x[i])
            got = c.load(which, 0, ctx)
            if kind == Q4:   # zero bytes are code 0 of scale 0: -0
                got = got + 0.0
            np.testing.assert_array_equal(got, want)


# ---------------------------------------------------------------- attend ----
def attend(c, q, pos0, window=0, sinks=0, scale=0.0, pos=None, stride=None, stream=None, ws=None, shift=0):
    lib, (n, nh, hd) = _native.lib(), q.shape
    w = nh * hd
    stride = stride or w
    qb = R.Buf(np.concatenate([np.zeros(shift, np.float32), np.pad(q.reshape(n, w), ((0, 0), (0, stride - w))).ravel()]))
    out = rows_buf(n, w, stride)
    need = lib.ehip_attend_workspace(c.c, nh, n)
    ws = ws or R.Buf(np.zeros(need, np.uint8))
    a = _native.EhipAttend(q=qb.ptr + 4 * shift, out=out.ptr, q_stride=stride, out_stride=stride, n_tok=n, n_heads=nh, pos0=pos0, window=window,
                           sinks=sinks, scale=scale, pos=pos, workspace=ws.ptr, workspace_bytes=ws.nbytes)
    ok(lib.ehip_attend(c.c, a, stream))
    R.hip().sync()
    assert not ws.nbytes or not ws.read()[:4096].any()   # the counters are zero again
    flat = out.read()
    assert untouched(flat, n, w, stride)
    return as_rows(flat, n, w, stride).reshape(n, nh, hd)


def check_attend(got, c, q, k, v, pos0, window=0, sinks=0, scale=0.0):
    end = pos0 + len(q)
    want, bound = R.attended(q, R.cache_values(c.kind, k[:end]), R.cache_values(c.kind, v[:end]), pos0, window, sinks, scale)
    err = np.abs(got - want)
    within(err, bound)


def filled(kind, hd, n_kv, n, ctx, seed):
    """A cache with n stored positions of ctx; what lies behind them is NaN."""
    rng = np.random.default_rng(seed)
    c = Cache(kind, n_kv, hd, ctx, fill=0xff)
    k, v = kv_rows(rng, n, n_kv, hd)
    c.store(k, v, 0)
    return c, k, v, rng


@pytest.mark.parametrize("kind,hd", KINDS)
@pytest.mark.parametrize("G,n_kv", [(1, 2), (2, 1), (7, 1), (8, 2), (3, 3), (20, 1)])
def test_attend_single_tokens(kind, hd, G, n_kv):
    """One token at the first positions, at tile borders and behind many tiles
    (ranges over workgroups, joined by the last)."""
    c, k, v, rng = filled(kind, hd, n_kv, 1400, 1411, G)
    for pos0 in (0, 1, 15, 16, 31, 32, 33, 127, 128, 500, 1399):
        q = (1.5 * rng.standard_normal((1, G * n_kv, hd))).astype(np.float32)
        check_attend(attend(c, q, pos0), c, q, k, v, pos0)


@pytest.mark.parametrize("kind,hd", KINDS)
@pytest.mark.parametrize("G,n,pos0", [(1, 2, 0), (1, 8, 5), (2, 4, 60), (2, 5, 0), (3, 3, 100), (4, 2, 31), (1, 33, 0), (2, 40, 17), (3, 23, 517),
                                      (7, 61, 0), (1, 200, 3), (2, 300, 0)])
def test_attend_several_tokens(kind, hd, G, n, pos0):
    c, k, v, rng = filled(kind, hd, 2, pos0 + n, pos0 + n + 3, n)
    q = rng.standard_normal((n, G * 2, hd)).astype(np.float32)
    check_attend(attend(c, q, pos0), c, q, k, v, pos0)


@pytest.mark.parametrize("kind,hd", KINDS)
@pytest.mark.parametrize("n,pos0,window,sinks", [(1, 0, 1, 0), (1, 700, 1, 0), (1, 700, 1, 1), (1, 700, 33, 4), (1, 700, 64, 0), (1, 40, 64, 4), (1, 700, 300, 200),
                                                 (1, 700, 10, 1000), (1, 700, 701, 0), (1, 700, 2000, 4), (50, 650, 32, 4), (50, 650, 31, 33),
                                                 (130, 0, 16, 1), (130, 0, 40, 0), (130, 300, 100, 64), (64, 600, 1, 0)])
def test_attend_windows_and_sinks(kind, hd, n, pos0, window, sinks):
    c, k, v, rng = filled(kind, hd, 2, 701, 720, n + window)
    q = rng.standard_normal((n, 4, hd)).astype(np.float32)
    check_attend(attend(c, q, pos0, window, sinks), c, q, k, v, pos0, window, sinks)


@pytest.mark.parametrize("kind,hd", KINDS)
def test_attend_reads_only_what_it_sees(kind, hd):
    """NaN and infinities at positions that a row does not see (later tokens of
    the call, behind the window, never stored) leave it alone; rows that see
    them are not finite."""
    for n, pos0, window, sinks, bad in ((1, 300, 32, 2, (5, 200, 268)), (70, 64, 0, 0, (100, 130)), (70, 200, 20, 3, (150, 231, 3)), (9, 40, 0, 0, (44, 48))):
        c, k, v, rng = filled(kind, hd, 1, pos0 + n, pos0 + n + 40, n)
        q = rng.standard_normal((n, 2, hd)).astype(np.float32)
        kb, vb = k.copy(), v.copy()
        for i, b in enumerate(bad):
            kb[b] = (np.nan, np.inf, -np.inf)[i % 3]
            vb[b, 0, ::3] = (np.inf, np.nan, -np.inf)[i % 3]
        c.store(kb, vb, 0)
        p = pos0 + np.arange(n)[:, None]
        sees = np.zeros(n, bool)
        for b in bad:
            sees |= ((b <= p) & ((b > p - window) | (b < sinks) if window else True))[:, 0]
        assert sees.any() or n == 1
        got = attend(c, q, pos0, window, sinks)
        assert not np.isfinite(got[sees]).all(-1).any()
        clean = ~sees
        want, bound = R.attended(q, R.cache_values(kind, k), R.cache_values(kind, v), pos0, window, sinks)
        within(np.abs(got - want)[clean], bound[clean])


@pytest.mark.parametrize("kind,hd", [(F32, 64), (F16, 128), (Q4, 128), (Q4, 64)])
def test_attend_scales_of_rows(kind, hd):
    """Large and tiny queries, values from tiny to large within a row's reach
    (the split's exponents move), a flat softmax, a peaked one, a negative and
    a custom scale, and a row of zeros."""
    c, k, v, rng = filled(kind, hd, 1, 400, 400, 9)
    v = (v * np.exp2(rng.integers(-12, 9, (400, 1, 1)))).astype(np.float32)
    v[:64] *= np.float32(1e-3)
    c.store(k, v, 0)
    for n in (1, 5, 20, 64):
        q = rng.standard_normal((n, 2, hd)).astype(np.float32)
        for f in (0.0, 1e-30, 1e-3, 1.0, 12.0):
            check_attend(attend(c, q * np.float32(f), 300), c, q * np.float32(f), k, v, 300)
        for scale in (-0.07, 0.5):
            check_attend(attend(c, q, 300, scale=scale), c, q, k, v, 300, scale=scale)


@pytest.mark.parametrize("kind,hd", KINDS)
def test_attend_strides_positions_streams_and_workspaces(kind, hd):
    """Padded and unaligned rows, a position on the device (with rows outside
    the cache, which are zeros), another stream, one workspace for calls of
    many shapes one after the other."""
    c, k, v, rng = filled(kind, hd, 2, 330, 330, 2)
    lib = _native.lib()
    ws = R.Buf(np.zeros(max(lib.ehip_attend_workspace(c.c, 6, n) for n in (1, 2, 5, 20, 330)), np.uint8))
    stream = R.hip().stream()
    for n, pos0 in ((1, 329), (5, 310), (20, 100), (2, 3), (1, 200)):
        q = rng.standard_normal((n, 6, hd)).astype(np.float32)
        want = attend(c, q, pos0)
        check_attend(want, c, q, k, v, pos0)
        np.testing.assert_array_equal(attend(c, q, pos0, stride=6 * hd + 12, ws=ws), want)
        np.testing.assert_array_equal(attend(c, q, pos0, stride=6 * hd + 5, shift=1, stream=stream, ws=ws), want)
        pos = R.Buf(np.array([pos0], np.int32))
        got = attend(c, q, 0, pos=pos.ptr, ws=ws)
        check_attend(got, c, q, k, v, pos0)
    q = rng.standard_normal((20, 6, hd)).astype(np.float32)
    for p in (320, 329, 330, 5000, -7, -20, -2 ** 31, 2 ** 31 - 1):
        pos = R.Buf(np.array([p], np.int32))
        got = attend(c, q, 0, pos=pos.ptr, ws=ws)
        for i in range(20):
            if 0 <= p + i < 330:
                check_attend(got[i:i + 1], c, q[i:i + 1], k, v, p + i)
            else:
                assert (got[i] == 0).all()
    R.hip().h.hipStreamDestroy(stream)


# Many rows over an fp32 cache: units of 128 rows, of 2048 tiles and more over
# all units.  (n, pos0, window, sinks, heads of a key head, key heads)
MANY = [(1, 1100, 0, 0, 4096, 2), (900, 0, 0, 0, 3, 8), (2200, 0, 0, 0, 1, 4), (333, 777, 0, 0, 7, 5), (130, 0, 16, 1, 512, 2), (64, 60, 1, 0, 1400, 3),
        (130, 300, 100, 64, 256, 2), (200, 1000, 777, 33, 8, 8), (130, 0, 40, 0, 515, 2)]


@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("n,pos0,window,sinks,G,n_kv", MANY)
def test_attend_many_rows_of_fp32(hd, n, pos0, window, sinks, G, n_kv):
    c, k, v, rng = filled(F32, hd, n_kv, pos0 + n, pos0 + n + 3, n + window)
    q = rng.standard_normal((n, G * n_kv, hd)).astype(np.float32)
    check_attend(attend(c, q, pos0, window, sinks), c, q, k, v, pos0, window, sinks)


@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("n,pos0,window,sinks,bad,G", [(70, 64, 0, 0, (100, 130), 1000), (70, 200, 20, 3, (150, 231, 3), 2000)])
def test_attend_many_rows_read_only_what_they_see(hd, n, pos0, window, sinks, bad, G):
    c, k, v, rng = filled(F32, hd, 1, pos0 + n, pos0 + n + 40, n)
    q = rng.standard_normal((n, G, hd)).astype(np.float32)
    kb, vb = k.copy(), v.copy()
    for i, b in enumerate(bad):
        kb[b] = (np.nan, np.inf, -np.inf)[i % 3]
        vb[b, 0, ::3] = (np.inf, np.nan, -np.inf)[i % 3]
    c.store(kb, vb, 0)
    p = pos0 + np.arange(n)
    sees = np.zeros(n, bool)
    for b in bad:
        sees |= (b <= p) & ((b > p - window) | (b < sinks) if window else True)
    assert sees.any() and not sees.all()
    got = attend(c, q, pos0, window, sinks)
    assert not np.isfinite(got[sees]).all(-1).any()
    want, bound = R.attended(q, k.astype(np.float64), v.astype(np.float64), pos0, window, sinks)
    within(np.abs(got - want)[~sees], bound[~sees])


@pytest.mark.parametrize("hd", [64, 128])
def test_attend_scales_of_many_rows(hd):
    c, k, v, rng = filled(F32, hd, 1, 400, 400, 9)
    v = (v * np.exp2(rng.integers(-12, 9, (400, 1, 1)))).astype(np.float32)
    v[:64] *= np.float32(1e-3)
    c.store(k, v, 0)
    q = rng.standard_normal((64, 360, hd)).astype(np.float32)
    for f in (0.0, 1e-30, 1e-3, 1.0, 12.0):
        check_attend(attend(c, q * np.float32(f), 300), c, q * np.float32(f), k, v, 300)
    for scale in (-0.07, 0.5):
        check_attend(attend(c, q, 300, scale=scale), c, q, k, v, 300, scale=scale)


@pytest.mark.parametrize("hd", [48, 128])
def test_attend_strides_and_positions_of_many_rows(hd):
    c, k, v, rng = filled(F32, hd, 2, 330, 330, 2)
    stream = R.hip().stream()
    n, heads = 20, 2 * 650
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    want = attend(c, q, 300)
    check_attend(want, c, q, k, v, 300)
    np.testing.assert_array_equal(attend(c, q, 300, stride=heads * hd + 12), want)
    np.testing.assert_array_equal(attend(c, q, 300, stride=heads * hd + 5, shift=1, stream=stream), want)
    for p in (300, 100, 3, 0, 320, 329, 330, 5000, -7, -20, -2 ** 31, 2 ** 31 - 1):
        pos = R.Buf(np.array([p], np.int32))
        got = attend(c, q, 0, pos=pos.ptr)
        a, b = max(0, -p), max(0, min(n, 330 - p))
        if a < b:
            check_attend(got[a:b], c, q[a:b], k, v, p + a)
        assert (got[:min(a, n)] == 0).all() and (got[max(b, 0):] == 0).all()
    R.hip().h.hipStreamDestroy(stream)


@pytest.mark.parametrize("kind,hd", [(F32, 64), (F16, 128), (Q4, 128), (Q4, 64)])
@pytest.mark.parametrize("step", [0.4, 1.9, 2.1, -1.5])
@pytest.mark.parametrize("n,heads", [(1, 2), (40, 2), (48, 500)])
def test_attend_a_rising_maximum(kind, hd, step, n, heads):
    """Scores that rise from tile to tile by less and by more (in powers of
    two) than the running maximum lags behind, or fall."""
    rng = np.random.default_rng(n)
    ctx = 400
    k, v = kv_rows(rng, ctx, 1, hd)
    v *= (1 + np.arange(ctx) % 7)[:, None, None].astype(np.float32)
    k *= np.float32(0.1)
    k[:, 0, 0] += (np.arange(ctx) // 32 * step).astype(np.float32)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    q[:, :, 0] = math.log(2) * math.sqrt(hd)
    c = Cache(kind, 1, hd, ctx)
    c.store(k, v, 0)
    check_attend(attend(c, q, ctx - n), c, q, k, v, ctx - n)


@pytest.mark.parametrize("kind,hd,n,heads", [(Q4, 128, 1, 2), (Q4, 128, 23, 4), (Q4, 64, 70, 14), (F16, 64, 9, 6), (F32, 64, 30, 6), (F32, 128, 40, 1300)])
def test_captured_calls_on_two_streams(kind, hd, n, heads):
    """Two captured calls with a workspace each, replayed at the same time on
    two streams with eager calls between: every replay gives the eager rows."""
    lib, h = _native.lib(), R.hip()
    c, k, v, rng = filled(kind, hd, 2, 700, 700, n)
    qs = [rng.standard_normal((n, heads, hd)).astype(np.float32) for _ in range(2)]
    at = (700 - n, 411)
    want = [attend(c, q, p) for q, p in zip(qs, at)]
    check_attend(want[0], c, qs[0], k, v, at[0])
    w = heads * hd
    bufs, outs = [R.Buf(q) for q in qs], [R.Buf(np.zeros((n, w), np.float32)) for _ in qs]
    spaces = [R.Buf(np.zeros(lib.ehip_attend_workspace(c.c, heads, n), np.uint8)) for _ in qs]
    calls = [_native.EhipAttend(q=b.ptr, out=o.ptr, q_stride=w, out_stride=w, n_tok=n, n_heads=heads, pos0=p, workspace=s.ptr, workspace_bytes=s.nbytes)
             for b, o, p, s in zip(bufs, outs, at, spaces)]
    streams = [h.stream() for _ in qs]
    made = [h.capture(s, lambda x=x, s=s: ok(lib.ehip_attend(c.c, x, s))) for x, s in zip(calls, streams)]
    for _ in range(4):
        for o in outs:
            o.write(np.full((n, w), 7, np.float32))
        for _ in range(3):
            for (_, run), s in zip(made, streams):
                assert h.h.hipGraphLaunch(run, s) == 0
        for s in streams:
            assert h.h.hipStreamSynchronize(s) == 0
        for o, x in zip(outs, want):
            np.testing.assert_array_equal(o.read().reshape(x.shape), x)
        np.testing.assert_array_equal(attend(c, qs[0], at[0]), want[0])
    for (graph, run), s in zip(made, streams):
        h.h.hipGraphExecDestroy(run)
        h.h.hipGraphDestroy(graph)
        h.h.hipStreamDestroy(s)


@pytest.mark.parametrize("kind,hd", KINDS)
def test_attend_long_caches(kind, hd):
    """Units of 8, 16 and 32 rows over 20,000 positions (many tiles to a wave,
    workgroups of eight waves over 4 bits), whole and behind a window."""
    c, k, v, rng = filled(kind, hd, 2, 20011, 20032, 3)
    for n, G in ((1, 2), (2, 4), (1, 12), (2, 8), (3, 7)):
        q = rng.standard_normal((n, 2 * G, hd)).astype(np.float32)
        check_attend(attend(c, q, 20011 - n), c, q, k, v, 20011 - n)
        check_attend(attend(c, q, 20011 - n, 9000, 70), c, q, k, v, 20011 - n, 9000, 70)


def test_attend_far_positions():
    """A token at the end of a long cache: 40,000 positions in 4 bits, and fp16
    rows whose offsets pass 2^31 bytes."""
    rng = np.random.default_rng(1)
    c = Cache(Q4, 2, 128, 40960, fill=0xff)
    k, v = kv_rows(rng, 40001, 2, 128)
    for a in range(0, 40001, 8000):
        c.store(k[a:a + 8000], v[a:a + 8000], a)
    q = rng.standard_normal((1, 4, 128)).astype(np.float32)
    check_attend(attend(c, q, 40000), c, q, k, v, 40000)
    check_attend(attend(c, q, 39990, 500, 4), c, q, k, v, 39990, 500, 4)
    del c
    ctx = (1 << 31) // (16 * 128 * 2) + 2000
    c = _native.EhipCache(type=F16, n_kv=16, head_dim=128, ctx=ctx)
    lib = _native.lib()
    n = lib.ehip_cache_bytes(c)
    assert n > 1 << 31
    h, p = R.hip().h, [ctypes.c_void_p(), ctypes.c_void_p()]
    for x in p:
        assert h.hipMalloc(ctypes.byref(x), n) == 0 and h.hipMemset(x, 0xff, n) == 0
    far = Cache(F16, 16, 128, 64)
    far.c, far.ctx = c, ctx
    far.c.k, far.c.v = p[0].value, p[1].value
    k, v = kv_rows(rng, 700, 16, 128)
    first = ctx - 700
    far.store(k, v, first)
    np.testing.assert_array_equal(far.load(1, first, 700), R.cache_values(F16, v).astype(np.float32))
    q = rng.standard_normal((3, 16, 128)).astype(np.float32)
    got = attend(far, q, ctx - 3, 600)
    want, bound = R.attended(q, R.cache_values(F16, k), R.cache_values(F16, v), 697, 600)
    within(np.abs(got - want), bound)
    for x in p:
        h.hipFree(x)


# ------------------------------------------------------ a run of them all ----
@pytest.mark.parametrize("kind,hd", [(F32, 64), (F16, 128), (Q4, 128), (Q4, 64)])
def test_a_captured_layer_step(kind, hd):
    """Rotary positions, the store and the attention of one token as one
    captured graph whose position advances on the device: every replay, with
    eager calls on the same buffers between them, gives the eager result."""
    lib, h = _native.lib(), R.hip()
    nh, n_kv, ctx = 4, 2, 90
    rng = np.random.default_rng(hd)
    cfg = config(N, scaling=3, factor=4.0, theta=1e5)
    plan = _native.EhipRopePlan()
    ok(lib.ehip_rope_plan(cfg, hd, plan))
    w = (nh + 2 * n_kv) * hd
    x, pos, out = R.Buf(np.zeros((1, w), np.float32)), R.Buf(np.zeros(1, np.int32)), R.Buf(np.zeros((1, nh * hd), np.float32))
    turned = R.Buf(np.zeros((1, (nh + n_kv) * hd), np.float32))
    caches = [Cache(kind, n_kv, hd, ctx, fill=0xff) for _ in range(2)]
    spaces = [R.Buf(np.zeros(lib.ehip_attend_workspace(caches[0].c, nh, 1), np.uint8)) for _ in range(2)]

    def step(c, ws, stream):
        r = _native.EhipRopeRows(x=x.ptr, out=turned.ptr, x_stride=w, out_stride=(nh + n_kv) * hd, n_tok=1, n_q=nh, n_k=n_kv, pos=pos.ptr)
        ok(lib.ehip_rope_rows(plan, r, stream))
        s = _native.EhipCacheRows(k=turned.ptr + 4 * nh * hd, v=x.ptr + 4 * (nh + n_kv) * hd, k_stride=0, v_stride=0, n_tok=1, pos=pos.ptr)
        ok(lib.ehip_cache_store(c.c, s, stream))
        a = _native.EhipAttend(q=turned.ptr, out=out.ptr, n_tok=1, n_heads=nh, pos=pos.ptr, window=40, sinks=3, workspace=ws.ptr, workspace_bytes=ws.nbytes)
        ok(lib.ehip_attend(c.c, a, stream))

    stream = h.stream()
    graph, run = h.capture(stream, lambda: step(caches[0], spaces[0], stream))
    ks, vs = np.zeros((2, ctx, n_kv, hd), np.float32)
    for p in range(ctx):
        row = rng.standard_normal((1, w)).astype(np.float32)
        x.write(row)
        pos.write(np.array([p], np.int32))
        assert h.h.hipGraphLaunch(run, stream) == 0 and h.h.hipStreamSynchronize(stream) == 0
        got, t = out.read(), turned.read()
        step(caches[1], spaces[1], None)
        h.sync()
        np.testing.assert_array_equal(got, out.read())
        ks[p], vs[p] = t[0, nh * hd:].reshape(n_kv, hd), row[0, (nh + n_kv) * hd:].reshape(n_kv, hd)
        check_rope(t, cfg, hd, row, nh, n_kv, np.array([p]))
        check_attend(got.reshape(1, nh, hd), caches[0], t[:, :nh * hd].reshape(1, nh, hd), ks, vs, p, 40, 3)
    h.h.hipGraphExecDestroy(run)
    h.h.hipGraphDestroy(graph)
    h.h.hipStreamDestroy(stream)
