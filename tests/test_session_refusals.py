"""What the device-row operators refuse, and their host functions: no GPU is
needed, as every check comes before a launch."""
import ctypes
import math
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import session_ref as R  # noqa: E402

from emberllm_amd import _native  # noqa: E402

L = _native.lib()
P = 1 << 20          # a pointer that no refused call follows


def refused(rc, *words):
    assert rc != 0
    for w in words:
        assert w in _native.last_error(), _native.last_error()


def rope_config(**kw):
    return _native.EhipRopeConfig(**dict(dict(style=1, theta=1e4, factor=2.0, orig_ctx=100), **kw))


@pytest.mark.parametrize("kw,hd,word", [
    (dict(), 0, "head_dim"), (dict(), 65, "head_dim"), (dict(), 258, "head_dim"), (dict(rotary_dim=3), 64, "rotary_dim"),
    (dict(rotary_dim=66), 64, "rotary_dim"), (dict(rotary_dim=-2), 64, "rotary_dim"), (dict(style=2), 64, "style"),
    (dict(scaling=5), 64, "scaling"), (dict(scaling=-1), 64, "scaling"), (dict(theta=1.0), 64, "theta"),
    (dict(theta=math.inf), 64, "theta"), (dict(theta=math.nan), 64, "theta"), (dict(scaling=1, factor=0.5), 64, "factor"),
    (dict(scaling=1, factor=math.nan), 64, "factor"), (dict(scaling=2, rotary_dim=2), 64, "NTK"),
    (dict(scaling=3, orig_ctx=0), 64, "orig_ctx"), (dict(scaling=4, low=4.0, high=4.0), 64, "bounds"),
    (dict(scaling=3, low=0.0, high=4.0), 64, "bounds"), (dict(magnitude=-1.0), 64, "magnitude"),
    (dict(magnitude=math.inf), 64, "magnitude")])
def test_rope_plan_refuses(kw, hd, word):
    refused(L.ehip_rope_plan(rope_config(**kw), hd, _native.EhipRopePlan()), "ehip_rope_plan", word)


@pytest.mark.parametrize("scaling", range(5))
@pytest.mark.parametrize("hd,rd", [(128, 0), (64, 32), (48, 48), (256, 256)])
def test_rope_plan_frequencies(scaling, hd, rd):
    c = rope_config(scaling=scaling, rotary_dim=rd, factor=8.0, orig_ctx=4096, theta=5e5)
    plan = _native.EhipRopePlan()
    assert L.ehip_rope_plan(c, hd, plan) == 0
    f = R.frequencies(c, rd or hd)
    assert (plan.head_dim, plan.rotary_dim, plan.style) == (hd, rd or hd, 1)
    got = np.array([int(t) / 2.0 ** 64 * 2 * math.pi for t in plan.turns[:len(f)]])
    np.testing.assert_allclose(got, f, rtol=1e-14, atol=2.0 ** -60)   # steps of 2^-62 of a turn
    assert abs(plan.magnitude - R.magnitude(c)) < 1e-7 and not any(plan.turns[len(f):])


def test_rope_rows_refuses():
    plan = _native.EhipRopePlan()
    assert L.ehip_rope_plan(rope_config(), 64, plan) == 0
    good = dict(x=P, out=P, x_stride=256, out_stride=256, n_tok=2, n_q=3, n_k=1)
    rows = lambda **kw: _native.EhipRopeRows(**dict(good, **kw))  # noqa: E731
    refused(L.ehip_rope_rows(None, rows(), None), "null")
    refused(L.ehip_rope_rows(plan, None, None), "null")
    refused(L.ehip_rope_rows(_native.EhipRopePlan(), rows(), None), "plan")
    for kw, word in ((dict(n_tok=-1), "-1"), (dict(n_q=-1), "heads"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(x_stride=255), "strides"),
                     (dict(out_stride=0), "strides"), (dict(pos0=2 ** 31 - 1), "positions"), (dict(q_norm=P, eps=math.nan), "eps"),
                     (dict(n_q=2 ** 31 - 1, n_k=2 ** 31 - 1), "heads")):
        refused(L.ehip_rope_rows(plan, rows(**kw), None), "ehip_rope_rows", word)
    for kw in (dict(n_tok=0), dict(n_tok=0, x=None, out=None), dict(n_q=0, n_k=0)):
        assert L.ehip_rope_rows(plan, rows(**kw), None) == 0


BAD_CACHES = [(dict(type=3), "type"), (dict(type=-1), "type"), (dict(head_dim=48), "head_dim"), (dict(head_dim=0), "head_dim"),
              (dict(head_dim=256), "head_dim"), (dict(n_kv=0), "key heads"), (dict(n_kv=70000), "key heads"), (dict(ctx=0), "positions"),
              (dict(ctx=2 ** 30 + 1), "positions"), (dict(reserved=1), "reserved")]
BAD_POINTERS = [(dict(k=None), "null"), (dict(v=None), "null"), (dict(k=P + 8), "aligned")]


def cache(**kw):
    return _native.EhipCache(**dict(dict(k=P, v=P, ctx=100, type=2, n_kv=2, head_dim=64), **kw))


@pytest.mark.parametrize("kw,word", BAD_CACHES + BAD_POINTERS)
def test_every_call_refuses_a_bad_cache(kw, word):
    c = cache(**kw)
    refused(L.ehip_cache_store(c, _native.EhipCacheRows(k=P, v=P, k_stride=128, v_stride=128, n_tok=2), None), "ehip_cache_store", word)
    refused(L.ehip_cache_load(c, 0, 0, 2, P, 128, None), "ehip_cache_load", word)
    refused(L.ehip_attend(c, _native.EhipAttend(q=P, out=P, q_stride=256, out_stride=256, n_tok=1, n_heads=4), None), "ehip_attend", word)
    if (kw, word) in BAD_CACHES:
        assert L.ehip_cache_bytes(c) == 0 and word in _native.last_error()
        assert L.ehip_attend_workspace(c, 4, 1) == 0 and word in _native.last_error()


def test_cache_bytes():
    assert L.ehip_cache_bytes(cache(type=0)) == 100 * 128 * 4 and L.ehip_cache_bytes(cache(type=1)) == 100 * 128 * 2
    assert L.ehip_cache_bytes(cache()) == 4 * 2 * 64 * 18 and L.ehip_cache_bytes(cache(ctx=96, head_dim=128)) == 3 * 2 * 128 * 18
    assert L.ehip_cache_bytes(cache(type=0, ctx=2 ** 30, n_kv=65535, head_dim=128)) == 2 ** 30 * 65535 * 512
    assert L.ehip_cache_bytes(None) == 0


def test_cache_rows_refused():
    good = dict(k=P, v=P, k_stride=128, v_stride=128, n_tok=2)
    rows = lambda **kw: _native.EhipCacheRows(**dict(good, **kw))  # noqa: E731
    refused(L.ehip_cache_store(cache(), None, None), "null")
    refused(L.ehip_cache_store(None, rows(), None), "null")
    for kw, word in ((dict(n_tok=-1), "tokens"), (dict(n_tok=101), "tokens"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(k_stride=127), "strides"),
                     (dict(v_stride=127), "strides"), (dict(pos0=-1), "exceed"), (dict(pos0=99), "exceed"), (dict(pos0=2 ** 31 - 1), "exceed")):
        refused(L.ehip_cache_store(cache(), rows(**kw), None), "ehip_cache_store", word)
    assert L.ehip_cache_store(cache(), rows(n_tok=0, k=None), None) == 0
    for which, pos0, n, out, stride, word in ((2, 0, 1, P, 128, "neither"), (-1, 0, 1, P, 128, "neither"), (0, -1, 1, P, 128, "exceed"), (0, 0, -1, P, 128, "exceed"),
                                              (0, 99, 2, P, 128, "exceed"), (0, 2 ** 40, 1, P, 128, "exceed"), (1, 0, 1, None, 128, "null"), (1, 0, 2, P, 127, "stride")):
        refused(L.ehip_cache_load(cache(), which, pos0, n, out, stride, None), "ehip_cache_load", word)
    assert L.ehip_cache_load(cache(), 1, 100, 0, None, 0, None) == 0


def test_attend_refuses():
    good = dict(q=P, out=P, q_stride=256, out_stride=256, n_tok=2, n_heads=4, pos0=3)
    call = lambda **kw: _native.EhipAttend(**dict(good, **kw))  # noqa: E731
    refused(L.ehip_attend(cache(), None, None), "null")
    refused(L.ehip_attend(None, call(), None), "null")
    for kw, word in ((dict(n_tok=-1), "tokens"), (dict(n_tok=101), "tokens"), (dict(n_heads=3), "query heads"), (dict(n_heads=0), "query heads"),
                     (dict(n_heads=-2), "query heads"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(q_stride=255), "strides"),
                     (dict(out_stride=255), "strides"), (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(scale=math.nan), "scale"),
                     (dict(scale=math.inf), "scale"), (dict(pos0=-1), "exceed"), (dict(pos0=99), "exceed"), (dict(pos0=2 ** 31 - 1), "exceed")):
        refused(L.ehip_attend(cache(), call(**kw), None), "ehip_attend", word)
    assert L.ehip_attend(cache(), call(n_tok=0, q=None), None) == 0
    big = cache(ctx=4096)   # shared by workgroups: a workspace is needed
    need = L.ehip_attend_workspace(big, 4, 2)
    assert need > 4096
    for kw in (dict(), dict(workspace=P), dict(workspace=P, workspace_bytes=4096), dict(workspace=P + 8, workspace_bytes=need)):
        refused(L.ehip_attend(big, call(pos0=4000, **kw), None), "workspace")


def test_attend_refuses_what_no_launch_holds():
    c = cache(type=1, head_dim=48, n_kv=65535, ctx=1 << 30)   # fp16: units of 32 rows
    n = 1 << 20
    a = _native.EhipAttend(q=P, out=P, q_stride=65535 * 48, out_stride=65535 * 48, n_tok=n, n_heads=65535, workspace=P, workspace_bytes=1 << 40)
    assert L.ehip_attend(c, a, None) != 0 and "threads" in _native.last_error()


def test_attend_workspace_covers_every_call():
    """No call of up to n tokens at any position asks for more than
    ehip_attend_workspace(n) (the refusal names what a call needs)."""
    rng = np.random.default_rng(0)
    for _ in range(300):
        kind, hd = [(0, 48), (0, 128), (1, 64), (2, 64), (2, 128)][rng.integers(5)]
        n_kv, G = int(rng.choice([1, 2, 3, 8])), int(rng.choice([1, 2, 3, 7, 8, 20]))
        ctx = int(2 ** rng.uniform(0, 16))
        c = cache(type=kind, head_dim=hd, n_kv=n_kv, ctx=ctx)
        most = int(rng.integers(1, min(ctx, 400) + 1))
        need = L.ehip_attend_workspace(c, G * n_kv, most)
        for n in {1, most, int(rng.integers(1, most + 1)), int(rng.integers(1, min(most, 20) + 1))}:
            for kw in (dict(pos0=0), dict(pos0=ctx - n), dict(pos0=int(rng.integers(0, ctx - n + 1))), dict(pos=P),
                       dict(pos0=ctx - n, window=int(rng.integers(1, 3000)), sinks=int(rng.integers(0, 100)))):
                a = _native.EhipAttend(q_stride=G * n_kv * hd, out_stride=G * n_kv * hd, n_tok=n, n_heads=G * n_kv, **kw)
                assert L.ehip_attend(c, a, None) != 0   # its rows are null
                err = _native.last_error()
                if "workspace" in err:
                    assert int(err.split("this call's ")[1].split()[0]) <= need, (kind, hd, n_kv, G, ctx, most, n, kw)
                else:
                    assert "null rows" in err


def test_struct_layouts():
    assert ctypes.sizeof(_native.EhipRopePlan) == 1040 and _native.EhipRopePlan.turns.offset == 16
    assert _native.EhipAttend.pos.offset == 56 and _native.EhipCache.ctx.offset == 16
