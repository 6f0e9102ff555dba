"""States with options (ember_state_new_options): their layers' rotation, cache
and attention against 64-bit recomputations of what the state captured, their
logits against an ordinary state's, and their loops, graphs and cache access."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import session_ref as R  # noqa: E402

from emberllm_amd import _native, configs, emberllm  # noqa: E402

pytestmark = pytest.mark.gpu
KIND = {"f32": _native.KV_F32, "f16": _native.KV_F16, "q4": _native.KV_Q4}


def wide(name, **kw):
    """Two layers whose passes of few tokens take the few-token products."""
    cfg = dict(configs.TINY["t_qwen3"], dim=256, hidden_dim=1056, n_heads=4, n_kv_heads=2, head_dim=64, qk_norm=0, tied=1, vocab_size=640, max_seq_len=400)
    cfg.update(kw)
    return configs.model_path("session_" + name, cfg), cfg


def model(name):
    if name == "w64":
        return wide(name)
    if name == "w128":
        return wide(name, head_dim=128, qk_norm=1, rope_style=_native.ROPE_INTERLEAVED)
    return configs.model_path(name), configs.ALL[name]


def rope_config(cfg, **kw):
    return _native.EhipRopeConfig(**dict(dict(style=cfg["rope_style"], theta=cfg["rope_theta"]), **kw))


def cached(eng, which, layer, n):
    """The first n positions as fp32 [n][n_kv][hd]."""
    h = eng.header
    raw = eng.kv_read(which, layer, n)
    if eng.kv == "q4":
        b = raw.reshape(-1, 18)
        d = b[:, :2].copy().view(np.float16).astype(np.float32)
        x = (np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1).astype(np.float32) - 8) * d
    else:
        x = raw.view(np.float16 if eng.kv == "f16" else np.float32).astype(np.float32)
    return x.reshape(n, h.n_kv_heads, h.head_dim)


def check_layer(eng, cfg, rc, layer, qkv, o, pos0, window, sinks):
    """Raw q|k|v rows and attention outputs of tokens at pos0 .. against the
    cache that the state holds."""
    n, nh, nkv, hd = len(qkv), cfg["n_heads"], cfg["n_kv_heads"], cfg["head_dim"]
    x = qkv.reshape(n, nh + 2 * nkv, hd)
    norms = np.ones((nh + nkv, hd)) if cfg["qk_norm"] else None   # the synthetic norms are 1
    pos = pos0 + np.arange(n)
    want, size = R.turned(rc, hd, x[:, :nh + nkv], pos, norms, cfg["norm_eps"])
    k, v = (cached(eng, w, layer, pos0 + n) for w in (0, 1))
    off = 24 * R.EPS * size[:, nh:]
    if eng.kv == "q4":   # a turned key within rounding of a code's border may take either: one step of its block
        np.testing.assert_array_equal(v[pos0:], R.q4_values(x[:, nh + nkv:]).astype(np.float32))
        steps = np.abs(want[:, nh:].reshape(n, nkv, -1, 32)).max(-1, keepdims=True) / 8 * np.ones(32)
        err = np.abs(k[pos0:] - R.q4_values(want[:, nh:].astype(np.float32)))
        assert (err <= 1.01 * steps.reshape(err.shape) + off).all() and (err > 1e-3 * steps.reshape(err.shape)).mean() < 1e-2
    else:
        half = 2.0 ** -11 if eng.kv == "f16" else 0
        assert (np.abs(k[pos0:] - want[:, nh:]) <= off + half * np.abs(want[:, nh:]) + 2.0 ** -25).all()
        np.testing.assert_array_equal(v[pos0:], R.cache_values(KIND[eng.kv], x[:, nh + nkv:]).astype(np.float32))
    ref, bound = R.attended(want[:, :nh], k, v, pos0, window, sinks)
    # the rows that the state turned carry 24 half steps of their own, where
    # the reference's are exact: attended()'s bound takes 40 of sum |q k|
    err = np.abs(o.reshape(ref.shape) - ref)
    assert (err <= 2 * bound).all(), (err.max(), (err / bound).max())


CASES = [("t_llama", "f32", 0, 0, None), ("t_gqa", "q4", 20, 3, None), ("t_qwen3", "f16", 0, 0, dict(scaling=3, factor=4.0, orig_ctx=96)),
         ("t_qwen3", "q4", 0, 0, None), ("t_f32", "f32", 16, 1, dict(rotary_dim=24)), ("t_f32", "f16", 0, 0, dict(scaling=1, factor=2.0)),
         ("t_bias", "q4", 33, 0, dict(scaling=4, factor=8.0, orig_ctx=64)), ("t_g7", "q4", 100, 5, dict(rotary_dim=32, scaling=2, factor=2.0)),
         ("w64", "q4", 64, 4, None), ("w128", "q4", 0, 0, dict(scaling=3, factor=2.0, orig_ctx=400)), ("w128", "f32", 40, 2, None),
         ("t_gqa", "q4", 0, 0, dict(rotary_dim=20)), ("t_qwen3", "f16", 30, 2, dict(rotary_dim=10)), ("t_f32", "f32", 0, 0, dict(rotary_dim=14))]


@pytest.mark.parametrize("name,kv,window,sinks,scaled", CASES)
def test_layers_of_a_state(name, kv, window, sinks, scaled):
    path, cfg = model(name)
    rc = rope_config(cfg, **(scaled or {}))
    eng = emberllm.Engine(path, ctx=0, kv=kv, window=window, sinks=sinks, rope=rc if scaled else None)
    rng = np.random.default_rng(len(name))
    V, ctx = cfg["vocab_size"], eng.ctx
    start = 0
    for n in (5, 1, ctx // 3, 17):   # passes behind each other
        for layer in (0, 1):
            eng.debug_capture_prefill(layer)
            logits = eng.prefill(rng.integers(0, V, n), start=start)
            assert np.isfinite(logits).all()
            qkv, p0 = eng.debug_read_prefill(1)
            o, _ = eng.debug_read_prefill(2)
            assert p0 == start and len(qkv) == n
            check_layer(eng, cfg, rc, layer, qkv, o, start, window, sinks)
        eng.debug_capture_prefill(-1)
        start += n
    for layer in (0, 1):
        eng.debug_capture(layer)
        for _ in range(3):
            assert np.isfinite(eng.forward(int(rng.integers(0, V)), start)).all()
            check_layer(eng, cfg, rc, layer, eng.debug_read(1)[None], eng.debug_read(2)[None], start, window, sinks)
            start += 1
    eng.close()


@pytest.mark.parametrize("name,kv", [("t_llama", "f32"), ("t_qwen3", "f16"), ("t_f32", "f32"), ("t_g7", "f32"), ("w64", "f16"), ("w128", "f32")])
def test_logits_of_an_ordinary_state(name, kv):
    """Without a window or scaling, an fp32 or fp16 cache gives an ordinary
    state's logits, to the noise of sums in another order (and of its fp32
    angles)."""
    path, cfg = model(name)
    eng, plain = emberllm.Engine(path, kv=kv), emberllm.Engine(path, kv_fp16=kv == "f16")
    rng = np.random.default_rng(1)
    rel = 1e-5 if cfg["dtype"] == _native.DT_F32 else 2e-2   # (quantized inputs: a last bit can move a code)
    start = 0
    for n in (9, 30):
        ids = rng.integers(0, cfg["vocab_size"], n)
        a, b = eng.prefill(ids, start), plain.prefill(ids, start)
        assert np.linalg.norm(a - b) <= rel * np.linalg.norm(b)
        start += n
    for _ in range(5):
        tok = int(rng.integers(0, cfg["vocab_size"]))
        a, b = eng.forward(tok, start), plain.forward(tok, start)
        assert np.linalg.norm(a - b) <= rel * np.linalg.norm(b)
        start += 1
    eng.close()
    plain.close()


@pytest.mark.parametrize("name,kv,window", [("t_qwen3", "q4", 0), ("t_gqa", "q4", 24), ("t_f32", "f32", 16), ("w64", "f16", 50), ("w128", "q4", 0)])
def test_graphs_and_device_loops(name, kv, window):
    """Passes, steps and device loops replayed from graphs equal plain
    launches, and the greedy loop the steps it stands for."""
    path, cfg = model(name)
    eng, plain = (emberllm.Engine(path, kv=kv, window=window, sinks=2) for _ in range(2))
    plain.set_graph(False)
    rng = np.random.default_rng(7)
    V = cfg["vocab_size"]
    for call in range(4):
        ids = rng.integers(0, V, 21)
        np.testing.assert_array_equal(eng.prefill(ids), plain.prefill(ids))
        for pos in (21, 22):
            tok = int(rng.integers(0, V))
            np.testing.assert_array_equal(eng.forward(tok, pos), plain.forward(tok, pos))
        tok = int(rng.integers(0, V))
        toks, _ = eng.generate_greedy(tok, 23, 19)
        again, _ = plain.generate_greedy(tok, 23, 19)
        np.testing.assert_array_equal(toks, again)
        t = tok
        for i in range(19):
            t = int(np.argmax(plain.forward(t, 23 + i)))
            assert t == toks[i]
    smp = [_native.EmberSampler() for _ in range(2)]
    for s in smp:
        eng.lib.ember_sampler_init(s, 0.9, 0.95, 20, 5)
    a, b = (e.generate_sampled(3, 0, 20, s)[0] for e, s in zip((eng, plain), smp))
    np.testing.assert_array_equal(a, b)
    assert eng.time_decode(0, 3) > 0 and eng.time_kernel(0, 30, 3) > 0 and eng.decode_fusion() == 0
    eng.close()
    plain.close()


@pytest.mark.parametrize("name,kv", [("t_qwen3", "q4"), ("t_gqa", "q4"), ("t_f32", "f16")])
def test_cache_access(name, kv):
    """A conversation's cache read from one state and written into another."""
    path, cfg = model(name)
    a, b = (emberllm.Engine(path, kv=kv) for _ in range(2))
    ids = np.random.default_rng(0).integers(0, cfg["vocab_size"], 37)
    a.prefill(ids)
    b.prefill(ids[::-1].copy())
    for layer in range(2):
        for which in (0, 1):
            rows = a.kv_read(which, layer, 37)
            b.kv_write(which, layer, rows)
            np.testing.assert_array_equal(b.kv_read(which, layer, 37), rows)
    np.testing.assert_array_equal(a.forward(5, 37), b.forward(5, 37))
    a.close()
    b.close()


def test_positions_behind_the_context_of_training():
    path, cfg = model("t_qwen3")
    rc = rope_config(cfg, scaling=_native.ROPE_YARN, factor=4.0, orig_ctx=96)
    eng = emberllm.Engine(path, ctx=10 ** 6, kv="q4", window=64, sinks=4, rope=rc)
    assert eng.ctx == 4 * 96
    toks, _ = eng.generate_greedy(1, 0, 384)
    assert len(toks) == 384 and np.isfinite(eng.forward(int(toks[-1]), 383)).all()
    eng.close()


def test_options_refused(monkeypatch):
    path, cfg = model("t_f32")

    def refused(word, **kw):
        with pytest.raises(RuntimeError, match=word):
            emberllm.Engine(path, **kw)

    refused("head_dim 48", kv="q4")
    refused("window", kv="f32", window=-1)
    refused("sinks", kv="f32", sinks=-3)
    refused("rotary_dim", kv="f32", rope=rope_config(cfg, rotary_dim=50))
    refused("factor", kv="f32", rope=rope_config(cfg, scaling=1, factor=0.0))
    with pytest.raises(ValueError):
        emberllm.Engine(path, kv="q8")
    lib = _native.lib()
    assert not lib.ember_state_new_options(None, 0, _native.EhipStateOptions()) and "null" in _native.last_error()
    assert not lib.ehip_state_create_options(None, 8, _native.EhipStateOptions()) and "null" in _native.last_error()
    monkeypatch.setenv("EHIP_ORDER", "reference")
    refused("EHIP_ORDER", kv="f32")
    monkeypatch.delenv("EHIP_ORDER")
    eng = emberllm.Engine(path, kv="f16", window=8)   # and goes on after refusals
    assert np.isfinite(eng.prefill([1, 2, 3])).all()
    eng.close()
