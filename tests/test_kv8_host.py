"""Host side of the 8-bit cache and of the token log probabilities: which
caches are taken, which arguments are refused, and the numpy restatement that
the GPU tests compare with.  Nothing here touches a device."""
import ctypes

import numpy as np
import pytest

import _kv8_np as N
from oracle import llama_ref as R
from spirv_inference_b200 import _lib, llama
from spirv_inference_b200.graph import DeviceTensor, Kv8Cache


def _struct(**kw):
    d = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, k_tail=4096, v_tail=4096, lens=4096,
             batch=2, kv_heads=4, max_seq=64, head_dim=64, block=32)
    d.update(kw)
    return _lib.Kv8CacheStruct(*d.values())


def test_supported_caches(spx_built):
    l = _lib.lib()
    for kw in (dict(), dict(head_dim=128), dict(block=16), dict(block=64), dict(block=128,
               max_seq=128), dict(k_scale=4100, lens=4100)):
        assert l.spx_kv8_supported(ctypes.byref(_struct(**kw))) == 1, kw


@pytest.mark.parametrize("kw,code", [
    (dict(k=0), "null"), (dict(lens=0), "null"), (dict(batch=0), "shape"),
    (dict(kv_heads=-1), "shape"), (dict(max_seq=0), "shape"), (dict(head_dim=80), "head_dim"),
    (dict(block=24), "block"), (dict(block=0), "block"), (dict(max_seq=80), "whole number"),
    (dict(k=4104), "aligned"), (dict(v_tail=4100), "aligned"),
    (dict(batch=1 << 20), "too large"), (dict(max_seq=(1 << 30) + 128), "too large")])
def test_refused_caches(spx_built, kw, code):
    assert _lib.lib().spx_kv8_supported(ctypes.byref(_struct(**kw))) == 0
    assert code in _lib.last_error()


def test_null_graph_and_null_cache(spx_built):
    l = _lib.lib()
    assert l.spx_kv8_supported(None) == 0
    c = ctypes.byref(_struct())
    bad = _lib.SPX_ERR_INVALID_ARGUMENT
    assert l.spx_op_rope_kv8_append(None, None, 0, None, None, 1, None, None, 1, 1, None, c) == bad
    assert l.spx_op_attention_kv8(None, None, c, None, 1, 1, 1.0, None, None, None) == bad
    assert l.spx_op_kv8_read(None, c, None, 0, None, 1, None, None) == bad
    assert l.spx_op_kv8_evict(None, c, None, 1, 0, 0, None, c, None) == bad
    assert l.spx_op_kv8_advance(None, None, None, None, 1, 1, 1) == bad
    assert l.spx_op_token_logprobs(None, None, 1, 1, 1, None, None, None, None, 0, None,
                                   None) == bad


def test_cache_object_checks_shapes():
    def t(shape, dtype=np.float32):
        return DeviceTensor(4096, shape, np.dtype(dtype), None)

    def make(**kw):
        d = dict(k=t((1, 2, 64, 64), np.int8), v=t((1, 2, 64, 64), np.int8), k_scale=t((1, 2, 2)),
                 v_scale=t((1, 2, 2)), k_tail=t((1, 2, 32, 64)), v_tail=t((1, 2, 32, 64)),
                 lens=t((1,), np.int32))
        d.update(kw)
        return Kv8Cache(**d, block=32)

    assert make().max_seq == 64
    for kw in (dict(v=t((1, 2, 32, 64), np.int8)), dict(k_scale=t((1, 2, 4))),
               dict(lens=t((1,))), dict(k_tail=t((1, 2, 16, 64))), dict(lens=t((2,), np.int32))):
        with pytest.raises(ValueError):
            make(**kw)
    with pytest.raises(ValueError):
        Kv8Cache(t((1, 2, 60, 64), np.int8), *[t((1,))] * 6, block=32)


def test_decoder_refuses_what_does_not_fit():
    cfg, W = llama.TINY_TEST, {}
    for kw in (dict(kv_cache="int4"), dict(kv_keep=16), dict(kv_cache="int8", kv_keep=64),
               dict(kv_cache="int8", kv_keep=16, kv_recent=14),
               dict(kv_cache="int8", kv_keep=16, kv_recent=-1), dict(logprobs=65),
               dict(logprobs=2, world=2)):
        with pytest.raises(ValueError):
            llama.LlamaDecoder(cfg, W, 1, 32, 20, **kw)
    with pytest.raises(ValueError):
        llama.LlamaDecoder(cfg, W, 1, 65, 20, kv_cache="int8", kv_keep=16)
    with pytest.raises(ValueError):
        llama.LlamaDecoder(cfg, W, 1, 60, 20, kv_cache="int8")


@pytest.mark.parametrize("block", [0, 8, 24, 256])
def test_decoder_refuses_blocks_of_other_sizes(block):
    cfg = llama.LlamaConfig(hidden=128, layers=1, heads=2, kv_heads=1, ffn=64, vocab=50,
                            max_seq=64)
    with pytest.raises(ValueError, match="kv_block"):
        llama.LlamaDecoder(cfg, {}, 1, 4, 4, kv_cache="int8", kv_block=block)


def test_restatement_of_the_cache():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((70, 64)).astype(np.float32)
    one, cut = N.Cache(96, 32, 64), N.Cache(96, 32, 64)
    one.append(x)
    for a, b in ((0, 1), (1, 40), (40, 63), (63, 64), (64, 70)):
        cut.append(x[a:b])
    assert np.array_equal(one.q8, cut.q8) and np.array_equal(one.scale, cut.scale)
    assert np.array_equal(one.values(), cut.values())
    v = one.values()
    assert np.array_equal(v[64:].astype(np.float32), x[64:])
    # half a step of the block's scale at most
    step = np.repeat(one.scale[:2].astype(np.float64), 32)[:, None]
    assert np.all(np.abs(v[:64] - x[:64]) <= step * (0.5 + 1e-6))
    # rows of one block keep their values exactly when they are moved together
    same = one.cut(np.arange(32))
    assert np.array_equal(same.values(), v[:32])
    # a NaN is not hidden
    x[3, 5] = np.nan
    bad = N.Cache(96, 32, 64)
    bad.append(x)
    assert np.isnan(bad.values()[:32]).all() and np.isfinite(bad.values()[32:]).all()


def test_restated_decoder_is_near_the_fp32_one():
    """8-bit K / V move the logits of the small configuration by little: the
    rounding is at most 1/254 of a block's largest value."""
    from dataclasses import replace
    cfg = replace(llama.TINY_TEST, layers=1, vocab=100)
    W = llama.make_weights(cfg, 0)
    rope = llama.rope_tables(cfg, cfg.max_seq)
    prompt = llama.make_prompt(cfg, 1, 40)[0]
    toks, want = R.generate_cached(cfg, W, prompt, 4, rope, forced=np.arange(4))
    got = N.decode(cfg, W, prompt, np.arange(4), rope, 16)
    err = np.abs(got - want).max() / np.abs(want).max()
    assert 0 < err < 2e-2
    # a tail as long as the prompt: nothing is rounded
    full = N.decode(cfg, W, prompt, np.arange(4), rope, 64)
    assert np.abs(full - want).max() <= 1e-4 * np.abs(want).max()


def test_choose():
    w = np.array([9, 1, 5, 5, 2, 5, 0, 0], float)
    assert N.choose(w, 8, 8, 2, 1).tolist() == list(range(8))
    assert N.choose(w, 8, 5, 2, 1).tolist() == [0, 2, 3, 6, 7]
    assert N.choose(w, 8, 3, 0, 0).tolist() == [0, 2, 3]
    assert N.choose(w, 4, 5, 2, 1).tolist() == [0, 1, 2, 3]
