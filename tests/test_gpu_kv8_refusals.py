"""Calls on the 8-bit cache that are refused before anything runs, and the largest
arguments that are not."""
import numpy as np
import pytest

from spirv_inference_b200 import _lib
from spirv_inference_b200.graph import Graph
from test_gpu_kv8 import Setup

pytestmark = pytest.mark.gpu


@pytest.fixture
def g(gpu):
    with Graph(gpu) as graph:
        yield graph


def test_new_tokens_and_rotated_queries_apart(g):
    s = Setup(g, 1, 1, 2, 64, 64, 32)
    both = g.alloc((3 * 4 * 64 + 3 * 2 * 64,))
    end = 3 * 4 * 64
    for qkv, q in ((0, 0), (0, 4 * 64), (0, end - 64), (3 * 2 * 64 - 64, 0)):
        with pytest.raises(_lib.SpxError) as e:
            g.rope_kv8_append(both.view((end,), qkv), 4 * 64, s.cos, s.sin, s.pos,
                              both.view((3, 2, 64), q), s.cache, q_len=3, q_heads=2)
        assert e.value.code == _lib.SPX_ERR_INVALID_ARGUMENT
    for qkv, q in ((0, end), (3 * 2 * 64, 0)):
        g.rope_kv8_append(both.view((end,), qkv), 4 * 64, s.cos, s.sin, s.pos,
                          both.view((3, 2, 64), q), s.cache, q_len=3, q_heads=2)
    g.sync()


def test_more_new_tokens_than_32_bits_add_up(g):
    """lens + q_len past 2^31: as many as the cache has slots."""
    most = 2 ** 31 - 1
    s = Setup(g, 3, 1, 1, 64, 64, 32, lens=[64, 64, 64])
    got = []
    for q_len in (0, most):
        k, v = g.alloc((3, 1, 64, 64)), g.alloc((3, 1, 64, 64))
        g.kv8_read(s.cache, k, v, count=64, q_len=q_len)
        got.append((k.download(), v.download()))
    assert np.abs(got[0][0]).max() > 1
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    s.cache.lens.upload(np.array([0, 3, 64], np.int32))
    g.kv8_advance(s.cache, q_len=most)
    assert s.cache.lens.download().tolist() == [64, 64, 64]
    s.cache.lens.upload(np.array([0, 3, 64], np.int32))
    g.kv8_advance(s.cache, q_len=most, new_lens=g.tensor(np.array([most, 2, most], np.int32),
                                                         np.int32), limit=most)
    assert s.cache.lens.download().tolist() == [most, 5, most]
