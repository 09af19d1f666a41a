"""Two host threads, each with a graph of its own, calling at the same time."""
import threading

import numpy as np
import pytest

from spirv_inference_b200.graph import Graph
from test_gpu_kv8 import Setup

pytestmark = pytest.mark.gpu


def test_attention_of_few_rows_from_two_threads(gpu):
    """One cache of 64 slots (four warps) and one of 1024 (eight): a launch's shared
    memory is not cut by the other's."""
    errors, outs = [], {}
    start = threading.Barrier(2)

    def work(S, seed):
        try:
            with Graph(gpu) as g:
                s = Setup(g, 1, 1, 8, 64, S, 32, lens=[S - 20], seed=seed)
                d_q, q = s.append(1)
                _, _, w = s.check_attention(d_q, q, [S - 20])
                out = g.alloc((1, 8, 64))
                g.attention_kv8(d_q, s.cache, out, q_len=1, q_heads=8, scale=0.125)
                want = out.download()
                start.wait(timeout=60)
                for i in range(20000):
                    g.attention_kv8(d_q, s.cache, out, q_len=1, q_heads=8, scale=0.125)
                    if i % 500 == 499:
                        g.sync()
                outs[S] = np.array_equal(out.download(), want)
        except Exception as e:  # noqa: BLE001
            errors.append((S, repr(e)))

    threads = [threading.Thread(target=work, args=a) for a in ((64, 1), (1024, 2))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert outs == {64: True, 1024: True}


def test_many_graphs_over_a_process(gpu):
    """More graphs than there are status words for attention of many rows, some at
    the same time: each syncs, and so does one that never ran it."""
    with Graph(gpu) as other:
        for _ in range(22):
            graphs = [Graph(gpu) for _ in range(50)]
            try:
                outs = []
                for g in graphs:
                    c = g.kv8_cache(1, 1, 64, 64, block=32)
                    for t in (c.k_tail, c.v_tail):
                        t.upload(np.ones(t.shape, np.float32))
                    q, out = g.tensor(np.ones((10, 8, 64), np.float32)), g.alloc((10, 8, 64))
                    g.attention_kv8(q, c, out, q_len=10, q_heads=8, scale=1.0)
                    outs.append(out)
                for g, out in zip(graphs, outs):
                    g.sync()
                    assert np.all(out.download() == 1.0)
                other.sync()
            finally:
                for g in graphs:
                    g.close()
