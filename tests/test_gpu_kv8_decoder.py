"""The decoder around the 8-bit cache: what one call leaves for the next."""
import threading
from dataclasses import replace

import numpy as np
import pytest

import _kv8_np as N
from spirv_inference_b200 import llama

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_cache", ["fp32", "int8"])
@pytest.mark.parametrize("logprobs", [None, 0, 3])
def test_score_leaves_the_last_answer(gpu, kv_cache, logprobs):
    cfg = llama.TINY_TEST
    W = llama.make_weights(cfg, 2)
    a, b = (llama.make_prompt(cfg, 2, 20, seed=s) for s in (1, 2))
    dec = llama.LlamaDecoder(cfg, W, 2, 20, 6, device=gpu, logprobs=logprobs, kv_cache=kv_cache)
    try:
        def answer():
            lp = dec.token_logprobs() if logprobs is not None else {}
            return dict(lp, tokens=dec.tokens())

        def same(x, y):
            return x.keys() == y.keys() and all(np.array_equal(x[n], y[n]) for n in x)

        dec.generate(b)
        of_b = answer()
        dec.generate(a)
        of_a = answer()
        assert not np.array_equal(of_a["tokens"][:, 0], of_b["tokens"][:, 0])
        for top_k in (0, 2):
            dec.score(b, top_k=top_k)
            assert same(answer(), of_a)
        # ... and a step goes on from the text that was scored
        for _ in range(5):
            dec.decode_step()
        dec.g.sync()
        assert same(answer(), of_b)
        dec.score(a)
        dec.generate(a)
        assert same(answer(), of_a)
    finally:
        dec.close()


def test_logprobs_false_is_off(gpu):
    cfg = llama.TINY_TEST
    dec = llama.LlamaDecoder(cfg, llama.make_weights(cfg, 0), 1, 4, 2, device=gpu, logprobs=False)
    try:
        dec.generate(llama.make_prompt(cfg, 1, 4))
        with pytest.raises(ValueError):
            dec.token_logprobs()
    finally:
        dec.close()


class _Ranks:
    """The collectives of `world` decoders, each in a thread of this process, on the
    host: between a rank's kernels, none of which waits for another's."""

    def __init__(self, world):
        self.world, self.meet = world, threading.Barrier(world)
        self.part = [None] * world

    def exchange(self, rank, x):
        self.part[rank] = x
        self.meet.wait(timeout=60)
        parts = list(self.part)
        self.meet.wait(timeout=60)
        return parts


@pytest.mark.parametrize("world,batch,keep", [(2, 1, None), (2, 12, None), (2, 2, 24), (4, 1, None)])
def test_ranks_with_an_8_bit_cache(gpu, monkeypatch, world, batch, keep):
    """Heads over ranks (4 ranks: two kv heads, each held twice): every rank's tokens
    are the same, and the logits those of the restatement."""
    import torch
    import torch.distributed as dist
    cfg = replace(llama.TINY_TEST, max_seq=48 if keep else 64)
    W = llama.make_weights(cfg, 3)
    prompt = llama.make_prompt(cfg, batch, 30)
    ranks, got, errors, kept = _Ranks(world), {}, [], {}

    def all_reduce(self, t, rows):
        view = self._torch_view(t, rows, self.cfg.hidden)
        self.g.sync()
        parts = ranks.exchange(self.rank, view.cpu())
        view.copy_(sum(parts[1:], parts[0].clone()))
        torch.cuda.synchronize()

    def gather(out, part, group=None):
        group.g.sync()
        parts = ranks.exchange(group.rank, part.cpu())
        out.copy_(torch.cat([p.reshape(1, -1) for p in parts]).reshape(out.shape))
        torch.cuda.synchronize()

    monkeypatch.setattr(llama.LlamaDecoder, "_all_reduce", all_reduce)
    monkeypatch.setattr(dist, "all_gather_into_tensor", gather)

    def work(rank):
        try:
            extra = dict(kv_keep=keep, kv_recent=8, kv_sink=2) if keep else {}
            dec = llama.LlamaDecoder(cfg, W, batch, 30, 24, device=gpu, rank=rank, world=world,
                                     capture=False, kv_cache="int8", kv_block=16, **extra)
            dec.group = dec
            evict, kept[rank] = dec.g.kv8_evict, []

            def spy(cache, w, n, **kw):
                evict(cache, w, n, **kw)
                kept[rank].append(kw["idx"].download())
            dec.g.kv8_evict = spy
            try:
                got[rank] = dec.generate(prompt), dec.last_logits(), dec.sh
            finally:
                dec.close()
        except Exception as e:  # noqa: BLE001
            errors.append((rank, repr(e)))
            ranks.meet.abort()

    threads = [threading.Thread(target=work, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    toks = got[0][0]
    assert all(np.array_equal(got[r][0], toks) for r in range(world))
    last = np.concatenate([got[r][1] for r in range(world)], 1)
    rope = llama.rope_tables(cfg, 64)
    for b in range(min(batch, 2)):
        seen = {}

        def cut(li, h, w, n, b=b, seen=seen):
            i = seen[li, h] = seen.get((li, h), -1) + 1
            rank = next(r for r in range(world) if got[r][2].kv0 <= h < got[r][2].kv0 + got[r][2].nkv)
            return kept[rank][i * cfg.layers + li][b, h - got[rank][2].kv0]

        logits = N.decode(cfg, W, prompt[b], toks[b], rope, 16, cut=cut)
        for i, t in enumerate(toks[b]):
            top2 = np.sort(logits[i])[-2:]
            assert int(np.argmax(logits[i])) == int(t) or top2[1] - top2[0] < 1e-3, (b, i)
        assert np.abs(last[b] - logits[-1]).max() <= 1e-3 * np.abs(logits[-1]).max()
