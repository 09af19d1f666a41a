"""The decoder around the 8-bit cache: what one call leaves for the next."""
import numpy as np
import pytest

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
