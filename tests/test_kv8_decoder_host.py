"""What the decoder refuses before it touches a device."""
import pytest

from spirv_inference_b200 import llama


def test_logprobs_is_a_number():
    with pytest.raises(ValueError, match="a number"):
        llama.LlamaDecoder(llama.TINY_TEST, {}, 1, 4, 4, logprobs=True)


@pytest.mark.parametrize("head_dim", [32, 80, 96, 256])
def test_heads_of_other_sizes_in_8_bits(head_dim):
    cfg = llama.LlamaConfig(hidden=2 * head_dim, layers=1, heads=2, kv_heads=1, head_dim=head_dim,
                            ffn=64, vocab=50)
    with pytest.raises(ValueError, match="head_dim"):
        llama.LlamaDecoder(cfg, {}, 1, 4, 4, kv_cache="int8")
