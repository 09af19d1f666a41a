"""What the decoder refuses before it touches a device."""
import pytest

from spirv_inference_b200 import llama


def test_logprobs_is_a_number():
    with pytest.raises(ValueError, match="a number"):
        llama.LlamaDecoder(llama.TINY_TEST, {}, 1, 4, 4, logprobs=True)
