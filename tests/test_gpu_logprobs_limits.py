"""Token log probabilities at the largest number of rows."""
import numpy as np
import pytest

from spirv_inference_b200.graph import Graph

pytestmark = pytest.mark.gpu


def test_rows_up_to_the_last_32_bit_number(gpu):
    """2^31 - 1 rows of one logit each, of which a token has log probability 0."""
    rows, part = 2 ** 31 - 1, 1 << 20
    with Graph(gpu) as g:
        x, out = g.alloc((rows,)), g.alloc((rows,))
        ends = [0, rows // 2, rows - part]
        for at in ends:
            x.view((part,), at).upload(np.full(part, 3.0, np.float32))
            out.view((part,), at).upload(np.full(part, 5.0, np.float32))
        g.token_logprobs(x, 1, rows, 1, None, None, entropy=out)
        for at in ends:
            assert np.all(out.view((part,), at).download() == 0.0)
