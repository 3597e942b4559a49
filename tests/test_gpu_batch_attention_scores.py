"""lcr_batch_attention with scores of up to 2^26 in size: the largest has all the
weight, and its value comes out bit for bit (of its weight w, w v / w in fp32 is
off by 2^-22 at most, and v is a value of the element type)."""

import numpy as np
import pytest

from helpers import elems, expect_bits_equal
from test_gpu_batch_attention import Case
from test_gpu_batch_attention_cut import wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 72])
@pytest.mark.parametrize("size", [10, 20, 24, 26])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("past,new,positions", [(300, 2, 0), (700, 40, 0), (1500, 3, 1600), (1500, 40, 1600)])
def test_large_scores(lcr, gpu, variant, d, size, sign, past, new, positions):
    for heavy in (0, 40, past - 1):
        c = Case(variant, [past], [new], heads=4, kv=1, d=d, seed=95)
        if positions:
            wide(c, positions)
        c.scale = 0.125
        e = lambda x: elems(np.array([x], np.float32), c.kind)[0]  # noqa: E731
        # score = 2^14 k 2^-3: of the heavy key +-2^size, of others half of that, or twice
        c.q[:] = 0
        c.q[np.arange(c.tokens * c.heads) * d] = e(2.0 ** 14)
        c.keys[:] = 0
        for position in range(past + new):
            c.keys[c.position_index(0, 0, position)] = e(sign * 2.0 ** (size - 11) * (0.5 if sign > 0 else 1.0))
        at = c.position_index(0, 0, heavy)
        c.keys[at] = e(sign * 2.0 ** (size - 11) * (1.0 if sign > 0 else 0.5))
        got = c.run(lcr)
        expect_bits_equal(got, np.broadcast_to(c.values[at:at + d], got.shape), f"key {heavy}")
