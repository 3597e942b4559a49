"""lcr_batch_attention: an infinite value that a row sees with a weight too small
for the element type. By the definition the row's element is that infinity; it
may come out as NaN (a weight of 0 times infinity), but as no number."""

import numpy as np
import pytest

from helpers import elems, expect_bits_equal, to_f32
from test_gpu_batch_attention import Case
from test_gpu_batch_attention_cut import wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 72])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("below", [25.0, 200.0])  # under 2^-25, fp16's least weight; under fp32's
def test_infinities_of_no_weight(lcr, gpu, variant, d, value, below):
    for past, new, positions in (([37], [5], 0), ([0], [40], 0), ([100], [90], 0), ([1437], [5], 1100), ([1100], [90], 1100)):
        c = Case(variant, past, new, heads=4, kv=1, d=d, seed=50)
        if positions:
            wide(c, positions)
        # every query's first element is 8; a key of -k there alone scores -8 k scale
        first = np.arange(c.tokens * c.heads) * d
        c.q[first] = elems(np.array([8.0], np.float32), c.kind)[0]
        spoilt = [past[0] + new[0] - 2, 3]  # seen by the last two rows, by all
        for position in spoilt:
            at = c.position_index(0, 0, position)
            c.keys[at:at + d] = 0
            c.keys[at] = elems(np.array([-(below + 25.0) / (8.0 * c.scale)], np.float32), c.kind)[0]
            c.values[at:at + d] = 0
        clean = c.check(lcr)
        bits = c.run(lcr)
        late, early = (c.position_index(0, 0, position) for position in spoilt)
        c.values[late + 3] = elems(np.array([value], np.float32), c.kind)[0]
        got = c.run(lcr)
        expect_bits_equal(got[: new[0] - 2], bits[: new[0] - 2], "rows before the value")
        seen = to_f32(got[new[0] - 2:], c.kind)
        assert not np.isfinite(seen[..., 3]).any()
        assert (np.delete(seen, 3, -1) == np.delete(clean[new[0] - 2:], 3, -1)).all()
        if past[0] == 0:
            continue
        c.values[early + 7] = elems(np.array([value], np.float32), c.kind)[0]
        seen = to_f32(c.run(lcr), c.kind)
        assert not np.isfinite(seen[..., 7]).any()
        assert (np.delete(seen[: new[0] - 2], 7, -1) == np.delete(clean[: new[0] - 2], 7, -1)).all()
