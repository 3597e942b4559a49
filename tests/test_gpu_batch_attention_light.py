"""lcr_batch_attention where one key outweighs each of many others by up to e^20,
and their sum counts all the same: weights of 2^-25 and less of the largest."""

import numpy as np
import pytest

from helpers import elems, to_f32
from test_gpu_batch_attention import Case

pytestmark = pytest.mark.gpu

# Weights are held against a largest of 128 at least in fp16, whose subnormals
# end at 2^-24: off by 2^-25 / 128 of the largest each; exact in size for bf16
# and where no matrix core takes part.
LEAST = {"fp16": 2.0 ** -32, "bf16": 0.0}


@pytest.mark.parametrize("variant", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 72])
@pytest.mark.parametrize("below", [10.0, 16.0, 17.0, 17.3, 18.0, 20.0])
@pytest.mark.parametrize("past,new,at", [(40000, 1, 0), (40000, 1, 39000), (9000, 30, 5)])
def test_many_light_keys(lcr, gpu, variant, d, below, past, new, at):
    c = Case(variant, [past], [new], heads=2, kv=1, d=d, page=64, seed=90)
    e = lambda x: elems(np.array([x], np.float32), c.kind)[0]  # noqa: E731
    # scores: 8 k scale at the heavy key, 0 elsewhere
    c.q[:] = 0
    c.q[np.arange(c.tokens * c.heads) * d] = e(8.0)
    c.keys[:] = 0
    heavy = c.position_index(0, 0, at)
    c.keys[heavy] = e(below / (8.0 * c.scale))
    c.values[:] = e(1.0)
    c.values[heavy:heavy + d] = 0
    gap = 8.0 * float(to_f32(c.keys[heavy:heavy + 1], c.kind)[0]) * np.float64(np.float32(c.scale))
    others = np.arange(past, past + new)        # visible keys but the heavy one
    light = np.exp(-gap)
    total = 1.0 + others * light
    want = others * light / total
    got = to_f32(c.run(lcr), c.kind).astype(np.float64)
    half = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}[variant]
    # the output's rounding; each light weight's, in the sum of values and in
    # that of weights; fp32 scores and exponents (2^-22 of the exponent's size);
    # fp32 sums of as many terms
    off = half + half * (1.0 + want) + 2 * (gap + 1) * 2.0 ** -22 * 1.5 + 2 * others * 2.0 ** -24
    allow = off * want + LEAST[variant] * others / total + 2.0 ** -25
    assert (np.abs(got - want[:, None, None]) <= allow[:, None, None]).all(), (got.ravel()[0], want[0], allow[0])
