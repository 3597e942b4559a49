"""lcr_batch_attention with row starts whose sequences overlap, as no lcr_batch_map
writes them: more work than 32 bits count."""

import ctypes

import numpy as np
import pytest

from helpers import dev, expect_bits_equal, host, p, random_elems, rng
from test_gpu_batch_attention import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("positions", [200704, 1024])  # units cut and joined; not cut
def test_row_starts_that_overlap(lcr, gpu, d, positions):
    """Every second sequence has all of the buffer's rows, which counts for more
    work than 32 bits hold. Nothing says what comes out; nothing is read or
    written out of bounds, and the next call is as it was."""
    tokens, batch, page = 200_000, 4096, 4096 if positions > 4096 else 1024
    stride = positions // page
    c = Case("bf16", [700, 20], [3, 40], heads=4, kv=2, d=d, seed=70)
    before = c.run(lcr)
    lib = lcr.load_library("bf16")
    starts = np.where(np.arange(batch + 1) % 2 == 0, 0, tokens).astype(np.int32)
    lengths = np.full(batch, tokens, np.int32)
    pool = stride * page * d
    keys, values = (dev(random_elems(rng(n), pool)) for n in (71, 72))
    tables = dev(np.tile(np.arange(stride, dtype=np.int32), (batch, 1)))
    guard = random_elems(rng(73), 4096)
    out = dev(np.concatenate([np.zeros(tokens * d, np.uint16), guard]))
    size = lib.lcr_batch_attention_workspace_bytes(batch, tokens, tokens, 1, 1, d)
    ws = dev(np.concatenate([np.zeros(size // 2, np.uint16), guard]))
    view = lcr.KvView(p(keys), p(values), p(tables), page, page * d, page * d, 1, d)
    status = lib.lcr_batch_attention(p(out), p(dev(random_elems(rng(74), tokens * d))), ctypes.byref(view),
                                     p(dev(starts)), p(dev(lengths)), batch, tokens, tokens, 1, 1, stride, stride, d,
                                     d ** -0.5, p(ws), size, None)
    assert status == 0, lib.lcr_last_error_message()
    expect_bits_equal(host(out)[tokens * d:], guard, "behind the output")
    expect_bits_equal(host(ws)[size // 2:], guard, "behind the workspace")
    expect_bits_equal(c.run(lcr), before, "the next call")
