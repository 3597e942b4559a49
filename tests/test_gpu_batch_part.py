"""Attention and draft verification of a part of a step's sequences: row starts
from the part's first sequence on, over the whole step's rows. The other
sequences' rows, before and behind, stay as they were."""

import ctypes

import numpy as np
import pytest

from helpers import dev, expect_bits_equal, host, p, rng
from test_gpu_batch_attention import Case
from test_gpu_batch_attention_cut import wide
from test_gpu_batch_verify import random_case, run_verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 72])
@pytest.mark.parametrize("positions", [0, 1100])
@pytest.mark.parametrize("new", [[3, 2, 1, 4, 2], [40, 2, 33, 0, 50]], ids=str)
def test_attention_of_some_sequences(lcr, gpu, d, positions, new):
    c = Case("bf16", [30, 400, 0, 77, 9], new, heads=4, kv=2, d=d, seed=80, tail=2)
    if positions:
        wide(c, positions)
    whole = c.check(lcr)
    lib = lcr.load_library("bf16")
    q, keys, values, tables = dev(c.q), dev(c.keys), dev(c.values), dev(c.tables)
    for lo, hi in ((0, 2), (2, 5), (1, 3), (4, 5)):
        out = dev(c.before)
        view = lcr.KvView(p(keys), p(values), p(tables) + 4 * lo * c.tables.shape[1], c.page, c.page_stride,
                          c.head_stride, c.kv, c.d)
        size = lib.lcr_batch_attention_workspace_bytes(hi - lo, c.tokens, max(new), 4, 2, d)
        ws = dev(np.full(size // 4 + 4, np.nan, np.float32))
        assert lib.lcr_batch_attention(
            p(out), p(q), ctypes.byref(view), p(dev(c.starts)) + 4 * lo, p(dev(c.lengths)) + 4 * lo, hi - lo, c.tokens,
            max(new), 4, 2, c.tables.shape[1], c.pool, c.q_stride, c.scale, p(ws), size, None) == 0
        got = host(out)[: c.tokens * 4 * d].reshape(c.tokens, 4, d)
        held = c.before[: got.size].reshape(got.shape)
        first, last = int(c.starts[lo]), int(c.starts[hi])
        expect_bits_equal(got[:first], held[:first], "the sequences before")
        expect_bits_equal(got[last:], held[last:], "the sequences behind")
        _, allow = c.want()
        ours = (got[first:last].astype(np.uint32) << 16).view(np.float32)
        assert (np.abs(ours - whole[first:last]) <= 2 * allow[first:last]).all()


def test_verification_of_some_sequences(gpu):
    r = rng(81)
    target, draft, ids, starts, accept, sample = random_case(r, [3, 1, 5, 2, 4, 5], 5000)
    heat = np.array([0.8, 0.0, 1.0, 1.2, 0.0, 0.7], np.float32)
    whole = run_verify(gpu, target, draft, ids, starts, heat, accept, sample, 4)
    for lo, hi in ((0, 2), (2, 6), (5, 6), (1, 4)):
        got = run_verify(gpu, target, draft, ids, starts[lo:hi + 1], heat[lo:hi], accept, sample[lo:hi], 4)
        assert got[0].tolist() == whole[0][lo:hi].tolist() and got[1].tolist() == whole[1][lo:hi].tolist()
