"""lcr_batch_verify where the temperature is small beside the spacing of floats
at a row's largest logit: every other logit of the row then weighs nothing, and
the largest keeps the probability that the definition in 64 bits gives it."""

import numpy as np
import pytest

from helpers import rng
from test_gpu_batch_verify import check, random_case, run_verify

pytestmark = pytest.mark.gpu

NEAR_ONE = np.nextafter(np.float32(1), np.float32(0))


@pytest.mark.parametrize("vocab", [5, 1024, 3000])
@pytest.mark.parametrize("heat", [1e-45, 1e-30, 1e-12, 5e-10, 1e-9, 2e-9, 1e-8, 1e-6, 1e-3])
def test_the_largest_is_kept_without_a_draft_distribution(gpu, vocab, heat):
    """The draft is the target's largest logit, which has all the weight."""
    r = rng(vocab)
    target, _, _, starts, _, sample = random_case(r, [3] * 4, vocab)
    target[:, r.integers(0, vocab, target.shape[0])] += 1.0
    best = target.argmax(1)
    target[np.arange(len(best)), best] += 3.0
    accept = np.full(len(best), NEAR_ONE)
    want = check(gpu, target, None, best, starts, [heat] * 4, accept, sample, 2)
    assert (want[1] == 3).all()


@pytest.mark.parametrize("largest,heat", [
    (1e9, 0.05), (1e9, 1.0), (1e10, 1.0), (3e38, 1.0), (3e38, 1e30), (-1e9, 0.05), (1e5, 1e-6), (20.0, 2e-9),
    (2.0 ** 24, 1e-3), (-2.0 ** 24, 1e-3), (0.0, 1e-45), (0.0, 1e-30), (1e-40, 1e-43), (1e-40, 1e-30), (8.0, 1e-9),
])
def test_rows_of_one_large_logit(gpu, largest, heat):
    """A forced token: its logit beside others far below, drafted by itself or by
    a model whose own largest is of another size, and others drafted instead."""
    r = rng(31)
    vocab = 2500
    target, draft, _, starts, _, sample = random_case(r, [3] * 4, vocab)
    at = r.integers(0, vocab, target.shape[0])
    rows = np.arange(target.shape[0])
    if largest < 100.0:
        target = -np.abs(target) * np.float32(max(2.0 * abs(largest), 1.0)) + np.float32(min(1.5 * largest, 0.0))
    target[rows, at] = np.float32(largest)
    assert (target.argmax(1) == at).all()
    for accept in (np.full(len(at), NEAR_ONE), np.full(len(at), np.float32(0.4)), np.zeros(len(at), np.float32)):
        for ids in (at, (at + 1) % vocab, draft.argmax(1)):
            check(gpu, target, None, ids, starts, [heat] * 4, accept, sample, 2)
            check(gpu, target, draft, ids, starts, [heat] * 4, accept, sample, 2)
            check(gpu, draft, target, ids, starts, [heat] * 4, accept, sample, 2)


@pytest.mark.parametrize("apart", [1, 300, 1024, 2900])
def test_ties_of_the_largest(gpu, apart):
    """Two equal largest logits share the draws evenly, in one part or in two."""
    vocab, batch = 4000, 64
    target = np.tile((2.5 * rng(33).normal(size=vocab)).astype(np.float32), (batch, 1))
    target[:, 70] = target[:, 70 + apart] = np.float32(20.0)
    for heat in (1e-45, 1e-30, 1e-9, 2e-9):
        sample = ((np.arange(batch) + 0.5) / batch).astype(np.float32)
        want = check(gpu, target, None, np.zeros(batch), np.arange(batch + 1), [heat] * batch, np.zeros(batch), sample, 0)
        assert (want[0][:, 0] == 70).sum() == (want[0][:, 0] == 70 + apart).sum() == batch // 2
    # half of the weight: kept below it, not above
    starts = np.arange(0, 2 * batch + 1, 2)
    accept = (np.arange(2 * batch) // 2 / batch).astype(np.float32)
    got = run_verify(gpu, target.repeat(2, 0), None, np.full(2 * batch, 70), starts, [1e-30] * batch, accept,
                     [0.25] * batch, 1)
    assert got[1].tolist() == [2 if b < batch // 2 else 1 for b in range(batch)]


@pytest.mark.parametrize("other", [np.nan, -np.inf])
def test_nothing_else_weighs(gpu, other):
    """NaN, -inf and what lies behind the vocabulary beside the largest."""
    vocab = 1500
    target = np.full((4, vocab), other, np.float32)
    target[:, 3], target[:, 1400] = 7.0, 6.0
    for heat in (1e-45, 1e-9, 1e-3):
        want = check(gpu, target, None, [3, 3, 1400, 3], [0, 2, 4], [heat] * 2, np.full(4, NEAR_ONE), [0.0, NEAR_ONE], 1)
        assert want[0].tolist() == [[3, 3], [3, -1]]


def test_drafts_of_a_cold_distribution(gpu):
    """q of the drafted token is 1, not a part's share of it: drafts that the
    target gives less than 1 are kept as often as it says."""
    r = rng(34)
    vocab, batch = 1000, 200
    target = np.tile(r.normal(size=vocab).astype(np.float32), (2 * batch, 1))
    target[:, 9] = 1e-9
    target[:, 8] = 0.0
    target[:] = np.where(np.arange(vocab) < 10, target, -np.inf)
    draft = np.tile(r.normal(size=vocab).astype(np.float32), (2 * batch, 1))
    draft[:, 9] = 1e9
    check(gpu, target, draft, np.full(2 * batch, 9), np.arange(0, 2 * batch + 1, 2), [0.5] * batch,
          r.random(2 * batch), r.random(batch), 1)
