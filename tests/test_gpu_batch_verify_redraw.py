"""lcr_batch_verify where a draft is refused and max(p - q, 0) is 0 everywhere:
the id is drawn a second time, from p, by the same blocks."""

import numpy as np
import pytest

import batch_reference
from helpers import rng
from test_gpu_batch_verify import check, random_case, run_verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [40, 1024, 5000, 40000])
def test_second_draws(gpu, vocab):
    """Target and draft agree and the draft is no id of the vocabulary."""
    r = rng(vocab)
    batch = 200 if vocab < 40000 else 64
    target, _, ids, starts, accept, sample = random_case(r, [2] * batch, vocab, spread=1.0)
    ids[::4], ids[2::4] = -1, vocab
    heat = 0.5 + r.random(batch)
    want = check(gpu, target, target, ids, starts, heat, accept, sample, 1)
    assert (want[1] == 1).all()
    for _ in range(8):
        got = run_verify(gpu, target, target, ids, starts, heat, accept, sample, 1)
        assert got[0].tolist() == want[0].tolist()


def test_second_draws_beside_first_ones(gpu):
    """Some sequences draw once, some twice, some keep their drafts."""
    r = rng(61)
    target, draft, ids, starts, accept, sample = random_case(r, [3] * 96, 9000, spread=1.0)
    same = np.repeat(np.arange(96) % 3 == 0, 3)
    draft[same] = target[same]
    ids[np.flatnonzero(same)[::3]] = 9000
    accept[np.repeat(np.arange(96) % 3 == 1, 3)] = np.nan
    with np.errstate(invalid="ignore"):
        want = batch_reference.verify(target, draft, ids, starts, [0.9] * 96, accept, sample, 2)
    for _ in range(8):
        got = run_verify(gpu, target, draft, ids, starts, [0.9] * 96, accept, sample, 2)
        assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()
