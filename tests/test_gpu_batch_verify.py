"""lcr_batch_verify against its definition in 64 bits: ids and counts, equal."""

import numpy as np
import pytest

import batch_reference
from helpers import dev, host, p, rng

pytestmark = pytest.mark.gpu

GUARD = 5


def run_verify(lib, target, draft, ids, row_starts, temperatures, accept, sample, max_draft, stride=None, shift=0,
               rows=None, stream=None, workspace=None):
    batch, vocab = len(row_starts) - 1, target.shape[1]
    rows = target.shape[0] if rows is None else rows
    stride = stride or vocab

    def spread(x):
        if x is None:
            return None
        # what lies between the rows is not looked at
        wide = np.full((x.shape[0], stride), np.float32(1e30))
        wide[:, :vocab] = x
        return p(dev(np.concatenate([np.zeros(shift, np.float32), wide.ravel()]).astype(np.float32))) + 4 * shift

    size = lib.lcr_batch_verify_workspace_bytes(batch, rows, vocab)
    ws = workspace or dev(np.full(size // 4 + 1, np.nan, np.float32))
    out_ids = dev(np.full(batch * (max_draft + 1) + GUARD, -9, np.int32))
    out_counts = dev(np.full(batch + GUARD, -9, np.int32))
    status = lib.lcr_batch_verify(
        p(out_ids), p(out_counts), spread(target), spread(draft), p(dev(np.asarray(ids, np.int32))),
        p(dev(np.asarray(row_starts, np.int32))), p(dev(np.asarray(temperatures, np.float32))),
        p(dev(np.asarray(accept, np.float32))), p(dev(np.asarray(sample, np.float32))), batch, rows, max_draft, vocab,
        stride, p(ws), size, stream)
    assert status == 0, lib.lcr_last_error_message()
    got, counts = host(out_ids, np.int32), host(out_counts, np.int32)
    assert (got[-GUARD:] == -9).all() and (counts[-GUARD:] == -9).all(), "written past the end"
    return got[:-GUARD].reshape(batch, max_draft + 1), counts[:-GUARD]


def check(lib, target, draft, ids, row_starts, temperatures, accept, sample, max_draft, **more):
    got = run_verify(lib, target, draft, ids, row_starts, temperatures, accept, sample, max_draft, **more)
    with np.errstate(over="ignore"):
        want = batch_reference.verify(target, draft, ids, row_starts, temperatures, accept, sample, max_draft)
    assert got[1].tolist() == want[1].tolist()
    assert got[0].tolist() == want[0].tolist()
    return want


def random_case(r, counts, vocab, noise=0.5, spread=2.5):
    """Row counts (drafts + 1) of the sequences; drafts drawn from their own
    distribution at temperature 1."""
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1])
    target = (spread * r.normal(size=(rows, vocab))).astype(np.float32)
    draft = (target + noise * r.normal(size=(rows, vocab))).astype(np.float32)
    ids = (draft + r.gumbel(size=draft.shape)).argmax(1).astype(np.int32)
    return target, draft, ids, starts, r.random(rows).astype(np.float32), r.random(len(counts)).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4095, 4096, 4097, 8192, 20001, 128256])
def test_verify_of_random_drafts(gpu, vocab):
    r = rng(vocab)
    counts = [5, 1, 3, 5, 2, 5, 4, 5] if vocab < 100000 else [5, 2, 4]
    target, draft, ids, starts, accept, sample = random_case(r, counts, vocab)
    heat = [(0.7, 0.0, 1.0, 1.3)[b % 4] for b in range(len(counts))]
    want = check(gpu, target, draft, ids, starts, heat, accept, sample, 4)
    if 100 < vocab < 100000:  # both ends are met
        assert (want[1] == counts).any() and (want[1] < counts).any()
    check(gpu, target, None, ids, starts, heat, accept, sample, 4)


@pytest.mark.parametrize("draft_like", ["near", "same", "far"])
def test_verify_over_many_draws(gpu, draft_like):
    """64 sequences over a flat vocabulary, where the running sum's intervals
    are narrow: every drawn id is the 64-bit one."""
    r = rng(7)
    noise = {"near": 0.3, "same": 0.0, "far": 3.0}[draft_like]
    target, draft, ids, starts, accept, sample = random_case(r, [3] * 64, 30000, noise, spread=1.0)
    want = check(gpu, target, draft, ids, starts, [1.0] * 64, accept, sample, 2)
    if draft_like == "same":
        assert (want[1] == 3).all()
    if draft_like == "far":
        assert (want[1] == 1).sum() > 32


def test_verify_layouts(gpu):
    r = rng(8)
    target, draft, ids, starts, accept, sample = random_case(r, [4, 0, 1, 3, 0, 5], 5003)
    heat = [0.8, 1.0, 0.0, 1.1, 0.0, 0.9]
    for more in (dict(stride=5003), dict(stride=5004), dict(stride=6001), dict(stride=5004, shift=1),
                 dict(stride=5004, shift=4)):
        want = check(gpu, target, draft, ids, starts, heat, accept, sample, 4, **more)
        assert want[1][1] == 0 and (want[0][1] == -1).all()


def test_verify_takes_at_most_max_draft(gpu):
    r = rng(9)
    target, draft, ids, starts, accept, sample = random_case(r, [6, 2, 9], 700, noise=0.05)
    for most in (0, 1, 3, 20):
        check(gpu, target, draft, ids, starts, [1.0, 0.0, 0.7], accept, sample, most)


def test_verify_leaves_rows_behind_the_last_sequence(gpu):
    r = rng(10)
    target, draft, ids, starts, accept, sample = random_case(r, [3, 2], 300)
    pad = lambda a, v: np.concatenate([a, np.full((4, *a.shape[1:]), v, a.dtype)])  # noqa: E731
    check(gpu, pad(target, np.nan), pad(draft, np.nan), pad(ids, 2 ** 30), starts, [1.0, 0.6], pad(accept, np.nan),
          sample, 4)


def test_verify_greedy_ties_and_specials(gpu):
    """Ties go to the lowest index; NaN counts as -inf; zeros of both signs tie."""
    vocab = 9000
    target = np.full((8, vocab), -3.0, np.float32)
    target[0, [4100, 70, 8999]] = 5.0
    target[1, [5000, 5001]] = -0.0, 0.0
    target[2, 4097], target[2, 10] = np.inf, np.nan
    target[3] = -np.inf
    target[4] = np.nan
    target[5, 17], target[5, 8200] = np.nan, 2.0
    target[6, [3, 4099]] = np.inf
    target[7, 4096] = 1e38
    best = [70, 5000, 4097, 0, 0, 8200, 3, 4096]
    for b, row in enumerate(best):
        rows = target[b:b + 1].repeat(2, 0)
        for x, count in ((row, 2), ((row + 1) % vocab, 1), (-1, 1), (vocab, 1), (2 ** 31 - 1, 1)):
            for heat in (0.0, -1.0, np.nan):
                got = run_verify(gpu, rows, None, [x, 0], [0, 2], [heat], [0.5, 0.5], [0.5], 1)
                assert got[1][0] == count and got[0][0].tolist() == ([x, row] if count == 2 else [row, -1]), (b, x)


def test_verify_sampled_specials(gpu):
    """Logits that are masked (-inf, the lowest value), infinite or NaN; a row
    without a distribution; drafts outside the vocabulary; draws at the ends."""
    r = rng(12)
    vocab = 6000
    low = np.finfo(np.float32).min
    cases = []
    for kind in ("masked", "lowest", "nan", "one left", "inf", "all -inf", "all nan"):
        target, draft, ids, starts, accept, sample = random_case(r, [2] * 6, vocab)
        for x in (target, draft):
            if kind in ("masked", "lowest"):
                x[:, r.random(vocab) < 0.7] = -np.inf if kind == "masked" else low
            elif kind == "nan":
                x[:, ::3] = np.nan
            elif kind == "one left":
                x[:] = -np.inf
                x[:, 4321] = 1.0
            elif kind == "inf":
                x[:, [4500, 77]] = np.inf
            else:
                x[:] = -np.inf if kind == "all -inf" else np.nan
        ids[::2] = [0, 4321, 77, -5, vocab, 4500]
        cases.append((kind, target, draft, ids, starts, accept, sample))
    for kind, target, draft, ids, starts, accept, sample in cases:
        top = np.nextafter(np.float32(1), np.float32(0))
        for u in (accept, np.zeros_like(accept), np.full_like(accept, top)):
            for s in (sample, np.zeros_like(sample), np.full_like(sample, top)):
                check(gpu, target, draft, ids, starts, [0.9] * 6, u, s, 1)
                check(gpu, target, None, ids, starts, [0.9] * 6, u, s, 1)


def test_verify_temperatures(gpu):
    r = rng(14)
    target, draft, ids, starts, accept, sample = random_case(r, [2] * 8, 3000)
    target[:, 5] = draft[:, 9] = -np.inf
    heat = [1e-6, 1e-30, 1e-45, 100.0, 1e30, np.inf, 0.5, 3e38]
    check(gpu, target, draft, ids, starts, heat, accept, sample, 1)


def test_verify_draw_that_is_no_number(gpu):
    """NaN draws keep no draft and give an id of the vocabulary that has weight."""
    r = rng(15)
    target, draft, ids, starts, _, _ = random_case(r, [3, 3], 500)
    target[:, 400:] = -np.inf
    got = run_verify(gpu, target, draft, ids, starts, [1.0, 1.0], [np.nan] * 6, [np.nan] * 2, 2)
    assert got[1].tolist() == [1, 1] and ((got[0][:, 0] >= 0) & (got[0][:, 0] < 400)).all()


def test_verify_draws_follow_the_target(gpu):
    """Kept and drawn first tokens together are distributed as the target's row:
    each frequency within 5 standard deviations of its share over 40000 draws."""
    r = rng(16)
    vocab, batch, rounds = 6, 4000, 10
    logits = np.array([1.0, 0.2, -0.5, 0.9, -2.0, 0.0], np.float32)
    other = np.array([0.0, 1.0, 0.5, 0.9, -1.0, -3.0], np.float32)
    p_row = batch_reference.distribution(logits, 0.8)
    seen = np.zeros(vocab)
    for _ in range(rounds):
        ids = (other / np.float32(0.8) + r.gumbel(size=(batch, vocab))).argmax(1).astype(np.int32)
        ids = np.stack([ids, np.zeros_like(ids)], 1).ravel()
        rows = 2 * batch
        got = run_verify(gpu, np.broadcast_to(logits, (rows, vocab)), np.broadcast_to(other, (rows, vocab)), ids,
                         np.arange(0, rows + 1, 2), [0.8] * batch, r.random(rows), r.random(batch), 1)
        seen += np.bincount(got[0][:, 0], minlength=vocab)
    n = batch * rounds
    assert (np.abs(seen - n * p_row) <= 5 * np.sqrt(n * p_row * (1 - p_row))).all(), seen / n
