"""lcr_batch_map against its definition (tests/batch_reference.py), bit for bit:
every output array, the page tables, and what lies behind the arrays' ends."""

import numpy as np
import pytest

import batch_reference
from helpers import dev, expect_bits_equal, host, p, rng

pytestmark = pytest.mark.gpu

GUARD = 7  # elements behind each output that stay as they were
MARK = -77


def guarded(n):
    return dev(np.full(n + GUARD, MARK, np.int32))


def run_map(lib, lengths, new, mapped, tables, free, free_count, max_rows, page_size, pool_pages, stream=None):
    batch, stride = tables.shape
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    out = {"row_starts": guarded(batch + 1), "positions": guarded(max_rows), "slots": guarded(max_rows),
           "lengths_out": guarded(batch), "mapped_out": guarded(batch), "counts": guarded(2)}
    table_dev = dev(np.concatenate([tables.ravel(), np.full(GUARD, MARK)]).astype(np.int32))
    inputs = [i32(lengths), i32(new), i32(mapped), i32(free if len(free) else [0]), i32([free_count])]
    status = lib.lcr_batch_map(*[p(b) for b in out.values()], p(table_dev), *[p(b) for b in inputs], batch, max_rows,
                               stride, page_size, pool_pages, len(free), stream)
    assert status == 0, lib.lcr_last_error_message()
    got = {}
    for name, buf in {**out, "tables": table_dev}.items():
        values = host(buf, np.int32)
        assert (values[-GUARD:] == MARK).all(), f"{name}: written past its end"
        got[name] = values[:-GUARD]
    return got


def check(lib, lengths, new, mapped, tables, free, free_count, max_rows, page_size, pool_pages):
    a = [np.asarray(x, np.int32) for x in (lengths, new, mapped, tables, free)]
    got = run_map(lib, *a, free_count, max_rows, page_size, pool_pages)
    want = batch_reference.batch_map(*a[:4], a[4], free_count, max_rows, page_size, pool_pages)
    for name, values in want.items():
        expect_bits_equal(got[name], values, name)
    return want


def random_batch(r, batch, page_size, longest, most_new, spare_pages=2, extra_mapped=1):
    lengths = r.integers(0, longest + 1, batch)
    new = r.integers(0, most_new + 1, batch)
    mapped = -(-lengths // page_size) + r.integers(0, extra_mapped + 1, batch)
    stride = int(max((-(-(lengths + new) // page_size)).max(), mapped.max(), 1)) + 1
    need = int(np.maximum(-(-(lengths + new) // page_size) - mapped, 0).sum())
    held = int(mapped.sum())
    pool = held + need + spare_pages
    pages = r.permutation(pool)
    tables = np.full((batch, stride), -1)
    at = 0
    for b in range(batch):
        tables[b, : mapped[b]] = pages[at:at + mapped[b]]
        at += mapped[b]
    return lengths, new, mapped, tables, pages[held:], need + spare_pages, pool


@pytest.mark.parametrize("batch,page_size,longest,most_new", [
    (1, 16, 0, 1), (1, 16, 40, 1), (3, 1, 9, 4), (8, 16, 900, 1), (63, 7, 50, 9), (64, 16, 100, 5), (65, 32, 500, 3),
    (255, 16, 64, 2), (256, 8, 300, 33), (257, 16, 30, 130), (1000, 64, 4000, 5), (1024, 16, 0, 3), (4096, 16, 100, 3),
])
def test_map_of_random_batches(gpu, batch, page_size, longest, most_new):
    r = rng(batch * 1000 + page_size)
    lengths, new, mapped, tables, free, count, pool = random_batch(r, batch, page_size, longest, most_new)
    rows = int(new.sum())
    want = check(gpu, lengths, new, mapped, tables, free, count, rows + 5, page_size, pool)
    assert want["counts"][0] == batch and want["counts"][1] == 2
    # exactly as many rows, and none at all behind them
    check(gpu, lengths, new, mapped, tables, free, count, rows, page_size, pool)


@pytest.mark.parametrize("lack", ["pages", "rows", "table", "negative new", "negative length", "negative mapped"])
def test_map_stops_at_the_first_sequence_that_does_not_fit(gpu, lack):
    r = rng(11)
    lengths, new, mapped, tables, free, count, pool = random_batch(r, 70, 16, 200, 20, extra_mapped=0)
    at, max_rows, stride = 41, int(new.sum()), tables.shape[1]
    new[at] = 40
    if lack == "pages":
        count = int(np.maximum(-(-(lengths + new) // 16) - mapped, 0)[: at + 1].sum()) - 1
        max_rows += 100
    elif lack == "rows":
        count, free = 500, np.concatenate([free, np.arange(pool, pool + 500)])
        max_rows = int(new[: at + 1].sum()) - 1
    elif lack == "table":
        count, free, max_rows = 500, np.concatenate([free, np.arange(pool, pool + 500)]), max_rows + 100
        lengths[at] = stride * 16 - 39
    else:
        max_rows += 100
        {"negative new": new, "negative length": lengths, "negative mapped": mapped}[lack][at] = -1
    want = check(gpu, lengths, new, mapped, tables, free, count, max_rows, 16, pool + 500)
    assert want["counts"][0] == at


def test_map_places_nothing(gpu):
    r = rng(12)
    lengths, new, mapped, tables, free, count, pool = random_batch(r, 5, 16, 60, 9)
    lengths[0], new[0], mapped[0] = 16, 1, 1
    want = check(gpu, lengths, new, mapped, tables, free, 0, 50, 16, pool)
    assert want["counts"].tolist() == [0, 0] and (want["positions"] == -1).all()
    # a free list of no pages, and a count beyond its list
    check(gpu, lengths, new, mapped, tables, np.zeros(0), 3, 50, 16, pool)
    check(gpu, lengths, new, mapped, tables, free, 10 ** 9, 50, 16, pool)
    check(gpu, lengths, new, mapped, tables, free, -4, 50, 16, pool)


def test_map_of_pages_outside_the_pool(gpu):
    """Their positions come out, their slots are -1."""
    tables = np.array([[3, -1, -1], [9, 1, -1]])
    want = check(gpu, [15, 15], [2, 2], [1, 2], tables, [4, 12], 2, 8, 16, 9)
    assert want["slots"].tolist() == [3 * 16 + 15, -1, -1, 16, -1, -1, -1, -1]


def test_map_steps_follow_each_other(gpu):
    """Outputs fed back as inputs over many steps, with rollbacks as rejected
    drafts give them: pages of a sequence never change, no page is held twice."""
    r = rng(13)
    batch, page, stride, pool = 9, 4, 30, 260
    lengths, mapped = np.zeros(batch, np.int32), np.zeros(batch, np.int32)
    tables = np.full((batch, stride), -1, np.int32)
    free, count = r.permutation(pool).astype(np.int32), pool
    for _ in range(12):
        new = r.integers(0, 9, batch).astype(np.int32)
        before = tables
        want = check(gpu, lengths, new, mapped, tables, free, count, 80, page, pool)
        tables, mapped, count = want["tables"], want["mapped_out"], int(want["counts"][1])
        for b in range(batch):
            held = before[b] >= 0
            assert (tables[b][held] == before[b][held]).all()
        used = tables[tables >= 0]
        assert len(set(used.tolist())) == len(used) == pool - count
        lengths = want["lengths_out"] - np.minimum(new, r.integers(0, 4, batch)).astype(np.int32)
