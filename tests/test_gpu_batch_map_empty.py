"""lcr_batch_map of no sequences: a step like any other, whose outputs feed the
next one. Its row starts, rows and counts are written, whatever stands in the
arrays of sequences that it does not have."""

import numpy as np
import pytest

import batch_reference
from helpers import dev, host, p, rng
from test_gpu_batch_map import GUARD, MARK, check, random_batch

pytestmark = pytest.mark.gpu


def run_empty(lib, free_count, max_rows, free_capacity, arrays="all", stream=None):
    """The outputs of a call over stale buffers, with guards behind each."""
    out = {name: dev(np.full(n + GUARD, MARK, np.int32))
           for name, n in (("row_starts", 1), ("positions", max_rows), ("slots", max_rows), ("counts", 2))}
    other = [p(dev(np.full(8, MARK, np.int32))) if arrays != "none" else None for _ in range(7)]
    lengths_out, mapped_out, tables, lengths, new, mapped, free = other
    lengths = None if arrays == "some" else lengths
    status = lib.lcr_batch_map(p(out["row_starts"]), p(out["positions"]), p(out["slots"]), lengths_out, mapped_out,
                               p(out["counts"]), tables, lengths, new, mapped, free, p(dev(np.array([free_count], np.int32))),
                               0, max_rows, 4, 16, 9, free_capacity, stream)
    assert status == 0, lib.lcr_last_error_message()
    got = {}
    for name, buf in out.items():
        values = host(buf, np.int32)
        assert (values[-GUARD:] == MARK).all(), f"{name}: written past its end"
        got[name] = values[:-GUARD]
    return got


@pytest.mark.parametrize("arrays", ["all", "some", "none"])
@pytest.mark.parametrize("max_rows", [0, 1, 257, 200000])
@pytest.mark.parametrize("free_count,capacity,left", [(0, 0, 0), (3, 8, 3), (8, 8, 8), (100, 8, 8), (-4, 8, 0)])
def test_a_step_of_no_sequences(gpu, arrays, max_rows, free_count, capacity, left):
    got = run_empty(gpu, free_count, max_rows, capacity, arrays)
    assert got["row_starts"].tolist() == [0]
    assert got["counts"].tolist() == [0, left]
    assert (got["positions"] == -1).all() and (got["slots"] == -1).all()


def test_a_step_of_no_sequences_without_its_arrays(gpu):
    """Nothing to write to, nothing written."""
    assert gpu.lcr_batch_map(*[None] * 12, 0, 8, 4, 16, 9, 3, None) == 0
    assert gpu.lcr_batch_map(*[None] * 12, 0, 0, 4, 16, 9, 0, None) == 0


def test_steps_with_none_between_them(gpu):
    """The free count of a step of none is the next one's, in exchanged buffers:
    no page is handed out twice."""
    r = rng(21)
    page, stride = 4, 30
    lengths, _, mapped, tables, free, count, pool = random_batch(r, 6, page, 0, 0, spare_pages=120, extra_mapped=0)
    tables = np.full((6, stride), -1, np.int32)
    counts = [dev(np.array([0, count], np.int32)), dev(np.array([0, -1], np.int32))]
    free_dev = dev(np.asarray(free, np.int32))
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    for step in range(9):
        batch = 0 if step % 3 == 1 else 6
        new = r.integers(0, 7, 6).astype(np.int32)
        outs = [i32(np.full(7, MARK)), i32(np.full(60, MARK)), i32(np.full(60, MARK)), i32(np.full(6, MARK)),
                i32(np.full(6, MARK))]
        table_dev = i32(tables)
        now, then = counts[(step + 1) % 2], counts[step % 2]
        status = gpu.lcr_batch_map(*[p(o) for o in outs], p(now), p(table_dev), p(i32(lengths)), p(i32(new)),
                                   p(i32(mapped)), p(free_dev), p(then) + 4, batch, 60, stride, page, pool, len(free), None)
        assert status == 0
        want = batch_reference.batch_map(np.asarray(lengths, np.int32)[:batch], new[:batch],
                                         np.asarray(mapped, np.int32)[:batch], tables[:batch],
                                         np.asarray(free, np.int32), count, 60, page, pool)
        assert host(now, np.int32).tolist() == want["counts"].tolist()
        assert host(outs[0], np.int32)[: batch + 1].tolist() == want["row_starts"].tolist()
        assert host(outs[2], np.int32).tolist() == want["slots"].tolist()
        count = int(want["counts"][1])
        if batch:
            tables, mapped, lengths = host(table_dev, np.int32).reshape(6, stride), want["mapped_out"], want["lengths_out"]
        used = tables[tables >= 0]
        assert len(set(used.tolist())) == len(used) == pool - count


def test_map_after_an_empty_step_is_as_before(gpu):
    r = rng(22)
    run_empty(gpu, 5, 300, 8)
    lengths, new, mapped, tables, free, count, pool = random_batch(r, 65, 16, 90, 5)
    check(gpu, lengths, new, mapped, tables, free, count, int(new.sum()) + 3, 16, pool)
