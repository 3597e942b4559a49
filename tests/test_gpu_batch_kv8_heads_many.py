"""lcr_batch_norm_rope_write_kv8 with more rows than the device has waves for a head
each, so that a wave takes several heads of its rows: against the same rows in calls of
fewer, which tests/test_gpu_batch_kv8_heads.py holds to the definition, and where nothing
is rotated against the definition, bit for bit."""

import numpy as np
import pytest

import kv8_reference as ref
from helpers import dev, expect_bits_equal, host, to_f32
from test_gpu_batch_kv8_heads import Writer

pytestmark = pytest.mark.gpu

# kv heads and rows: 55 waves for 64 heads' keys and values, 32 for 64, 11 for 16
MANY = [(32, 4800), (32, 8200), (8, 24000)]


def sequences(w, rows):
    """Slots of sequences of 1 to 200 rows at any place in their pages, and their ends."""
    page, free = w.cache.page, list(w.r.permutation(w.cache.pool))
    slots, ends = [], []
    while len(slots) < rows:
        n, at = min(int(w.r.integers(1, 200)), rows - len(slots)), int(w.r.integers(0, page))
        pages = [free.pop() for _ in range((at + n - 1) // page + 1)]
        slots += [pages[(at + i) // page] * page + (at + i) % page for i in range(n)]
        ends.append(len(slots))
    return np.array(slots, np.int32), ends


def written(w, calls):
    """The cache's arrays and the queries after calls of (rows, positions, slots)."""
    c = w.cache
    c.upload(dev)
    queries = []
    for qkv, positions, slots in calls:
        out = dev(np.zeros(max(1, len(slots) * w.heads * c.d), np.uint16))
        w.launch(qkv, positions, slots, out)
        queries.append(host(out)[: len(slots) * w.heads * c.d])
    return [host(b, np.uint8) for b in c.on_device], np.concatenate(queries)


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv,rows", MANY)
def test_more_rows_than_waves(lcr, gpu, variant, d, kv, rows):
    w = Writer(lcr, variant, heads=2, kv=kv, d=d, page=32, pool=rows // 32 + 2 * rows // 100 + 60, norm=True, seed=rows)
    slots, ends = sequences(w, rows)
    positions = w.r.integers(0, len(w.table), rows).astype(np.int32)
    qkv = w.rows(rows)
    positions[5::97] = -1  # rows that are left alone
    whole, whole_q = written(w, [(qkv, positions, slots)])
    calls, start = [], 0
    for end in ends:
        if end - start > 900 or end == rows:
            calls.append((qkv[start:end], positions[start:end], slots[start:end]))
            start = end
    parts, parts_q = written(w, calls)
    for got, want, what in zip(whole, parts, ("keys", "values", "keys' scales", "values' scales")):
        expect_bits_equal(got, want, what)
    expect_bits_equal(whole_q, parts_q, "queries")
    before = [x.view(np.uint8) for x in (w.cache.keys, w.cache.values, w.cache.key_scales, w.cache.value_scales)]
    assert all((a != b).any() for a, b in zip(whole, before))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv,rows", MANY)
def test_more_rows_than_waves_by_definition(lcr, gpu, d, kv, rows):
    """Whole blocks, no norm and no rotation: scales and numbers are the definition's."""
    rows = rows // 16 * 16
    w = Writer(lcr, "bf16", heads=0, kv=kv, d=d, page=16, pool=rows // 16 + 3, norm=False, seed=rows + 1)
    w.table[:] = [1.0, 0.0]
    pages = w.r.permutation(w.cache.pool)[: rows // 16]
    slots = (16 * pages[:, None] + np.arange(16)).ravel().astype(np.int32)
    qkv = w.rows(rows)
    (keys, values, key_scales, value_scales), _ = written(w, [(qkv, np.zeros(rows, np.int32), slots)])
    x = to_f32(qkv).astype(np.float64).reshape(rows // 16, 16, 2, kv, d).transpose(2, 0, 3, 1, 4)
    for rows_of, got, got_scales, blocks_of in ((x[0], keys, key_scales, ref.to_blocks),
                                                (x[1], values, value_scales, ref.values_to_blocks)):
        largest = np.abs(rows_of).max((-1, -2))
        scales = 2.0 ** np.ceil(np.log2(largest / 448))
        assert (got_scales.view(np.float32)[w.cache.scales_at[pages][..., 0]] == scales).all()
        assert (blocks_of(got[w.cache.at[pages][:, :, 0]]) == ref.encode(rows_of / scales[..., None, None])).all()
