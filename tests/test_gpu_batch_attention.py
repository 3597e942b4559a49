"""lcr_batch_attention against its definition in 64 bits (tests/batch_reference.py
derives the allowance): lengths from one position up, ragged batches, head
layouts, page sizes, strides, rows that see nothing, masked infinities."""

import ctypes

import numpy as np
import pytest

import batch_reference
from helpers import BF16, FP16, dev, elems, expect_bits_equal, host, p, random_elems, rng, to_f32

pytestmark = pytest.mark.gpu

KINDS = {"bf16": BF16, "fp16": FP16}


class Case:
    """Random rows and caches of a batch: `past` cached positions and `new` rows
    each, pages in random order, every unused table entry a page of no use (-1)."""

    def __init__(self, variant, past, new, *, heads=32, kv=8, d=64, page=16, seed=1, q_scale=1.0, tail=0,
                 extra_stride=0, shift=0, page_pad=0, head_pad=0, spare=3):
        r = rng(seed)
        self.variant, self.kind = variant, KINDS[variant]
        self.heads, self.kv, self.d, self.page = heads, kv, d, page
        self.past, self.new = np.asarray(past), np.asarray(new)
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.lengths = (self.past + self.new).astype(np.int32)
        self.tokens = int(self.starts[-1]) + tail
        need = -(-np.maximum(self.lengths, 0) // page)
        self.pool = int(need.sum()) + spare
        order = r.permutation(self.pool).astype(np.int32)
        self.tables = np.full((len(self.past), max(1, int(need.max(initial=0)))), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n]
            at += n
        self.q_stride = heads * d + extra_stride
        self.shift = shift
        self.head_stride = page * d + head_pad
        self.page_stride = kv * self.head_stride + page_pad
        self.q = random_elems(r, self.tokens * self.q_stride + shift, q_scale, self.kind)
        self.keys = random_elems(r, self.pool * self.page_stride + shift, 1.0, self.kind)
        self.values = random_elems(r, self.pool * self.page_stride + shift, 1.0, self.kind)
        self.scale = d ** -0.5

    def cache_index(self, page, head, slot):
        return (self.shift + page * self.page_stride + head * self.head_stride + slot * self.d)

    def position_index(self, b, head, position):
        return self.cache_index(int(self.tables[b, position // self.page]), head, position % self.page)

    def run(self, lcr, workspace=True, max_new=None, stream=None, repeat=1):
        lib = lcr.load_library(self.variant)
        max_new = int(self.new.max(initial=0)) if max_new is None else max_new
        self.before = random_elems(rng(99), self.tokens * self.heads * self.d + 16, 1.0, self.kind)
        out, q, keys, values = dev(self.before), dev(self.q), dev(self.keys), dev(self.values)
        view = lcr.KvView(p(keys) + 2 * self.shift, p(values) + 2 * self.shift, p(dev(self.tables)), self.page,
                          self.page_stride, self.head_stride, self.kv, self.d)
        size = lib.lcr_batch_attention_workspace_bytes(len(self.past), self.tokens, max_new, self.heads,
                                                       self.heads // self.kv, self.d) if workspace else 0
        # a workspace may hold anything before a call
        ws = dev(np.full(size // 4 + 4, np.nan, np.float32)) if size else None
        starts, lengths = dev(self.starts), dev(self.lengths)
        for _ in range(repeat):
            status = lib.lcr_batch_attention(
                p(out), p(q) + 2 * self.shift, ctypes.byref(view), p(starts), p(lengths), len(self.past), self.tokens,
                max_new, self.heads, self.heads // self.kv, self.tables.shape[1], self.pool, self.q_stride, self.scale,
                p(ws) if ws else None, size, stream)
            assert status == 0, lib.lcr_last_error_message()
        got = host(out)
        expect_bits_equal(got[self.tokens * self.heads * self.d:], self.before[self.tokens * self.heads * self.d:],
                          "behind the output")
        return got[: self.tokens * self.heads * self.d].reshape(self.tokens, self.heads, self.d)

    def want(self):
        wide = lambda a: to_f32(a, self.kind).astype(np.float64)  # noqa: E731
        q = wide(self.q[self.shift:]).reshape(self.tokens, self.q_stride)[:, : self.heads * self.d]

        def pool(x):
            at = self.cache_index(np.arange(self.pool)[:, None, None], np.arange(self.kv)[:, None],
                                  np.arange(self.page))
            return wide(x)[at[..., None] + np.arange(self.d)]

        # entries of no use are never read
        with np.errstate(invalid="ignore"):
            return batch_reference.attention(q.reshape(self.tokens, self.heads, self.d), pool(self.keys),
                                             pool(self.values), np.maximum(self.tables, 0), self.starts, self.lengths,
                                             self.page, self.scale, self.variant)

    def check(self, lcr, **more):
        got = self.run(lcr, **more)
        want, allow = self.want()
        live = int(self.starts[-1])
        expect_bits_equal(got[live:], self.before[: self.tokens * self.heads * self.d].reshape(got.shape)[live:],
                          "rows behind the last sequence")
        ours = to_f32(got[:live], self.kind).astype(np.float64)
        off = np.abs(ours - want[:live])
        good = off <= allow[:live]
        if not good.all():
            at = np.unravel_index(np.argmax(np.where(good, 0, off / np.maximum(allow[:live], 1e-30))), off.shape)
            raise AssertionError(f"{(~good).sum()} of {good.size} off; worst at {at}: {ours[at]} for "
                                 f"{want[:live][at]}, allowed {allow[:live][at]}")
        return ours


LENGTHS = [
    # past, new
    ([0], [1]), ([0], [2]), ([1], [1]), ([14], [1]), ([15], [1]), ([16], [1]), ([31], [1]), ([62], [1]), ([63], [1]),
    ([64], [1]), ([127], [2]), ([300], [1]), ([2000], [1]),
    ([0, 500, 33], [1, 1, 1]), ([3, 0, 700, 129, 64], [5, 5, 2, 1, 4]),
    ([0], [16]), ([0], [17]), ([0], [63]), ([0], [64]), ([0], [65]), ([0], [130]), ([200], [33]), ([77], [100]),
    ([10, 900, 0, 45, 3], [40, 1, 70, 3, 0]),
]


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,d", [(32, 8, 64), (8, 4, 128)])
@pytest.mark.parametrize("past,new", LENGTHS, ids=str)
def test_attention_lengths(lcr, gpu, variant, heads, kv, d, past, new):
    Case(variant, past, new, heads=heads, kv=kv, d=d, seed=sum(past) + 3 * sum(new), tail=3).check(lcr)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("heads,kv,d", [
    (1, 1, 64), (2, 2, 64), (6, 3, 64), (12, 4, 64), (5, 1, 64), (16, 2, 64), (16, 1, 64), (40, 1, 64), (64, 8, 64),
    (4, 4, 128), (14, 2, 128), (33, 1, 128), (7, 7, 128),
    (4, 2, 32), (4, 2, 80), (2, 1, 96), (3, 3, 256), (2, 2, 1), (4, 1, 200),
])
def test_attention_head_layouts(lcr, gpu, workspace, heads, kv, d):
    Case("bf16", [70, 0, 9, 400], [1, 20, 3, 2], heads=heads, kv=kv, d=d, seed=heads + d).check(lcr, workspace=workspace)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("changed", [
    dict(page=1), dict(page=2), dict(page=3), dict(page=4), dict(page=5), dict(page=8), dict(page=12), dict(page=24),
    dict(page=32), dict(page=64), dict(page=100), dict(page=128), dict(page=1000), dict(page=4096),
    dict(extra_stride=8), dict(extra_stride=1), dict(extra_stride=64), dict(shift=1), dict(shift=4), dict(shift=8),
    dict(page_pad=40), dict(head_pad=16), dict(head_pad=3), dict(page_pad=1),
], ids=str)
def test_attention_layouts(lcr, gpu, d, changed):
    Case("bf16", [70, 0, 333, 9], [2, 20, 1, 90], heads=8, kv=2, d=d, seed=d, **changed).check(lcr)


@pytest.mark.parametrize("variant,d", [("bf16", 64), ("fp16", 64), ("bf16", 128)])
def test_attention_over_long_caches(lcr, gpu, variant, d):
    """Few rows over many positions: split over the device."""
    Case(variant, [9001], [1], heads=8, kv=2, d=d, seed=3).check(lcr)
    Case(variant, [4097, 20, 6000], [3, 1, 9], heads=8, kv=2, d=d, seed=4).check(lcr)
    Case(variant, [3000, 0], [70, 40], heads=4, kv=1, d=d, seed=5).check(lcr)


def test_attention_many_sequences(lcr, gpu):
    r = rng(21)
    Case("bf16", r.integers(0, 90, 300), r.integers(0, 3, 300), heads=4, kv=2, seed=6, tail=9).check(lcr)
    Case("bf16", r.integers(0, 9, 4096), np.ones(4096, int), heads=1, kv=1, seed=7).check(lcr)


@pytest.mark.parametrize("d", [64, 128, 40])
def test_attention_large_scores(lcr, gpu, d):
    """Scores in the hundreds, rising and falling along the keys."""
    for sign in (1.0, -1.0):
        c = Case("bf16", [500], [3], heads=4, kv=1, d=d, seed=8, q_scale=4.0)
        ramp = sign * np.linspace(0, 6, 503)
        for position in range(503):
            at = c.position_index(0, 0, position)
            c.keys[at:at + d] = elems(to_f32(c.keys[at:at + d]) * np.float32(abs(ramp[position])))
        c.check(lcr)


@pytest.mark.parametrize("d", [64, 128, 72])
def test_attention_rows_that_see_nothing(lcr, gpu, d):
    """More rows than positions: the rows before position 0 are zeros."""
    c = Case("bf16", [20, 5, 0], [3, 4, 2], heads=4, kv=2, d=d, seed=9)
    c.lengths = np.array([23, 2, 0], np.int32)
    ours = c.check(lcr)
    assert (ours[3:5] == 0).all() and (ours[5] != 0).any() and (ours[7:9] == 0).all()
    c.lengths = np.array([-3, -2 ** 31, 1], np.int32)
    ours = c.check(lcr)
    assert (ours[:8] == 0).all() and (ours[8] != 0).any()


@pytest.mark.parametrize("d", [64, 128, 72])
def test_attention_lengths_past_the_table(lcr, gpu, d):
    """Positions that the table has no pages for do not exist."""
    c = Case("bf16", [30, 60], [2, 30], heads=4, kv=2, d=d, seed=10)
    c.lengths = np.array([32, 2 ** 31 - 1], np.int32)
    c.check(lcr)
    c.lengths = np.array([200, 100], np.int32)
    c.tables = np.maximum(c.tables, 0)
    c.check(lcr)


@pytest.mark.parametrize("d", [64, 128, 72])
def test_attention_max_new(lcr, gpu, d):
    """Rows past max_new come out as zeros; a larger max_new changes nothing."""
    c = Case("bf16", [30, 10], [50, 3], heads=4, kv=2, d=d, seed=11)
    full = c.check(lcr)
    for most in (2, 7, 33, 49):
        ours = to_f32(c.run(lcr, max_new=most))
        want, allow = c.want()
        cut = np.concatenate([np.arange(50) < most, np.arange(3) < most])
        assert (ours[~cut] == 0).all()
        assert (np.abs(ours[cut] - want[cut]) <= allow[cut]).all()
    assert (np.abs(to_f32(c.run(lcr, max_new=5000)) - full) <= 2 * c.want()[1]).all()
    assert (to_f32(c.run(lcr, max_new=0)) == 0).all()


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 72])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_attention_masked_places_hold_anything(lcr, gpu, variant, d, value):
    """Infinities and NaN in keys and values that a row does not see leave it as
    it is, in its own chunk's later tokens, in unwritten slots and other pages."""
    for past, new in (([70], [1]), ([37], [5]), ([0], [40]), ([100], [90])):
        c = Case(variant, past, new, heads=4, kv=1, d=d, seed=12)
        clean = c.run(lcr)
        used = np.zeros(c.keys.size, bool)
        for position in range(int(c.lengths[0])):
            at = c.position_index(0, 0, position)
            used[at:at + d] = True
        bits = elems(np.array([value], np.float32), c.kind)[0]
        c.keys[~used], c.values[~used] = bits, bits
        expect_bits_equal(c.run(lcr), clean, "unused slots")
        if new[0] == 1:
            continue
        # a later token of the chunk itself
        late = past[0] + new[0] - 2
        at = c.position_index(0, 0, late)
        keep = c.keys[at:at + d].copy(), c.values[at:at + d].copy()
        c.values[at + 3] = bits
        got = c.run(lcr)
        expect_bits_equal(got[: new[0] - 2], clean[: new[0] - 2], "rows before the value")
        seen = to_f32(got[new[0] - 2:], c.kind)
        # what the definition gives: the value itself, or NaN
        assert (np.isnan(seen[..., 3]) if np.isnan(value) else (seen[..., 3] == value)).all()
        others = np.delete(seen, 3, -1) == np.delete(to_f32(clean[new[0] - 2:], c.kind), 3, -1)
        assert others.all()
        c.values[at:at + d] = keep[1]
        c.keys[at:at + d] = elems(np.full(d, np.nan, np.float32), c.kind)
        got = c.run(lcr)
        expect_bits_equal(got[: new[0] - 2], clean[: new[0] - 2], "rows before the key")
        assert np.isnan(to_f32(got[new[0] - 2:], c.kind)).all()


@pytest.mark.parametrize("d", [64, 128, 72])
def test_attention_pages_outside_the_pool(lcr, gpu, d):
    """Other sequences keep their bits; the one that reads such a page is NaN or
    untouched by it, row by row, and nothing faults."""
    c = Case("bf16", [70, 70, 300], [2, 1, 40], heads=4, kv=2, d=d, seed=13)
    clean = c.run(lcr)
    for bad in (-1, c.pool, 2 ** 31 - 1, -2 ** 31):
        c.tables[1, 2] = bad
        got = c.run(lcr)
        expect_bits_equal(got[:2], clean[:2], "the sequence before")
        expect_bits_equal(got[3:], clean[3:], "the sequence behind")
        assert np.isnan(to_f32(got[2])).all()


def test_attention_past_32_bits(lcr, gpu):
    """Pages that lie more than 2^31 elements into the pools."""
    page, kv, d = 4096, 8, 64
    page_stride = kv * page * d            # 2^21 elements
    pool = 1100                            # 4.6 GB a pool
    far = [1090, 1027, 3]                  # the first two past 2^31 elements
    c = Case("bf16", [5000, 30], [2, 1], heads=8, kv=kv, d=d, page=page, seed=14, spare=0)
    keys, values = (lcr.DeviceBuffer(2 * pool * page_stride, zero=False) for _ in range(2))
    lib = lcr.load_library("bf16")
    for old, new in enumerate(far):
        for small, big in ((c.keys, keys), (c.values, values)):
            part = np.ascontiguousarray(small[old * page_stride:(old + 1) * page_stride])
            lcr.check(lib, lib.lcr_memcpy_htod(big.ptr + 2 * new * page_stride, part.ctypes.data, part.nbytes))
    table = np.where(c.tables >= 0, np.array(far)[np.maximum(c.tables, 0)], -1).astype(np.int32)
    out = dev(np.zeros(3 * 8 * d, np.uint16))
    view = lcr.KvView(keys.ptr, values.ptr, p(dev(table)), page, page_stride, page * d, kv, d)
    size = lib.lcr_batch_attention_workspace_bytes(2, 3, 2, 8, 1, d)
    status = lib.lcr_batch_attention(p(out), p(dev(c.q)), ctypes.byref(view), p(dev(c.starts)), p(dev(c.lengths)), 2, 3,
                                     2, 8, 1, table.shape[1], pool, c.q_stride, c.scale,
                                     p(dev(np.zeros(size + 16, np.uint8))), size, None)
    assert status == 0
    got = to_f32(host(out)).reshape(3, 8, d)
    want, allow = c.want()
    assert (np.abs(got - want) <= allow).all()
    keys.free()
    values.free()


def test_attention_twice_gives_the_same_bits(lcr, gpu):
    c = Case("bf16", [5000, 10, 700], [1, 40, 5], heads=8, kv=2, seed=15)
    first = c.run(lcr)
    expect_bits_equal(c.run(lcr, repeat=3), first, "another call")
