"""lcr_batch_attention_kv8 against its definition in 64 bits: attention of the values
that the cache stands for (tests/kv8_reference.py), which are values of the element
type, so that what the rounding of weights, sums and outputs may come to is what
tests/batch_reference.py derives for the 16-bit cache."""

import ctypes

import numpy as np
import pytest

import batch_reference
import kv8_reference as ref
from helpers import BF16, FP16, dev, elems, expect_bits_equal, host, p, random_elems, rng, to_f32

pytestmark = pytest.mark.gpu

KINDS = {"bf16": BF16, "fp16": FP16}


class Case:
    """Random rows and caches of a batch: `past` cached positions and `new` rows
    each, pages in random order, every unused table entry a page of no use (-1)."""

    def __init__(self, variant, past, new, *, heads=32, kv=8, d=64, page=16, seed=1, q_scale=1.0, tail=0,
                 extra_stride=0, shift=0, spare=3, **pads):
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
        self.q = random_elems(r, self.tokens * self.q_stride + shift, q_scale, self.kind)
        self.cache = ref.Cache8(self.pool, kv, page, d, seed=seed, **pads)
        self.cache.fill(r, variant)
        # blocks whose values are small or large: scales of many sizes
        for scales in (self.cache.key_scales, self.cache.value_scales):
            scales *= (2.0 ** r.integers(-2, 2, scales.size)).astype(np.float32)
        self.scale = d ** -0.5

    def place(self, b, position):
        return int(self.tables[b, position // self.page]), position % self.page

    def run(self, lcr, workspace=True, max_new=None, stream=None, repeat=1):
        lib = lcr.load_library(self.variant)
        max_new = int(self.new.max(initial=0)) if max_new is None else max_new
        self.before = random_elems(rng(99), self.tokens * self.heads * self.d + 16 + self.shift, 1.0, self.kind)
        out, q = dev(self.before), dev(self.q)
        self.cache.upload(dev)
        view = self.cache.view(lcr, p, p(dev(self.tables)))
        group = self.heads // self.kv
        size = lib.lcr_batch_attention_kv8_workspace_bytes(len(self.past), self.tokens, max_new, self.heads, group,
                                                           self.d) if workspace else 0
        # a workspace may hold anything before a call
        ws = dev(np.full(size // 4 + 4, np.nan, np.float32)) if size else None
        starts, lengths = dev(self.starts), dev(self.lengths)
        for _ in range(repeat):
            status = lib.lcr_batch_attention_kv8(
                p(out) + 2 * self.shift, p(q) + 2 * self.shift, ctypes.byref(view), p(starts), p(lengths),
                len(self.past), self.tokens, max_new, self.heads, group, self.tables.shape[1], self.pool,
                self.q_stride, self.scale, p(ws) if ws else None, size, stream)
            assert status == 0, lib.lcr_last_error_message()
        got = host(out)
        expect_bits_equal(got[: self.shift], self.before[: self.shift], "ahead of the output")
        got = got[self.shift:]
        end = self.tokens * self.heads * self.d
        expect_bits_equal(got[end:], self.before[self.shift + end:], "behind the output")
        return got[:end].reshape(self.tokens, self.heads, self.d)

    def want(self):
        wide = lambda a: to_f32(a, self.kind).astype(np.float64)  # noqa: E731
        q = wide(self.q[self.shift:]).reshape(self.tokens, self.q_stride)[:, : self.heads * self.d]
        keys, values = self.cache.wide()
        # entries of no use are never read
        with np.errstate(invalid="ignore"):
            return batch_reference.attention(q.reshape(self.tokens, self.heads, self.d), keys, values,
                                             np.maximum(self.tables, 0), self.starts, self.lengths, self.page,
                                             self.scale, self.variant)

    def check(self, lcr, **more):
        got = self.run(lcr, **more)
        want, allow = self.want()
        live = int(self.starts[-1])
        end = self.tokens * self.heads * self.d
        expect_bits_equal(got[live:], self.before[self.shift : self.shift + end].reshape(got.shape)[live:],
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
def test_lengths(lcr, gpu, variant, heads, kv, d, past, new):
    Case(variant, past, new, heads=heads, kv=kv, d=d, seed=sum(past) + 3 * sum(new), tail=3).check(lcr)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("heads,kv,d", [
    (1, 1, 64), (2, 2, 64), (6, 3, 64), (12, 4, 64), (5, 1, 64), (16, 2, 64), (16, 1, 64), (40, 1, 64), (64, 8, 64),
    (160, 1, 64), (4, 4, 128), (14, 2, 128), (33, 1, 128), (7, 7, 128), (300, 1, 128),
    (4, 2, 32), (4, 2, 80), (2, 1, 96), (3, 3, 256), (2, 2, 16), (4, 1, 208),
])
def test_head_layouts(lcr, gpu, workspace, heads, kv, d):
    Case("bf16", [70, 0, 9, 400], [1, 20, 3, 2], heads=heads, kv=kv, d=d, seed=heads + d).check(lcr, workspace=workspace)


@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("changed", [
    dict(page=32), dict(page=48), dict(page=64), dict(page=112), dict(page=128), dict(page=1008), dict(page=4096),
    dict(extra_stride=8), dict(extra_stride=1), dict(extra_stride=64), dict(shift=1), dict(shift=4), dict(shift=8),
    dict(page_pad=48), dict(head_pad=16), dict(scale_head_pad=1), dict(scale_page_pad=7),
], ids=str)
def test_layouts(lcr, gpu, d, changed):
    Case("bf16", [70, 0, 333, 9], [2, 20, 1, 90], heads=8, kv=2, d=d, seed=d, **changed).check(lcr)


@pytest.mark.parametrize("variant,d", [("bf16", 64), ("fp16", 64), ("bf16", 128), ("fp16", 128)])
def test_long_caches(lcr, gpu, variant, d):
    """Few rows over many positions: split over the device."""
    Case(variant, [9001], [1], heads=8, kv=2, d=d, seed=3).check(lcr)
    Case(variant, [4097, 20, 6000], [3, 1, 9], heads=8, kv=2, d=d, page=32, seed=4).check(lcr)
    Case(variant, [3000, 0], [70, 40], heads=4, kv=1, d=d, seed=5).check(lcr)
    Case(variant, [2500, 1500, 40], [3, 50, 1], heads=8, kv=4, d=d, seed=16, tail=5).check(lcr)


def test_many_sequences(lcr, gpu):
    r = rng(21)
    Case("bf16", r.integers(0, 90, 300), r.integers(0, 3, 300), heads=4, kv=2, seed=6, tail=9).check(lcr)
    Case("bf16", r.integers(0, 9, 4096), np.ones(4096, int), heads=1, kv=1, seed=7).check(lcr)


@pytest.mark.parametrize("d", [64, 128, 48])
def test_large_scores(lcr, gpu, d):
    """Scores in the hundreds, rising and falling along the keys: scales of keys that
    differ by 2^12."""
    for sign in (1, -1):
        c = Case("bf16", [500], [3], heads=4, kv=1, d=d, seed=8, q_scale=4.0)
        for position in range(0, 503, 16):
            page, slot = c.place(0, position)
            c.cache.key_scales[c.cache.scales_at[page, 0, slot // 16]] *= 2.0 ** (sign * (position // 128 - 2))
        c.check(lcr)


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 32])
def test_scales_of_every_size(lcr, gpu, variant, d):
    """The least and the largest scales that the element type has use for."""
    span = (-117, 100) if variant == "bf16" else (-15, 6)
    c = Case(variant, [200, 30], [1, 20], heads=4, kv=1, d=d, seed=18)
    c.cache.value_scales[:] = 2.0 ** rng(1).integers(*span, c.cache.value_scales.size)
    c.cache.key_scales[:] = 2.0 ** rng(2).integers(span[0], -6, c.cache.key_scales.size)
    c.check(lcr)


@pytest.mark.parametrize("d", [64, 128, 80])
def test_rows_that_see_nothing(lcr, gpu, d):
    """More rows than positions: the rows before position 0 are zeros."""
    c = Case("bf16", [20, 5, 0], [3, 4, 2], heads=4, kv=2, d=d, seed=9)
    c.lengths = np.array([23, 2, 0], np.int32)
    ours = c.check(lcr)
    assert (ours[3:5] == 0).all() and (ours[5] != 0).any() and (ours[7:9] == 0).all()
    c.lengths = np.array([-3, -2 ** 31, 1], np.int32)
    ours = c.check(lcr)
    assert (ours[:8] == 0).all() and (ours[8] != 0).any()
    c = Case("bf16", [20, 5, 0], [33, 64, 80], heads=4, kv=2, d=d, seed=9)
    c.lengths = np.array([40, -5, 3], np.int32)
    ours = c.check(lcr)
    assert (ours[33:97 + 77] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 80])
def test_lengths_past_the_table(lcr, gpu, d):
    """Positions that the table has no pages for do not exist."""
    c = Case("bf16", [30, 60], [2, 30], heads=4, kv=2, d=d, seed=10)
    c.lengths = np.array([32, 2 ** 31 - 1], np.int32)
    c.check(lcr)
    c.lengths = np.array([200, 100], np.int32)
    c.tables = np.maximum(c.tables, 0)
    c.check(lcr)


@pytest.mark.parametrize("d", [64, 128, 80])
def test_max_new(lcr, gpu, d):
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
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("scale", [np.nan, np.inf, 0.0, 2.0 ** 127])
def test_unseen_places_hold_anything(lcr, gpu, variant, d, scale):
    """NaN numbers and any scales in places that no row sees leave them as they are;
    NaN in a chunk's own later tokens leaves the tokens before them."""
    for past, new in (([70], [1]), ([37], [5]), ([0], [40]), ([100], [90]), ([1500], [2]), ([1300, 40], [60, 1])):
        c = Case(variant, past, new, heads=4, kv=1, d=d, seed=12)
        clean = c.run(lcr)
        used, used_scales = np.zeros(c.cache.keys.size, bool), np.zeros(c.cache.key_scales.size, bool)
        used_values = used.copy()
        dims = np.arange(d)
        for b in range(len(past)):
            for position in range(int(c.lengths[b])):
                page, slot = c.place(b, position)
                base, t = c.cache.at[page, 0, slot // 16, 0], slot % 16
                used[base + t * d + dims] = True
                used_values[base + t // 4 * 4 * d + 4 * dims + t % 4] = True
                used_scales[c.cache.scales_at[page, 0, slot // 16]] = True
        c.cache.keys[~used] = c.cache.values[~used_values] = ref.NAN
        c.cache.key_scales[~used_scales] = c.cache.value_scales[~used_scales] = scale
        expect_bits_equal(c.run(lcr), clean, "unused slots")
        if new[0] == 1:
            continue
        # a later token of the first sequence's chunk
        rows = new[0]
        page, slot = c.place(0, past[0] + rows - 2)
        keep = c.cache.keys.copy(), c.cache.values.copy()
        c.cache.set_position("values", page, 0, slot, slice(3, 4), 0xFF)
        got = c.run(lcr)
        same = np.ones(c.tokens, bool)
        same[rows - 2 : rows] = False
        expect_bits_equal(got[same], clean[same], "rows that do not see the value")
        seen = to_f32(got[~same], c.kind)
        assert np.isnan(seen[..., 3]).all()
        assert (np.delete(seen, 3, -1) == np.delete(to_f32(clean[~same], c.kind), 3, -1)).all()
        c.cache.values = keep[1]
        c.cache.set_position("keys", page, 0, slot, slice(0, 1), ref.NAN)
        got = c.run(lcr)
        expect_bits_equal(got[same], clean[same], "rows that do not see the key")
        assert np.isnan(to_f32(got[~same], c.kind)).all()


@pytest.mark.parametrize("variant,gap", [("fp16", 30.0), ("bf16", 200.0)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 60])
def test_nan_of_no_weight(lcr, gpu, variant, gap, d, rows):
    """A NaN that a row sees makes its element NaN, also where its weight rounds to 0."""
    c = Case(variant, [400], [rows], heads=4, kv=2, d=d, seed=22)
    c.q[:] = elems(np.ones(1, np.float32), c.kind)[0]
    c.cache.keys[c.cache.at] = ref.encode(np.array(0.0))
    page, slot = c.place(0, 390)
    c.cache.set_position("keys", page, 0, slot, slice(None), ref.encode(np.array(8.0)))
    c.cache.set_position("keys", page, 1, slot, slice(None), ref.encode(np.array(8.0)))
    for head in (0, 1):
        c.cache.key_scales[c.cache.scales_at[page, head, slot // 16]] = 2.0 ** np.ceil(np.log2(gap / (8 * d ** 0.5)))
    page, slot = c.place(0, 17)
    c.cache.set_position("values", page, 0, slot, slice(5, 6), ref.NAN)
    seen = to_f32(c.run(lcr), c.kind)
    spoilt = np.isnan(seen)
    assert spoilt[:, :2, 5].all()
    spoilt[:, :2, 5] = False
    assert not spoilt.any()


@pytest.mark.parametrize("d", [64, 128, 80])
def test_pages_outside_the_pool(lcr, gpu, d):
    """Other sequences keep their bits; the one that reads such a page is NaN, and
    nothing faults."""
    c = Case("bf16", [70, 70, 300], [2, 1, 40], heads=4, kv=2, d=d, seed=13)
    clean = c.run(lcr)
    for bad in (-1, c.pool, 2 ** 31 - 1, -2 ** 31):
        c.tables[1, 2] = bad
        got = c.run(lcr)
        expect_bits_equal(got[:2], clean[:2], "the sequence before")
        expect_bits_equal(got[3:], clean[3:], "the sequence behind")
        assert np.isnan(to_f32(got[2])).all()


@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (4, 2, 128), (2, 1, 48)])
@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_32_bits(lcr, gpu, heads, kv, d, new):
    """Pages that lie 2^28 bytes apart, the last of them past 2^32."""
    stride, pool = 1 << 28, 18
    c = Case("bf16", [50], [new], heads=heads, kv=kv, d=d, page=64, seed=14, spare=0)
    far = np.array([17, 9])
    keys, values = (lcr.DeviceBuffer(pool * stride, zero=False) for _ in range(2))
    lib = lcr.load_library("bf16")
    for old in range(c.pool):
        for small, big in ((c.cache.keys, keys), (c.cache.values, values)):
            part = np.ascontiguousarray(small[old * c.cache.page_stride:(old + 1) * c.cache.page_stride])
            lcr.check(lib, lib.lcr_memcpy_htod(big.ptr + int(far[old]) * stride, part.ctypes.data, part.nbytes))
    scales = []
    for small in (c.cache.key_scales, c.cache.value_scales):
        big = np.ones(pool * c.cache.scale_page_stride, np.float32)
        for old in range(c.pool):
            n = c.cache.scale_page_stride
            big[far[old] * n : (far[old] + 1) * n] = small[old * n : (old + 1) * n]
        scales.append(dev(big))
    c.cache.on_device = [keys, values, *scales]
    table = np.where(c.tables >= 0, far[np.maximum(c.tables, 0)], -1).astype(np.int32)
    view = c.cache.view(lcr, p, p(dev(table)))
    view.page_stride = stride
    out = dev(np.zeros(new * heads * d, np.uint16))
    status = lib.lcr_batch_attention_kv8(
        p(out), p(dev(c.q)), ctypes.byref(view), p(dev(c.starts)), p(dev(c.lengths)), 1, new, new, heads, heads // kv,
        table.shape[1], pool, c.q_stride, c.scale, None, 0, None)
    assert status == 0, lib.lcr_last_error_message()
    got = to_f32(host(out)).reshape(new, heads, d)
    want, allow = c.want()
    assert (np.abs(got - want) <= allow).all()
    keys.free()
    values.free()


def test_twice_gives_the_same_bits(lcr, gpu):
    c = Case("bf16", [5000, 10, 700], [1, 40, 5], heads=8, kv=2, seed=15)
    first = c.run(lcr)
    expect_bits_equal(c.run(lcr, repeat=3), first, "another call")


def test_a_part_of_a_step(lcr, gpu):
    """Row starts from the third sequence on: the rows before stay as they were."""
    for d, heads, past, new in ((64, 8, [30, 1200, 40, 77], [2, 40, 1, 9]), (128, 4, [3, 50, 20, 60], [1, 2, 3, 1])):
        c = Case("bf16", past, new, heads=heads, kv=2, d=d, seed=23)
        whole = c.run(lcr)
        first = int(c.starts[2])
        c.starts, c.lengths, c.tables = c.starts[2:], c.lengths[2:], c.tables[2:].copy()
        c.past, c.new = c.past[2:], c.new[2:]
        got = c.run(lcr)
        expect_bits_equal(got[:first], c.before[: c.tokens * heads * d].reshape(got.shape)[:first], "rows before")
        want, allow = c.want()
        off = np.abs(to_f32(got[first:]).astype(np.float64) - want[first:])
        assert (off <= allow[first:]).all()
        assert (np.abs(to_f32(got[first:]) - to_f32(whole[first:])) <= 2 * allow[first:]).all()


def test_row_starts_that_do_not_ascend(lcr, gpu):
    """Nothing is said of the outputs but that nothing out of bounds is touched."""
    for starts in ([0, 9, 4, 12], [0, 2 ** 31 - 1, 5, 12], [-5, 3, 6, 12], [0, 12, 0, 12]):
        for d in (64, 128, 48):
            c = Case("bf16", [40, 90, 20], [4, 4, 4], heads=4, kv=2, d=d, seed=24)
            c.starts = np.array(starts, np.int32)
            c.run(lcr, max_new=12)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
def test_scales(lcr, gpu, scale):
    for d in (64, 128, 80):
        c = Case("bf16", [1300, 5], [2, 7], heads=4, kv=2, d=d, seed=38)
        c.scale = scale
        c.check(lcr)


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("columns", [1, 90])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_in_many_tiles_of_a_unit(lcr, gpu, variant, columns, d):
    """Values that only a unit's later rows see, in neighbouring tiles and in every
    second one, in one launch and (wide tables) cut: each reaches its element of the
    rows from its position on, and nothing else changes."""
    for past, new in (([0], [600]), ([330, 0], [290, 410])):
        c = Case(variant, past, new, heads=1, kv=1, d=d, seed=39)
        wide = np.full((len(past), max(columns, c.tables.shape[1])), -1, np.int32)
        wide[:, : c.tables.shape[1]] = c.tables
        c.tables = wide
        clean = c.run(lcr)
        expected = to_f32(clean, c.kind).copy()
        r = rng(40)
        for b, (first, n) in enumerate(zip(c.starts, new)):
            at = sorted(r.choice(n - 2, 9, replace=False).tolist()) + [n - 2]
            for dim, i in enumerate(at):
                page, slot = c.place(b, past[b] + i)
                c.cache.set_position("values", page, 0, slot, slice(dim, dim + 1), (ref.NAN, 0xFF)[dim % 2])
                expected[first + i:first + n, 0, dim] = np.nan
        got = to_f32(c.run(lcr), c.kind)
        assert (np.isnan(got) == np.isnan(expected)).all()
        assert ((got == expected) | np.isnan(expected)).all()


@pytest.mark.parametrize("d", [64, 128])
def test_a_workspace_keeps_what_lies_behind_it(lcr, gpu, d):
    lib = lcr.load_library("bf16")
    for past, new in (([2500, 40], [1, 1]), ([1800, 1100], [8, 3]), ([1500, 20], [60, 3])):
        c = Case("bf16", past, new, heads=4, kv=2, d=d, seed=52)
        size = lib.lcr_batch_attention_kv8_workspace_bytes(2, c.tokens, max(new), 4, 2, d)
        guard = np.full(size + 4096, 0x5A, np.uint8)
        ws, out = dev(guard), dev(np.zeros(c.tokens * 4 * d, np.uint16))
        c.cache.upload(dev)
        view = c.cache.view(lcr, p, p(dev(c.tables)))
        status = lib.lcr_batch_attention_kv8(
            p(out), p(dev(c.q)), ctypes.byref(view), p(dev(c.starts)), p(dev(c.lengths)), 2, c.tokens, max(new), 4, 2,
            c.tables.shape[1], c.pool, c.q_stride, c.scale, p(ws), size, None)
        assert status == 0, lib.lcr_last_error_message()
        expect_bits_equal(host(ws, np.uint8)[size:], guard[size:], "behind the workspace")
