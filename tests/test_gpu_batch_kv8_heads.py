"""lcr_batch_norm_rope_write_kv8 against its definition in 64 bits
(tests/kv8_reference.py), call after call on one cache.

Scales are equal: they are powers of two, decided by fp32 values that the kernel
computes in fp64, which tests/kv8_reference.py does too; the two can only differ
where a block's largest value is within fp64's error of such a power, and then the
test says so. A number written is the nearest to the value, which is off by its
rounding to fp32, 2^-24 of its size, on either side: no further from it than the
nearest is, and 2^-22 of its size. Numbers held that are rounded to a larger
scale are equal, as the product with a power of two is exact. Queries: half a step
of the output's rounding and fp32's own, at most (d + 12) 2^-24 of the two products
whose difference an element is."""

import ctypes

import numpy as np
import pytest

import batch_reference
import kv8_reference as ref
from helpers import BF16, FP16, dev, elems, expect_bits_equal, host, p, random_elems, rng, to_f32

pytestmark = pytest.mark.gpu

KINDS = {"bf16": BF16, "fp16": FP16}


class Writer:
    """A cache that calls append to, each checked against what the one before left."""

    def __init__(self, lcr, variant, *, heads=4, kv=2, d=64, page=16, pool=5, norm=True, extra_stride=0, shift=0,
                 table_positions=64, seed=1, eps=1e-5, **pads):
        self.lcr, self.variant, self.kind = lcr, variant, KINDS[variant]
        self.lib = lcr.load_library(variant)
        self.heads, self.shift, self.eps = heads, shift, eps
        self.cache = ref.Cache8(pool, kv, page, d, seed=seed, **pads)
        self.r = rng(seed)
        self.stride = (heads + 2 * kv) * d + extra_stride
        angle = np.arange(table_positions)[:, None] * 10000.0 ** (-np.arange(d // 2) / (d // 2))
        self.table = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
        self.norms = ((random_elems(self.r, d, 0.3, self.kind), random_elems(self.r, d, 0.3, self.kind))
                      if norm else (None, None))

    def rows(self, count, scale=1.0):
        return random_elems(self.r, (count, self.stride), scale, self.kind)

    def launch(self, qkv, positions, slots, q_out, stream=None):
        c, d = self.cache, self.cache.d
        src = dev(np.concatenate([np.zeros(self.shift, np.uint16), qkv.ravel()]))
        base = p(src) + 2 * self.shift
        w = [p(dev(x)) if x is not None else None for x in self.norms]
        status = self.lib.lcr_batch_norm_rope_write_kv8(
            p(q_out) + 2 * self.shift, ctypes.byref(c.view(self.lcr, p)), base, base + 2 * self.heads * d,
            base + 2 * (self.heads + c.kv) * d, *w, self.eps, p(dev(self.table)), len(self.table), p(dev(positions)),
            p(dev(slots)), len(slots), self.heads, c.pool, self.stride, stream)
        assert status == 0, self.lib.lcr_last_error_message()

    def call(self, qkv, slots, positions=None, check=True):
        c, d, heads, kv = self.cache, self.cache.d, self.heads, self.cache.kv
        slots = np.asarray(slots, np.int32)
        tokens = len(slots)
        if positions is None:
            positions = self.r.integers(0, len(self.table), tokens)
        positions = np.asarray(positions, np.int32)
        live = (slots >= 0) & (slots < c.pool * c.page) & (positions >= 0) & (positions < len(self.table))
        before_q = random_elems(self.r, tokens * heads * d + 8 + self.shift, 1.0, self.kind)
        q_out = dev(before_q)
        c.upload(dev)
        was = [x.copy() for x in (c.keys, c.values, c.key_scales, c.value_scales)]
        self.launch(qkv, positions, slots, q_out)
        c.keys, c.values = (host(b, np.uint8)[: w.size] for b, w in zip(c.on_device[:2], was[:2]))
        c.key_scales, c.value_scales = (host(b, np.float32)[: w.size] for b, w in zip(c.on_device[2:], was[2:]))
        if not check:
            return
        x = to_f32(qkv, self.kind).astype(np.float64)
        angles = self.table.astype(np.float64)[np.where(live, positions, 0)]
        wide = lambda a: None if a is None else to_f32(a, self.kind).astype(np.float64)  # noqa: E731
        self.check_queries(host(q_out), before_q, x, live, angles, wide(self.norms[0]))
        if kv == 0:
            return
        with np.errstate(invalid="ignore", over="ignore"):
            keys, _ = batch_reference.rotate_heads(x[:, heads * d : (heads + kv) * d].reshape(tokens, kv, d),
                                                   wide(self.norms[1]), self.eps, angles)
        values = x[:, (heads + kv) * d : (heads + 2 * kv) * d].reshape(tokens, kv, d)
        self.check_numbers("keys", keys, slots, live, was[0], was[2])
        self.check_numbers("values", values, slots, live, was[1], was[3])

    def check_queries(self, got, before, x, live, angles, norm):
        d, heads, tokens = self.cache.d, self.heads, len(live)
        expect_bits_equal(got[: self.shift], before[: self.shift], "ahead of the queries")
        got, before = got[self.shift:], before[self.shift:]
        expect_bits_equal(got[tokens * heads * d:], before[tokens * heads * d:], "behind the queries")
        got, before = (a[: tokens * heads * d].reshape(tokens, heads, d) for a in (got, before))
        expect_bits_equal(got[~live], before[~live], "a skipped row's queries")
        with np.errstate(invalid="ignore", over="ignore"):
            want, size = batch_reference.rotate_heads(x[:, : heads * d].reshape(tokens, heads, d), norm, self.eps, angles)
        half = batch_reference.HALF_STEP[self.variant]
        allow = half * np.abs(want) * (1 + half) + (d + 12) * 2.0 ** -24 * size
        allow += 2.0 ** -25 if self.variant == "fp16" else 1e-38
        finite = live[:, None, None] & np.isfinite(want) & (np.abs(want) < 60000)
        off = np.abs(to_f32(got, self.kind).astype(np.float64) - want)
        assert (off[finite] <= allow[finite]).all()

    def check_numbers(self, which, rows, slots, live, was, was_scales):
        c = self.cache
        blocks_of = ref.to_blocks if which == "keys" else ref.values_to_blocks
        got, got_scales = getattr(c, which), getattr(c, which[:-1] + "_scales")
        touched, touched_scales = np.zeros(was.size, bool), np.zeros(was_scales.size, bool)
        new = {}
        for row in np.nonzero(live)[0]:
            page, slot = divmod(int(slots[row]), c.page)
            new.setdefault((page, slot // ref.BLOCK), {})[slot % ref.BLOCK] = rows[row]
        for (page, n), at_rows in new.items():
            for h in range(c.kv):
                at, scale_at = c.at[page, h, n], c.scales_at[page, h, n]
                touched[at] = touched_scales[scale_at] = True
                scale, kept, fresh = ref.append(blocks_of(was[at]), was_scales[scale_at],
                                                {t: y[h] for t, y in at_rows.items()}, self.variant)
                where = (which, page, h, n)
                assert got_scales[scale_at] == np.float32(scale), (where, got_scales[scale_at], scale)
                block = blocks_of(got[at])
                for t in range(ref.BLOCK):
                    if t not in fresh:
                        assert (block[t] == kept[t]).all(), (where, t)
                        continue
                    y, have = fresh[t], ref.NUMBERS[block[t]]
                    spoilt = np.isnan(y)
                    assert (np.isnan(have) == spoilt).all(), (where, t)
                    nearest = ref.NUMBERS[ref.encode(np.where(spoilt, 0, y))]
                    allow = np.abs(nearest - y) + 2.0 ** -22 * np.abs(y)
                    off = np.abs(have - y)
                    assert (off[~spoilt] <= allow[~spoilt]).all(), (where, t, y, have)
        expect_bits_equal(got[~touched], was[~touched], "the rest of the " + which)
        expect_bits_equal(got_scales[~touched_scales].view(np.uint32), was_scales[~touched_scales].view(np.uint32),
                          "the rest of the scales of " + which)


SHAPES = [(4, 2, 64), (32, 8, 64), (1, 1, 64), (16, 8, 128), (3, 1, 128), (4, 4, 256), (4, 2, 16), (6, 3, 48), (2, 2, 80),
          (5, 5, 112), (2, 1, 240)]


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("heads,kv,d", SHAPES)
def test_appends(lcr, gpu, variant, norm, heads, kv, d):
    """Token by token, in twos and threes, a chunk over several blocks, several
    sequences in one call, growing and shrinking values."""
    w = Writer(lcr, variant, heads=heads, kv=kv, d=d, norm=norm, pool=12, seed=heads + d)
    for t in range(5):
        w.call(w.rows(1, 2.0 ** t), [16 * 3 + t])
    w.call(w.rows(3, 0.01), [16 * 3 + t for t in (5, 6, 7)])
    w.call(w.rows(8, 30.0), [16 * 3 + t for t in range(8, 16)])
    w.call(w.rows(45), list(range(16 * 5 + 3, 16 * 8)))
    w.call(w.rows(9, 4.0), [0, 1, 2, 16 * 9 + 15, 16 * 10, 16 * 10 + 1, 16 * 1 + 4, 16 * 2 + 9, 16 * 2 + 10])


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 96])
def test_sequences_of_many_lengths(lcr, gpu, variant, d):
    """Ragged sequences at any place in their blocks, pages in any order, page sizes."""
    for page in (16, 48, 64):
        w = Writer(lcr, variant, heads=2, kv=3, d=d, page=page, pool=40, seed=d + page)
        for step in range(4):
            slots, free = [], list(w.r.permutation(w.cache.pool))
            for n in w.r.integers(1, 2 * page + 20, 6):
                at = int(w.r.integers(0, page))
                pages = [free.pop() for _ in range((at + n - 1) // page + 1)]
                slots += [pages[(at + i) // page] * page + (at + i) % page for i in range(n)]
            w.call(w.rows(len(slots), float(10.0 ** (step - 2))), slots)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 63, 64, 65, 255, 256, 257, 1030, 2100])
def test_many_tokens(lcr, gpu, tokens):
    w = Writer(lcr, "bf16", heads=4, kv=2, d=64, page=32, pool=tokens // 32 + 3, seed=tokens)
    w.call(w.rows(tokens), np.arange(5, 5 + tokens))


def test_many_sequences(lcr, gpu):
    """A token each of 1500 sequences, most of them within their blocks."""
    w = Writer(lcr, "bf16", heads=2, kv=2, d=64, page=16, pool=1600, seed=4)
    slots = 16 * w.r.permutation(1600)[:1500] + w.r.integers(0, 16, 1500)
    w.call(w.rows(1500, 0.05), slots)
    w.call(w.rows(1500, 3.0), np.minimum(slots + 1, slots // 16 * 16 + 15))


@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("changed", [
    dict(extra_stride=8), dict(extra_stride=3), dict(shift=1), dict(shift=4), dict(head_pad=16, page_pad=32),
    dict(scale_head_pad=3, scale_page_pad=1), dict(kv=0), dict(heads=0), dict(eps=0.5), dict(page=112),
], ids=str)
def test_layouts(lcr, gpu, d, changed):
    w = Writer(lcr, "bf16", **{**dict(heads=8, kv=4, d=d, pool=4, seed=7), **changed})
    w.call(w.rows(21), np.arange(3, 24))
    w.call(w.rows(5, 9.0), [24, 25, 26, 40, 41])


@pytest.mark.parametrize("d", [64, 128, 80])
def test_skipped_rows(lcr, gpu, d):
    """Rows without a slot or a position are left alone; those about them, in the
    same block even, are written as ever."""
    w = Writer(lcr, "bf16", heads=6, kv=2, d=d, pool=6, seed=3)
    slots = np.arange(10, 50)
    positions = np.arange(40)
    slots[[0, 7, 8, 39]] = [-1, -1, 6 * 16, 2 ** 31 - 1]
    slots[20] = -2 ** 31
    positions[[3, 12, 30]] = [-1, 64, 2 ** 31 - 1]
    w.call(w.rows(40), slots, positions)
    w.call(w.rows(3), [-1, -1, -1])


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 32])
def test_rewritten_positions(lcr, gpu, variant, d):
    """Drafts that were rejected are written over; the scale that they raised stays
    until the block begins again."""
    w = Writer(lcr, variant, heads=2, kv=2, d=d, norm=False, seed=9)
    w.call(w.rows(6), np.arange(0, 6))
    w.call(w.rows(4, 200.0), np.arange(6, 10))
    raised = w.cache.value_scales.copy()
    w.call(w.rows(4), np.arange(7, 11))
    assert (w.cache.value_scales == raised).all()
    w.call(w.rows(2), [0, 1])
    assert (w.cache.value_scales[w.cache.scales_at[0]] < raised[w.cache.scales_at[0]]).all()


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 16])
def test_scales_at_powers_of_two(lcr, gpu, variant, d):
    """A largest value of 448 2^k has scale 2^k, the next one above it 2^(k+1); zeros,
    the smallest values and the largest."""
    w = Writer(lcr, variant, heads=0, kv=1, d=d, norm=False, pool=2, seed=2)
    kind = w.kind
    largest = 65504.0 if variant == "fp16" else 3.38e38
    step = 2.0 ** -7 if variant == "bf16" else 2.0 ** -10
    for value in (448.0, 448.0 / 64, 7.0, 7.0 + 4 * step, 6.999, 3.5, 3.5 + 2 * step, 1.75 * 2.0 ** -12, 0.0, 1e-7,
                  2.0 ** -24, 1e-30, 61440.0, 63000.0, largest, -largest):
        x = np.zeros((3, w.stride), np.float32)
        x[0, :d] = np.linspace(-0.5, 0.5, d) * value
        x[1, d + 3] = value
        x[1, 5] = value
        x[2, :] = value * 0.001
        # no rotation: cos 1, sin 0
        w.table[:] = [1.0, 0.0]
        with np.errstate(over="ignore"):
            w.call(elems(x, kind), [16, 17, 18])
            w.call(elems(x * 0.9, kind), [19, 20, 21])


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("d", [64, 128, 48])
def test_infinities_and_nan(lcr, gpu, variant, norm, d):
    """Held as NaN, in their own elements (with a norm: their own head), and of no
    weight for the scale."""
    w = Writer(lcr, variant, heads=2, kv=2, d=d, norm=norm, seed=12)
    x = to_f32(w.rows(7), w.kind)
    at = 2 * d
    x[0, at] = np.inf
    x[1, at + d + 3] = np.nan
    x[2, at + 2 * d + 1] = -np.inf
    x[3, at + 3 * d : at + 4 * d] = np.nan
    x[4, at : at + 4 * d] = np.inf
    w.call(elems(x, w.kind), [2, 3, 4, 5, 6, 7, 8])
    w.call(w.rows(3, 50.0), [9, 10, 11])  # NaN stays NaN at a larger scale
    assert (w.cache.values[w.cache.at[0]] == ref.NAN).any()


def test_offsets_past_32_bits(lcr, gpu):
    """Pages that lie 2^28 bytes apart."""
    d, kv, pool, stride = 64, 2, 18, 1 << 28
    w = Writer(lcr, "bf16", heads=2, kv=kv, d=d, norm=False, pool=pool, seed=5)
    keys, values = (lcr.DeviceBuffer(pool * stride, np.dtype(np.uint8), pool * stride) for _ in range(2))
    c = w.cache
    scales = [dev(np.ones(pool * c.scale_page_stride, np.float32)) for _ in range(2)]
    qkv, slots = w.rows(20), np.arange(16 * 17 - 4, 16 * 18, dtype=np.int32)
    c.on_device = [keys, values, *scales]
    view = c.view(lcr, p)
    view.page_stride = stride
    src, q_out = dev(qkv), dev(np.zeros(20 * 2 * d, np.uint16))
    w.table[:] = [1.0, 0.0]
    status = w.lib.lcr_batch_norm_rope_write_kv8(
        p(q_out), ctypes.byref(view), p(src), p(src) + 2 * 2 * d, p(src) + 2 * 4 * d, None, None, 1e-5,
        p(dev(w.table)), 64, p(dev(np.zeros(20, np.int32))), p(dev(slots)), 20, 2, pool, w.stride, None)
    assert status == 0, w.lib.lcr_last_error_message()
    x = to_f32(qkv, w.kind).astype(np.float64)[4:]
    for which, buf, first, blocks_of in ((0, keys, 2, ref.to_blocks), (1, values, 4, ref.values_to_blocks)):
        got = np.empty(kv * 16 * d, np.uint8)
        from helpers import sync
        sync()
        lcr.check(w.lib, w.lib.lcr_memcpy_dtoh(got.ctypes.data, p(buf) + 17 * stride, got.size))
        scale = host(scales[which], np.float32)[17 * c.scale_page_stride :][:kv]
        for h in range(kv):
            want = x[:, (first + h) * d : (first + h + 1) * d]
            assert scale[h] == ref.scale_for(np.abs(want).max(), "bf16")
            assert (blocks_of(got.reshape(kv, -1)[h]) == ref.encode(want / scale[h])).all()


def test_same_bits_again(lcr, gpu):
    """The same call gives the same bits, also upon what it left."""
    w = Writer(lcr, "fp16", heads=4, kv=2, d=128, pool=6, seed=8)
    qkv, slots, positions = w.rows(60), np.arange(7, 67), np.arange(60)
    w.call(qkv, slots, positions)
    first = [x.copy() for x in (w.cache.keys, w.cache.values, w.cache.key_scales, w.cache.value_scales)]
    w.call(qkv, slots, positions)
    for a, b in zip(first, (w.cache.keys, w.cache.values, w.cache.key_scales, w.cache.value_scales)):
        expect_bits_equal(a.view(np.uint8), b.view(np.uint8), "again")


@pytest.mark.parametrize("d", [64, 128, 48])
def test_slots_that_break_the_rules(lcr, gpu, d):
    """The same slot for many rows, a block's rows far apart: of those blocks nothing is
    said, the others keep what they held and the queries are as ever."""
    w = Writer(lcr, "bf16", heads=3, kv=2, d=d, norm=False, pool=8, seed=14)
    c = w.cache
    for slots in (np.full(40, 33), np.tile([16, 70, 17, 71, 40], 20), np.arange(100) % 32, np.arange(64)[::-1] % 48):
        was = [x.copy() for x in (c.keys, c.values, c.key_scales, c.value_scales)]
        w.call(w.rows(len(slots)), slots, np.zeros(len(slots)), check=False)
        touched, touched_scales = np.zeros(c.keys.size, bool), np.zeros(c.key_scales.size, bool)
        for slot in set(slots.tolist()):
            page, n = slot // 16, 0
            touched[c.at[page, :, n]] = True
            touched_scales[c.scales_at[page, :, n]] = True
        for got, old in zip((c.keys, c.values), was[:2]):
            expect_bits_equal(got[~touched], old[~touched], "other blocks")
        for got, old in zip((c.key_scales, c.value_scales), was[2:]):
            expect_bits_equal(got[~touched_scales], old[~touched_scales], "other blocks' scales")
