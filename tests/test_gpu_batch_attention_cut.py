"""lcr_batch_attention where tables are wide enough for units of keys to be cut
over the device and joined: the same definition, allowances and cases as for
one launch, and the workspace's use by captured, repeated and concurrent calls."""

import ctypes

import numpy as np
import pytest

from helpers import dev, elems, expect_bits_equal, host, p, random_elems, rng, to_f32
from test_gpu_batch_attention import LENGTHS, Case
from test_gpu_batch_step import Stream, hip

pytestmark = pytest.mark.gpu


def wide(case, positions=1100):
    """The case with entries of no use behind its tables."""
    more = -(-positions // case.page) - case.tables.shape[1]
    if more > 0:
        case.tables = np.pad(case.tables, ((0, 0), (0, more)), constant_values=-1)
    return case


@pytest.mark.parametrize("variant,heads,kv,d", [("bf16", 32, 8, 64), ("fp16", 8, 4, 128), ("bf16", 5, 1, 72)])
@pytest.mark.parametrize("past,new", LENGTHS, ids=str)
def test_wide_tables(lcr, gpu, variant, heads, kv, d, past, new):
    wide(Case(variant, past, new, heads=heads, kv=kv, d=d, seed=sum(past) + 3 * sum(new), tail=3)).check(lcr)


@pytest.mark.parametrize("heads,kv,d", [(1, 1, 64), (2, 2, 64), (12, 4, 64), (16, 1, 64), (33, 1, 64), (40, 2, 64),
                                        (130, 1, 64), (4, 4, 128), (14, 2, 128), (33, 1, 128), (260, 1, 128)])
@pytest.mark.parametrize("past,new", [
    ([575], [1]), ([576], [1]), ([640], [2]), ([2100], [1]), ([1500, 0, 900], [1, 1, 3]), ([1200], [16]),
    ([1200], [17]), ([1200], [33]), ([0], [1200]), ([700, 3000], [0, 1]), ([800, 1300, 10], [0, 0, 1]),
    ([1100, 5, 2050], [40, 1, 9]), ([900] * 6, [1, 2, 3, 4, 5, 6]),
], ids=str)
def test_cut_units(lcr, gpu, heads, kv, d, past, new):
    if heads > 100 and sum(new) > 100:
        new = [min(n, 30) for n in new]
    wide(Case("bf16", past, new, heads=heads, kv=kv, d=d, seed=heads + sum(new))).check(lcr)


@pytest.mark.parametrize("changed", [
    dict(page=1), dict(page=3), dict(page=5), dict(page=8), dict(page=12), dict(page=24), dict(page=48), dict(page=64),
    dict(page=100), dict(page=1000), dict(extra_stride=8), dict(extra_stride=1), dict(shift=8), dict(shift=1),
    dict(page_pad=40), dict(head_pad=16),
], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_cut_layouts(lcr, gpu, d, changed):
    wide(Case("fp16", [1700, 0, 650, 9], [2, 20, 1, 90], heads=8, kv=2, d=d, seed=d, **changed)).check(lcr)


@pytest.mark.parametrize("d", [64, 128])
def test_cut_rows_that_see_nothing_and_lengths_past_the_table(lcr, gpu, d):
    c = wide(Case("bf16", [20, 1500, 0], [3, 4, 2], heads=4, kv=2, d=d, seed=9))
    c.lengths = np.array([23, 2, 0], np.int32)
    ours = c.check(lcr)
    assert (ours[3:5] == 0).all() and (ours[5] != 0).any() and (ours[7:9] == 0).all()
    c.lengths = np.array([-3, 1504, -2 ** 31], np.int32)
    c.check(lcr)
    c = Case("bf16", [1500, 1500], [2, 30], heads=4, kv=2, d=d, seed=10)
    c.lengths = np.array([1502, 2 ** 31 - 1], np.int32)
    c.check(lcr)


@pytest.mark.parametrize("d", [64, 128])
def test_cut_large_scores(lcr, gpu, d):
    """The largest score in one piece, or rising from piece to piece."""
    for sign in (1.0, -1.0):
        c = wide(Case("bf16", [1900], [3], heads=4, kv=1, d=d, seed=8, q_scale=4.0))
        ramp = np.abs(sign * np.linspace(0, 6, 1903)) if sign > 0 else np.linspace(6, 0, 1903)
        for position in range(1903):
            at = c.position_index(0, 0, position)
            c.keys[at:at + d] = elems(to_f32(c.keys[at:at + d]) * np.float32(ramp[position]))
        c.check(lcr)


@pytest.mark.parametrize("variant,d", [("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_cut_masked_places_hold_anything(lcr, gpu, variant, d, value):
    for past, new in (([1470], [1]), ([1437], [5]), ([1100], [90])):
        c = wide(Case(variant, past, new, heads=4, kv=1, d=d, seed=12))
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
        at = c.position_index(0, 0, past[0] + new[0] - 2)
        c.values[at + 3] = bits
        got = c.run(lcr)
        expect_bits_equal(got[: new[0] - 2], clean[: new[0] - 2], "rows before the value")
        seen = to_f32(got[new[0] - 2:], c.kind)
        assert (np.isnan(seen[..., 3]) if np.isnan(value) else (seen[..., 3] == value)).all()
        assert (np.delete(seen, 3, -1) == np.delete(to_f32(clean[new[0] - 2:], c.kind), 3, -1)).all()
        # one seen by every row, in a piece that is not the last
        c.values[c.position_index(0, 0, 40) + 7] = bits
        seen = to_f32(c.run(lcr), c.kind)
        assert (np.isnan(seen[..., 7]) if np.isnan(value) else (seen[..., 7] == value)).all()
        assert (np.delete(seen[: new[0] - 2], 7, -1) ==
                np.delete(to_f32(clean[: new[0] - 2], c.kind), 7, -1)).all()


@pytest.mark.parametrize("d", [64, 128])
def test_cut_pages_outside_the_pool(lcr, gpu, d):
    """In each piece of the sequence: NaN or no trace, and the others' bits."""
    c = wide(Case("bf16", [70, 1970, 900], [2, 1, 40], heads=4, kv=2, d=d, seed=13))
    clean = c.run(lcr)
    for at in (2, 60, 122):
        kept = c.tables[1, at]
        for bad in (-1, c.pool, 2 ** 31 - 1, -2 ** 31):
            c.tables[1, at] = bad
            got = c.run(lcr)
            expect_bits_equal(got[:2], clean[:2], "the sequence before")
            expect_bits_equal(got[3:], clean[3:], "the sequence behind")
            assert np.isnan(to_f32(got[2])).all()
        c.tables[1, at] = kept


class Held:
    """A call's buffers, kept for further calls on other lengths."""

    def __init__(self, lcr, case, max_new, workspace=None):
        self.lib, self.case, self.max_new = lcr.load_library(case.variant), case, max_new
        self.q, self.keys, self.values = dev(case.q), dev(case.keys), dev(case.values)
        self.tables, self.starts, self.lengths = dev(case.tables), dev(case.starts), dev(case.lengths)
        self.view = lcr.KvView(p(self.keys), p(self.values), p(self.tables), case.page, case.page_stride,
                               case.head_stride, case.kv, case.d)
        self.out = dev(np.zeros(case.tokens * case.heads * case.d, np.uint16))
        self.size = self.lib.lcr_batch_attention_workspace_bytes(len(case.past), case.tokens, max_new, case.heads,
                                                                 case.heads // case.kv, case.d)
        self.ws = workspace or dev(np.full(self.size // 4 + 4, np.nan, np.float32))

    def set(self, past, new):
        """Other lengths of the same sequences, within what their pages hold."""
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        lengths = (np.asarray(past) + np.asarray(new)).astype(np.int32)
        for buf, values in ((self.starts, starts), (self.lengths, lengths)):
            assert self.lib.lcr_memcpy_htod(p(buf), values.ctypes.data, values.nbytes) == 0
        zero = np.zeros(self.case.tokens * self.case.heads * self.case.d, np.uint16)
        assert self.lib.lcr_memcpy_htod(p(self.out), zero.ctypes.data, zero.nbytes) == 0
        self.case.starts, self.case.lengths = starts, lengths

    def launch(self, stream=None):
        c = self.case
        assert self.lib.lcr_batch_attention(
            p(self.out), p(self.q), ctypes.byref(self.view), p(self.starts), p(self.lengths), len(c.past), c.tokens,
            self.max_new, c.heads, c.heads // c.kv, c.tables.shape[1], c.pool, c.q_stride, c.scale, p(self.ws),
            self.size, stream.handle if stream else None) == 0, self.lib.lcr_last_error_message()

    def read(self):
        c = self.case
        return host(self.out).reshape(c.tokens, c.heads, c.d)

    def check(self, got):
        want, allow = self.case.want()
        live = int(self.case.starts[-1])
        assert (got[live:] == 0).all()
        assert (np.abs(to_f32(got[:live], self.case.kind) - want[:live]) <= allow[:live]).all()


CHANGES = [([2000, 700, 0], [1, 3, 40]), ([5, 2500, 1000], [40, 1, 1]), ([0, 0, 0], [1, 1, 1]), ([2500, 2500, 2500], [1, 1, 1]),
           ([100, 2470, 1200], [0, 30, 14]), ([2450, 0, 2400], [4, 0, 40]), ([2000, 700, 0], [1, 3, 40])]


@pytest.mark.parametrize("variant,heads,kv,d", [("bf16", 8, 2, 64), ("fp16", 6, 3, 128), ("bf16", 40, 1, 64)])
def test_captured_attention_replays_for_other_lengths(lcr, gpu, variant, heads, kv, d):
    """One capture; every replay, with eager work between, has the eager bits."""
    case = Case(variant, [2500] * 3, [20] * 3, heads=heads, kv=kv, d=d, seed=30)
    held, stream, api = Held(lcr, case, 40), Stream(), hip()
    graph, runner = ctypes.c_void_p(), ctypes.c_void_p()
    assert api.hipStreamBeginCapture(stream.handle, 0) == 0
    held.launch(stream)
    assert api.hipStreamEndCapture(stream.handle, ctypes.byref(graph)) == 0
    assert api.hipGraphInstantiate(ctypes.byref(runner), graph, None, None, ctypes.c_size_t(0)) == 0
    for past, new in CHANGES:
        held.set(past, new)
        held.launch()
        eager = held.read()
        held.check(eager)
        held.set(past, new)
        assert api.hipGraphLaunch(runner, stream.handle) == 0
        stream.wait()
        expect_bits_equal(held.read(), eager, "replayed")
    api.hipGraphExecDestroy(runner)
    api.hipGraphDestroy(graph)
    stream.close()


def test_two_calls_at_once(lcr, gpu):
    """On two streams, a workspace each: each call's own bits."""
    cases = [Case("bf16", [2500] * 3, [20] * 3, heads=8, kv=2, d=64, seed=31),
             Case("bf16", [4000, 900], [1, 1], heads=16, kv=2, d=128, seed=32)]
    helds, streams = [Held(lcr, c, 20) for c in cases], [Stream(), Stream()]
    alone = []
    for h in helds:
        h.launch()
        alone.append(h.read())
        h.check(alone[-1])
    for _ in range(5):
        for _ in range(10):
            for h, s in zip(helds, streams):
                h.launch(s)
        for s in streams:
            s.wait()
        for h, want in zip(helds, alone):
            expect_bits_equal(h.read(), want, "at once")
    for s in streams:
        s.close()


def test_one_workspace_for_calls_of_other_shapes(lcr, gpu):
    """One after another in a workspace of the largest: nothing of an earlier
    call is seen by a later one."""
    cases = [Case("bf16", [3000, 2000], [1, 1], heads=8, kv=2, d=64, seed=33),
             Case("bf16", [1500] * 5, [9] * 5, heads=8, kv=1, d=128, seed=34),
             Case("bf16", [1200], [100], heads=4, kv=4, d=64, seed=35),
             Case("bf16", [1300], [1], heads=4, kv=4, d=72, seed=36)]
    alone = [Held(lcr, c, 100) for c in cases]
    shared = dev(np.full(max(h.size for h in alone) // 4 + 4, np.nan, np.float32))
    together = [Held(lcr, c, 100, shared) for c in cases]
    for h in alone:
        h.launch()
        h.check(h.read())
    for _ in range(3):
        for h in together:
            h.launch()
        for h, one in zip(together, alone):
            expect_bits_equal(h.read(), one.read(), "in a shared workspace")


@pytest.mark.parametrize("d", [64, 128])
def test_workspace_of_any_size(lcr, gpu, d):
    """None, too small and just enough: within the allowance, nothing past its end."""
    case = Case("bf16", [2500, 800], [1, 20], heads=8, kv=2, d=d, seed=37)
    held = Held(lcr, case, 20)
    size = held.size
    for take in (size, size - 1, 16, 0):
        guard = random_elems(rng(5), size // 2 + 64)
        held.ws = dev(guard)
        held.size = take
        held.launch()
        held.check(held.read())
        if take == size:
            expect_bits_equal(host(held.ws)[size // 2:], guard[size // 2:], "behind the workspace")
        else:
            expect_bits_equal(host(held.ws), guard, "a workspace that is too small")


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
def test_scales(lcr, gpu, scale):
    for d in (64, 128, 72):
        c = Case("bf16", [1300, 5], [2, 7], heads=4, kv=2, d=d, seed=38)
        c.scale = scale
        c.check(lcr)


@pytest.mark.parametrize("positions", [None, 1100])
@pytest.mark.parametrize("d", [64, 128])
def test_infinities_in_many_tiles_of_a_unit(lcr, gpu, d, positions):
    """Values that only a unit's later rows see, in neighbouring tiles and in
    every second one: each reaches its element of the rows from its position
    on, and nothing else changes."""
    for past, new in (([0], [600]), ([330, 0], [290, 410])):
        c = Case("bf16", past, new, heads=1, kv=1, d=d, seed=39)
        if positions:
            wide(c, positions)
        clean = c.run(lcr)
        expected = to_f32(clean, c.kind).copy()
        r = rng(40)
        for b, (first, n) in enumerate(zip(c.starts, new)):
            at = sorted(r.choice(n - 2, 9, replace=False).tolist()) + [n - 2]
            for dim, (i, value) in enumerate(zip(at, [np.inf, -np.inf, np.nan] * 4)):
                c.values[c.position_index(b, 0, past[b] + i) + dim] = elems(np.array([value], np.float32), c.kind)[0]
                expected[first + i:first + n, 0, dim] = value
        got = to_f32(c.run(lcr), c.kind)
        assert (np.isnan(got) == np.isnan(expected)).all()
        assert ((got == expected) | np.isnan(expected)).all()
