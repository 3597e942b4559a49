"""Calls of the 8-bit attention and of log probabilities as programs make them:
captured once and replayed for other lengths, two at once on two streams, workspaces of
other shapes and sizes, whatever a workspace held before."""

import ctypes

import numpy as np
import pytest

from helpers import dev, expect_bits_equal, host, p, rng, to_f32
from test_gpu_batch_kv8_attention import Case
from test_gpu_batch_logprobs import Call, normal
from test_gpu_batch_step import Stream, hip

pytestmark = pytest.mark.gpu


class Held:
    """A case's buffers on the device, for several launches."""

    def __init__(self, lcr, case, max_new):
        self.case, self.lib, self.max_new = case, lcr.load_library(case.variant), max_new
        c = case
        self.out, self.q = dev(np.zeros(c.tokens * c.heads * c.d, np.uint16)), dev(c.q)
        c.cache.upload(dev)
        self.tables, self.starts, self.lengths = dev(c.tables), dev(c.starts), dev(c.lengths)
        self.view = c.cache.view(lcr, p, p(self.tables))
        self.size = self.lib.lcr_batch_attention_kv8_workspace_bytes(len(c.past), c.tokens, max_new, c.heads,
                                                                     c.heads // c.kv, c.d)
        self.ws = dev(np.full(self.size // 4 + 4, np.nan, np.float32))

    def launch(self, stream=None, ws=None, size=None):
        c = self.case
        status = self.lib.lcr_batch_attention_kv8(
            p(self.out), p(self.q), ctypes.byref(self.view), p(self.starts), p(self.lengths), len(c.past), c.tokens,
            self.max_new, c.heads, c.heads // c.kv, c.tables.shape[1], c.pool, c.q_stride, c.scale,
            p(ws or self.ws), self.size if size is None else size, stream.handle if stream else None)
        assert status == 0, self.lib.lcr_last_error_message()

    def set_lengths(self, new, lengths):
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        for buf, a in ((self.starts, starts), (self.lengths, np.asarray(lengths, np.int32))):
            assert self.lib.lcr_memcpy_htod(p(buf), a.ctypes.data, a.nbytes) == 0
        return int(starts[-1])

    def result(self, rows):
        return host(self.out)[: rows * self.case.heads * self.case.d].copy()


@pytest.mark.parametrize("variant,heads,kv,d", [("bf16", 8, 2, 64), ("fp16", 4, 2, 128), ("bf16", 2, 1, 48)])
@pytest.mark.parametrize("most", [1, 40])
def test_captured_attention_replays_for_other_lengths(lcr, gpu, variant, heads, kv, d, most):
    case = Case(variant, [2600, 1300, 50], [most] * 3, heads=heads, kv=kv, d=d, seed=31)
    held, stream, api = Held(lcr, case, most), Stream(), hip()
    graph, runner = ctypes.c_void_p(), ctypes.c_void_p()
    assert api.hipStreamBeginCapture(stream.handle, 0) == 0
    held.launch(stream)
    assert api.hipStreamEndCapture(stream.handle, ctypes.byref(graph)) == 0
    assert api.hipGraphInstantiate(ctypes.byref(runner), graph, None, None, ctypes.c_size_t(0)) == 0
    r = rng(5)
    for _ in range(6):
        new = r.integers(0, most + 1, 3)
        rows = held.set_lengths(new, [int(r.integers(0, n + 1)) for n in case.lengths])
        held.launch()
        want = held.result(rows)
        assert held.lib.lcr_device_memset(p(held.out), 0x55, want.size * 2) == 0
        assert api.hipGraphLaunch(runner, stream.handle) == 0
        stream.wait()
        expect_bits_equal(held.result(rows), want, "a replay")
    api.hipGraphExecDestroy(runner)
    api.hipGraphDestroy(graph)
    stream.close()


def test_two_attentions_at_once(lcr, gpu):
    cases = [Case("bf16", [3000, 40], [1, 60], heads=8, kv=2, seed=41), Case("bf16", [1500, 2000], [2, 1], heads=8, kv=2, seed=42)]
    held = [Held(lcr, c, int(c.new.max())) for c in cases]
    want = []
    for h in held:
        h.launch()
        want.append(h.result(h.case.tokens))
    streams = [Stream(), Stream()]
    for _ in range(20):
        for h, s in zip(held, streams):
            h.launch(s)
    for s in streams:
        s.wait()
    for h, w in zip(held, want):
        expect_bits_equal(h.result(h.case.tokens), w, "beside another")
    for s in streams:
        s.close()


def test_one_workspace_for_calls_of_other_shapes(lcr, gpu):
    shapes = [dict(past=[2000], new=[1], heads=8, kv=2, d=64), dict(past=[1500, 30], new=[50, 3], heads=8, kv=2, d=64),
              dict(past=[1800], new=[9], heads=4, kv=2, d=128), dict(past=[1200], new=[70], heads=4, kv=1, d=128)]
    held = [Held(lcr, Case("bf16", s.pop("past"), s.pop("new"), seed=i, **s), 70) for i, s in enumerate(shapes)]
    ws = dev(np.full(max(h.size for h in held) // 4 + 4, np.nan, np.float32))
    for _ in range(2):
        for h in held:
            h.launch(ws=ws, size=h.size)
            want, allow = h.case.want()
            got = to_f32(h.result(h.case.tokens)).reshape(want.shape)
            assert (np.abs(got - want) <= allow).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 8, 50])
def test_workspace_of_any_size(lcr, gpu, d, new):
    """One that does not suffice is not used: nothing is split then."""
    case = Case("bf16", [2100, 90], [new, 1], heads=4, kv=2, d=d, seed=51)
    want, allow = case.want()
    held = Held(lcr, case, new)
    for size in (0, 16, held.size // 2 // 16 * 16, held.size - 16, held.size):
        held.launch(size=size, ws=held.ws)
        got = to_f32(held.result(case.tokens)).reshape(want.shape)
        assert (np.abs(got - want) <= allow).all(), size


@pytest.mark.parametrize("rows,vocab,top", [(3, 50000, 5), (200, 9000, 20), (3, 50000, 0)])
def test_captured_logprobs_replay_for_other_logits(lcr, gpu, rows, vocab, top):
    r = rng(rows)
    call = Call(lcr, normal(r, rows, vocab), r.integers(0, vocab, rows), top)
    stream, api = Stream(), hip()
    graph, runner = ctypes.c_void_p(), ctypes.c_void_p()
    assert api.hipStreamBeginCapture(stream.handle, 0) == 0
    call.run(stream.handle)
    assert api.hipStreamEndCapture(stream.handle, ctypes.byref(graph)) == 0
    assert api.hipGraphInstantiate(ctypes.byref(runner), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(4):
        call.logits, call.tokens = normal(r, rows, vocab), r.integers(0, vocab, rows)
        for buf, a in ((call.src, call.logits), (call.ids, call.tokens.astype(np.int32))):
            assert call.lib.lcr_memcpy_htod(p(buf), np.ascontiguousarray(a).ctypes.data, a.nbytes) == 0
        assert api.hipGraphLaunch(runner, stream.handle) == 0
        stream.wait()
        replayed = call.check()
        for name, want in call.run().check().items():
            expect_bits_equal(replayed[name], want, name)
    api.hipGraphExecDestroy(runner)
    api.hipGraphDestroy(graph)
    stream.close()


def test_two_logprobs_at_once(lcr, gpu):
    calls = [Call(lcr, normal(rng(i), 20, 60000), rng(i).integers(0, 60000, 20), 10) for i in range(2)]
    want = [c.run().check() for c in calls]
    streams = [Stream(), Stream()]
    for _ in range(10):
        for c, s in zip(calls, streams):
            c.run(s.handle)
    for s in streams:
        s.wait()
    for c, w in zip(calls, want):
        for name, got in c.outputs().items():
            expect_bits_equal(got, w[name], name)
    for s in streams:
        s.close()


def test_one_workspace_for_logprobs_of_other_shapes(lcr, gpu):
    calls = [Call(lcr, normal(rng(i), rows, vocab), rng(i).integers(0, vocab, rows), top)
             for i, (rows, vocab, top) in enumerate([(1, 100000, 20), (60, 30000, 3), (5, 128256, 0), (100, 20000, 32)])]
    ws = dev(np.full(max(c.ws[1] for c in calls) // 4 + 4, np.nan, np.float32))
    for _ in range(2):
        for c in calls:
            if c.ws[0] is not None:
                c.ws = (ws, c.ws[1])
            c.run().check()


def test_masks_of_the_lowest_value(lcr, gpu):
    """Masked vocabularies: few ids left, all others the type's lowest value or -inf, in
    the largest size, split and not."""
    r, vocab = rng(77), 128256
    for masked in (np.finfo(np.float32).min, -np.inf):
        for rows in (4, 140):
            x = np.full((rows, vocab), masked, np.float32)
            for t in range(rows):
                left = r.permutation(vocab)[: int(r.integers(1, 40))]
                x[t, left] = r.normal(0, 3, len(left))
            Call(lcr, x, r.integers(0, vocab, rows), 20).run().check()
