"""A server's step with an 8-bit cache: map, write, attention, verification and log
probabilities one after another on a small two-layer model, against a 64-bit forward
over the cache that the device holds; the step captured and replayed for other lengths;
two steps at once."""

import ctypes

import numpy as np
import pytest

import batch_reference
import kv8_reference as ref
from helpers import BF16, dev, expect_bits_equal, host, p, rng, to_f32
from test_gpu_batch_logprobs import definition, near
from test_gpu_batch_step import (BATCH, D, EPS, HEADS, HIDDEN, KV, LAYERS, MAX_DRAFT, MAX_NEW, MAX_ROWS, PAGE, POOL,
                                 POSITIONS, STRIDE, VOCAB, WIDTH, Server, Stream, Weights, hip, run_steps, steps)

pytestmark = pytest.mark.gpu

TOP = 4


class Server8(Server):
    """The step of test_gpu_batch_step.py over caches of numbers."""

    def __init__(self, lcr, weights, seed):
        super().__init__(lcr, weights, seed)
        self.caches = [ref.Cache8(POOL, KV, PAGE, D, seed=seed + i) for i in range(LAYERS)]
        self.on_device = [c.upload(dev) for c in self.caches]
        self.views = [c.view(lcr, p, p(self.tables)) for c in self.caches]
        size = self.lib.lcr_batch_attention_kv8_workspace_bytes(BATCH, MAX_ROWS, MAX_NEW, HEADS, HEADS // KV, D)
        self.attention_ws, self.attention_size = dev(np.zeros(size + 16, np.uint8)), size
        size = self.lib.lcr_batch_logprobs_workspace_bytes(MAX_ROWS, TOP, VOCAB)
        self.logprobs_ws, self.logprobs_size = dev(np.zeros(size + 16, np.uint8)), size
        self.answers = [dev(np.zeros(MAX_ROWS * n, np.int32)) for n in (1, 1, 1, TOP, TOP)]

    def launch(self, stream=None, turn=None):
        lib, s = self.lib, stream.handle if stream else None
        turn = self.turn if turn is None else turn

        def ok(status):
            assert status == 0, lib.lcr_last_error_message()

        before, after = self.mapped[turn], self.mapped[1 - turn]
        ok(lib.lcr_batch_map(p(self.row_starts), p(self.positions), p(self.slots), p(self.lengths_out), p(after),
                             p(self.counts[1 - turn]), p(self.tables), p(self.lengths), p(self.new), p(before),
                             p(self.free), p(self.counts[turn]) + 4, BATCH, MAX_ROWS, STRIDE, PAGE, POOL, POOL, s))
        ok(lib.lcr_embedding_lookup(p(self.x), p(self.w["embed"]), p(self.ids), MAX_ROWS, HIDDEN, s))
        for layer, view in zip(self.layers, self.views):
            ok(lib.lcr_gemm(p(self.proj), 0, p(self.x), p(layer["qkv"]), MAX_ROWS, WIDTH, HIDDEN, s))
            ok(lib.lcr_batch_norm_rope_write_kv8(
                p(self.q), ctypes.byref(view), p(self.proj), p(self.proj) + 2 * HIDDEN,
                p(self.proj) + 2 * (HIDDEN + KV * D), p(layer["q_norm"]), p(layer["k_norm"]), EPS, p(self.w["rope"]),
                POSITIONS, p(self.positions), p(self.slots), MAX_ROWS, HEADS, POOL, WIDTH, s))
            ok(lib.lcr_batch_attention_kv8(
                p(self.mixed), p(self.q), ctypes.byref(view), p(self.row_starts), p(self.lengths_out), BATCH, MAX_ROWS,
                MAX_NEW, HEADS, HEADS // KV, STRIDE, POOL, HIDDEN, D ** -0.5, p(self.attention_ws),
                self.attention_size, s))
            ok(lib.lcr_gemm(p(self.delta), 0, p(self.mixed), p(layer["o"]), MAX_ROWS, HIDDEN, HIDDEN, s))
            ok(lib.lcr_add_residual(p(self.x), p(self.delta), MAX_ROWS * HIDDEN, s))
        ok(lib.lcr_gemm(p(self.logits), 1, p(self.x), p(self.w["head"]), MAX_ROWS, VOCAB, HIDDEN, s))
        ok(lib.lcr_batch_verify(p(self.out_ids), p(self.out_counts), p(self.logits), None, p(self.ids) + 4,
                                p(self.row_starts), p(self.heat), p(self.accept), p(self.sample), BATCH, MAX_ROWS,
                                MAX_DRAFT, VOCAB, VOCAB, p(self.verify_ws), self.verify_size, s))
        ok(lib.lcr_batch_logprobs(*[p(b) for b in self.answers], p(self.logits), p(self.ids) + 4, MAX_ROWS, TOP, VOCAB,
                                  VOCAB, p(self.logprobs_ws), self.logprobs_size, s))

    def read(self):
        got = super().read()
        got["answers"] = [host(b, np.int32).copy() for b in self.answers]
        got["caches"] = []
        for cache, bufs in zip(self.caches, self.on_device):
            cache.keys, cache.values = (host(b, np.uint8)[: cache.keys.size] for b in bufs[:2])
            cache.key_scales, cache.value_scales = (host(b, np.float32)[: cache.key_scales.size] for b in bufs[2:])
            got["caches"].append(cache.wide())
        got["tables"] = host(self.tables, np.int32).reshape(BATCH, STRIDE).copy()
        return got


def forward64(w, ids, start, table, caches):
    """Logits of the rows at positions start .. of one request, in 64 bits, over the
    keys and values that the caches stand for; and how far those are from this
    forward's own, relative to their size."""
    wide = lambda a: to_f32(a, BF16).astype(np.float64)  # noqa: E731
    n = len(ids)
    x = wide(w.embed)[ids]
    at = np.arange(start + n)
    far = []
    for i, (keys, values) in enumerate(caches):
        keys, values = (c[table[at // PAGE], :, at % PAGE] for c in (keys, values))
        proj = x @ wide(w.qkv[i]).T
        q, k, v = (proj[:, a:b].reshape(n, -1, D) for a, b in
                   ((0, HIDDEN), (HIDDEN, HIDDEN + KV * D), (HIDDEN + KV * D, WIDTH)))
        angles = w.rope[start:start + n].astype(np.float64)
        q, _ = batch_reference.rotate_heads(q, wide(w.q_norm[i]), EPS, angles)
        k, _ = batch_reference.rotate_heads(k, wide(w.k_norm[i]), EPS, angles)
        far += [np.sqrt(((c[start:] - y) ** 2).mean() / (y ** 2).mean()) for c, y in ((keys, k), (values, v))]
        out = np.zeros((n, HEADS, D))
        for h in range(HEADS):
            s = q[:, h] @ keys[:, h // (HEADS // KV)].T * D ** -0.5
            s = np.where(at <= start + np.arange(n)[:, None], s, -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            out[:, h] = e / e.sum(1, keepdims=True) @ values[:, h // (HEADS // KV)]
        x = x + out.reshape(n, HIDDEN) @ wide(w.o[i]).T
    return x @ wide(w.head).T, far


def test_steps_of_a_small_model(lcr, gpu):
    w = Weights(rng(131))
    server = Server8(lcr, w, 132)
    prompts, draws, drafts = steps(rng(133), 6)
    for i, lengths, now, got in run_steps(server, prompts, draws, drafts, server.launch):
        starts = got["starts"]
        ids = np.zeros(MAX_ROWS, np.int64)
        flat = [x for t in now for x in t]
        ids[: len(flat)] = flat
        for b in range(BATCH):
            if not now[b]:
                continue
            want, far = forward64(w, now[b], lengths[b], got["tables"][b], got["caches"])
            ours = got["logits"][starts[b]:starts[b + 1]]
            # Activations are rounded to bf16 at six places a layer, as in the step over
            # a 16-bit cache, from which this allowance is.
            size = np.sqrt((want ** 2).mean())
            assert np.sqrt(((ours - want) ** 2).mean()) <= 12 * 2.0 ** -8 * size, (i, b)
            # A number is off by up to 2^-4 of its value, and by what the activations are.
            assert max(far) <= 2.0 ** -4 + 12 * 2.0 ** -8, (i, b, far)
        drafted = np.concatenate([ids[1:], [0]])
        want_ids, want_counts = batch_reference.verify(got["logits"], None, drafted, starts, host(server.heat, np.float32),
                                                       *draws[i], MAX_DRAFT)
        if i > 0:  # the prompts' chunk is longer than the drafts that are taken
            assert got["counts"].tolist() == want_counts.tolist() and got["ids"].tolist() == want_ids.tolist()
        logprobs, ranks, entropies, top_ids, tops = got["answers"]
        for t in range(int(starts[-1])):
            want = definition(got["logits"][t], int(drafted[t]), TOP)
            near(logprobs.view(np.float32)[t], want["logprob"], np.array(want["allow"]), t)
            near(entropies.view(np.float32)[t], want["entropy"], np.array(want["allow_entropy"]), t)
            assert ranks[t] == want["rank"] and (top_ids.reshape(-1, TOP)[t] == want["ids"]).all()
            near(tops.view(np.float32).reshape(-1, TOP)[t], want["tops"], want["allow_tops"], t)


def kept(got):
    rows = int(got["starts"][-1])
    return [got["ids"].copy(), got["counts"].copy(), got["logits"][:rows].view(np.uint32).copy()] \
        + [a.reshape(MAX_ROWS, -1)[:rows].copy() for a in got["answers"]]


def test_captured_step_replays_for_other_lengths(lcr, gpu):
    """Two graphs, as the page counts alternate between two buffers; eager work between
    the replays (the reads); each has the eager step's bits."""
    w = Weights(rng(141))
    prompts, draws, drafts = steps(rng(142), 5)
    eager = Server8(lcr, w, 143)
    want = [kept(got) for _, _, _, got in run_steps(eager, prompts, draws, drafts, eager.launch)]
    server, stream, api = Server8(lcr, w, 143), Stream(), hip()
    graphs = []
    for turn in range(2):
        assert api.hipStreamBeginCapture(stream.handle, 0) == 0
        server.launch(stream, turn)
        graph, runner = ctypes.c_void_p(), ctypes.c_void_p()
        assert api.hipStreamEndCapture(stream.handle, ctypes.byref(graph)) == 0
        assert api.hipGraphInstantiate(ctypes.byref(runner), graph, None, None, ctypes.c_size_t(0)) == 0
        graphs.append((graph, runner))

    def replay():
        assert api.hipGraphLaunch(graphs[server.turn][1], stream.handle) == 0
        stream.wait()

    for (_, _, _, got), expected in zip(run_steps(server, prompts, draws, drafts, replay), want):
        for a, b in zip(kept(got), expected):
            expect_bits_equal(a, b, "a replay")
    for graph, runner in graphs:
        api.hipGraphExecDestroy(runner)
        api.hipGraphDestroy(graph)
    stream.close()


def test_two_steps_at_once(lcr, gpu):
    """Two servers, a stream and workspaces each: each gives what it gives alone. (The
    same step again writes what it wrote.)"""
    w = Weights(rng(151))
    plan, other_plan = (steps(rng(152 + i), 4) for i in range(2))
    alone = Server8(lcr, w, 160)
    want = [kept(got) for _, _, _, got in run_steps(alone, *plan, alone.launch)]
    server, other, streams = Server8(lcr, w, 160), Server8(lcr, w, 161), [Stream(), Stream()]
    other.set([0] * BATCH, [t[:-1] for t in other_plan[0]], *other_plan[1][0])

    def launch():
        for _ in range(3):
            other.launch(streams[1])
            server.launch(streams[0])
        for s in streams:
            s.wait()

    for (_, _, _, got), expected in zip(run_steps(server, *plan, launch), want):
        for a, b in zip(kept(got), expected):
            expect_bits_equal(a, b, "beside another")
    for s in streams:
        s.close()
