"""The batched operators as a step of a server uses them, one after another: a
small two-layer model over several requests, with drafted tokens, against a
64-bit forward of each request by itself; the step captured into a graph and
replayed for other lengths; two steps at once on two streams."""

import ctypes

import numpy as np
import pytest

import batch_reference
from helpers import BF16, dev, elems, expect_bits_equal, host, p, random_elems, rng, to_f32

pytestmark = pytest.mark.gpu

HEADS, KV, D, PAGE, VOCAB, LAYERS = 4, 2, 64, 16, 700, 2
HIDDEN = HEADS * D
WIDTH = (HEADS + 2 * KV) * D
BATCH, MAX_ROWS, STRIDE, POOL, MAX_NEW, MAX_DRAFT = 5, 64, 40, 150, 40, 3
POSITIONS = STRIDE * PAGE
EPS = 1e-5


def hip():
    lib = ctypes.CDLL("libamdhip64.so")
    for name in ("hipStreamCreateWithFlags", "hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate",
                 "hipGraphLaunch", "hipStreamSynchronize", "hipGraphExecDestroy", "hipGraphDestroy", "hipStreamDestroy"):
        getattr(lib, name).restype = ctypes.c_int
    return lib


class Stream:
    def __init__(self):
        self.hip = hip()
        self.handle = ctypes.c_void_p()
        assert self.hip.hipStreamCreateWithFlags(ctypes.byref(self.handle), ctypes.c_uint(1)) == 0

    def wait(self):
        assert self.hip.hipStreamSynchronize(self.handle) == 0

    def close(self):
        self.hip.hipStreamDestroy(self.handle)


class Weights:
    def __init__(self, r):
        self.embed = random_elems(r, (VOCAB, HIDDEN))
        self.qkv = [random_elems(r, (WIDTH, HIDDEN), 0.08) for _ in range(LAYERS)]
        self.o = [random_elems(r, (HIDDEN, HIDDEN), 0.08) for _ in range(LAYERS)]
        self.q_norm = [elems(1 + 0.2 * r.normal(size=D)) for _ in range(LAYERS)]
        self.k_norm = [elems(1 + 0.2 * r.normal(size=D)) for _ in range(LAYERS)]
        self.head = random_elems(r, (VOCAB, HIDDEN), 0.1)
        angle = np.arange(POSITIONS)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))
        self.rope = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)


class Server:
    """Device buffers of a step, and the step."""

    def __init__(self, lcr, weights, seed):
        self.lib = lcr.load_library("bf16")
        r = rng(seed)
        i32 = lambda n, v=0: dev(np.full(n, v, np.int32))  # noqa: E731
        u16 = lambda *n: dev(np.zeros(n, np.uint16))  # noqa: E731
        w = weights
        self.w = {k: dev(getattr(w, k)) for k in ("embed", "head", "rope")}
        self.layers = [{k: dev(getattr(w, k)[i]) for k in ("qkv", "o", "q_norm", "k_norm")} for i in range(LAYERS)]
        self.pools = [(u16(POOL, KV, PAGE, D), u16(POOL, KV, PAGE, D)) for _ in range(LAYERS)]
        self.tables = i32(BATCH * STRIDE, -1)
        self.views = [lcr.KvView(p(k), p(v), p(self.tables), PAGE, KV * PAGE * D, PAGE * D, KV, D)
                      for k, v in self.pools]
        self.free = dev(r.permutation(POOL).astype(np.int32))
        self.mapped = [i32(BATCH), i32(BATCH)]
        self.counts = [dev(np.array([0, POOL], np.int32)), i32(2)]
        self.lengths, self.new, self.lengths_out = i32(BATCH), i32(BATCH), i32(BATCH)
        self.row_starts, self.positions, self.slots = i32(BATCH + 1), i32(MAX_ROWS), i32(MAX_ROWS)
        self.ids = i32(MAX_ROWS + 1)  # read from its second entry on as each row's drafted token
        self.x, self.proj, self.q, self.mixed = (u16(MAX_ROWS, HIDDEN), u16(MAX_ROWS, WIDTH), u16(MAX_ROWS, HIDDEN),
                                                 u16(MAX_ROWS, HIDDEN))
        self.delta = u16(MAX_ROWS, HIDDEN)
        self.logits = dev(np.zeros((MAX_ROWS, VOCAB), np.float32))
        self.accept, self.sample = dev(np.zeros(MAX_ROWS, np.float32)), dev(np.zeros(BATCH, np.float32))
        self.heat = dev(np.array([0.8, 0.0, 1.0, 0.7, 0.0], np.float32))
        self.out_ids, self.out_counts = i32(BATCH * (MAX_DRAFT + 1)), i32(BATCH)
        size = self.lib.lcr_batch_attention_workspace_bytes(BATCH, MAX_ROWS, MAX_NEW, HEADS, HEADS // KV, D)
        self.attention_ws, self.attention_size = dev(np.zeros(size + 16, np.uint8)), size
        size = self.lib.lcr_batch_verify_workspace_bytes(BATCH, MAX_ROWS, VOCAB)
        self.verify_ws, self.verify_size = dev(np.zeros(size + 16, np.uint8)), size
        self.turn = 0

    def put(self, buf, values):
        a = np.ascontiguousarray(values)
        assert self.lib.lcr_memcpy_htod(p(buf), a.ctypes.data, a.nbytes) == 0

    def launch(self, stream=None, turn=None):
        """Every launch of a step, none of which waits."""
        lib, s = self.lib, stream.handle if stream else None
        turn = self.turn if turn is None else turn
        ok = lambda status: (_ for _ in ()).throw(AssertionError(lib.lcr_last_error_message())) if status else None  # noqa: E731
        before, after = self.mapped[turn], self.mapped[1 - turn]
        left = p(self.counts[turn]) + 4
        ok(lib.lcr_batch_map(p(self.row_starts), p(self.positions), p(self.slots), p(self.lengths_out), p(after),
                             p(self.counts[1 - turn]), p(self.tables), p(self.lengths), p(self.new), p(before),
                             p(self.free), left, BATCH, MAX_ROWS, STRIDE, PAGE, POOL, POOL, s))
        ok(lib.lcr_embedding_lookup(p(self.x), p(self.w["embed"]), p(self.ids), MAX_ROWS, HIDDEN, s))
        for layer, view in zip(self.layers, self.views):
            ok(lib.lcr_gemm(p(self.proj), 0, p(self.x), p(layer["qkv"]), MAX_ROWS, WIDTH, HIDDEN, s))
            ok(lib.lcr_batch_norm_rope_write_kv(
                p(self.q), ctypes.byref(view), p(self.proj), p(self.proj) + 2 * HIDDEN,
                p(self.proj) + 2 * (HIDDEN + KV * D), p(layer["q_norm"]), p(layer["k_norm"]), EPS, p(self.w["rope"]),
                POSITIONS, p(self.positions), p(self.slots), MAX_ROWS, HEADS, POOL, WIDTH, s))
            ok(lib.lcr_batch_attention(p(self.mixed), p(self.q), ctypes.byref(view), p(self.row_starts),
                                       p(self.lengths_out), BATCH, MAX_ROWS, MAX_NEW, HEADS, HEADS // KV, STRIDE, POOL,
                                       HIDDEN, D ** -0.5, p(self.attention_ws), self.attention_size, s))
            ok(lib.lcr_gemm(p(self.delta), 0, p(self.mixed), p(layer["o"]), MAX_ROWS, HIDDEN, HIDDEN, s))
            ok(lib.lcr_add_residual(p(self.x), p(self.delta), MAX_ROWS * HIDDEN, s))
        ok(lib.lcr_gemm(p(self.logits), 1, p(self.x), p(self.w["head"]), MAX_ROWS, VOCAB, HIDDEN, s))
        ok(lib.lcr_batch_verify(p(self.out_ids), p(self.out_counts), p(self.logits), None, p(self.ids) + 4,
                                p(self.row_starts), p(self.heat), p(self.accept), p(self.sample), BATCH, MAX_ROWS,
                                MAX_DRAFT, VOCAB, VOCAB, p(self.verify_ws), self.verify_size, s))

    def set(self, lengths, tokens, accept, sample):
        """A step's inputs: positions kept, and each request's new token ids."""
        self.put(self.lengths, np.asarray(lengths, np.int32))
        self.put(self.new, np.array([len(t) for t in tokens], np.int32))
        ids = np.zeros(MAX_ROWS, np.int32)
        flat = [x for t in tokens for x in t]
        ids[: len(flat)] = flat
        self.put(self.ids, ids)
        self.put(self.accept, accept)
        self.put(self.sample, sample)

    def read(self):
        return {"ids": host(self.out_ids, np.int32).reshape(BATCH, MAX_DRAFT + 1),
                "counts": host(self.out_counts, np.int32), "lengths": host(self.lengths_out, np.int32),
                "logits": host(self.logits, np.float32).reshape(MAX_ROWS, VOCAB).copy(),
                "starts": host(self.row_starts, np.int32)}


def forward64(w, ids):
    """Logits of every position of one request, in 64 bits."""
    wide = lambda a: to_f32(a, BF16).astype(np.float64)  # noqa: E731
    n = len(ids)
    x = wide(w.embed)[ids]
    for i in range(LAYERS):
        proj = x @ wide(w.qkv[i]).T
        q, k, v = (proj[:, a:b].reshape(n, -1, D) for a, b in
                   ((0, HIDDEN), (HIDDEN, HIDDEN + KV * D), (HIDDEN + KV * D, WIDTH)))
        angles = w.rope[:n].astype(np.float64)
        q, _ = batch_reference.rotate_heads(q, wide(w.q_norm[i]), EPS, angles)
        k, _ = batch_reference.rotate_heads(k, wide(w.k_norm[i]), EPS, angles)
        out = np.zeros((n, HEADS, D))
        for h in range(HEADS):
            s = q[:, h] @ k[:, h // (HEADS // KV)].T * D ** -0.5
            s = np.where(np.tri(n, dtype=bool), s, -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            out[:, h] = e / e.sum(1, keepdims=True) @ v[:, h // (HEADS // KV)]
        x = x + out.reshape(n, HIDDEN) @ wide(w.o[i]).T
    return x @ wide(w.head).T


def steps(r, count):
    """The requests' prompts, then drafts after whatever was generated."""
    prompts = [r.integers(0, VOCAB, n).tolist() for n in (17, 1, 30, 5, 2)]
    draws = [(r.random(MAX_ROWS).astype(np.float32), r.random(BATCH).astype(np.float32)) for _ in range(count)]
    drafts = [[r.integers(0, VOCAB, int(r.integers(0, MAX_DRAFT + 1))).tolist() for _ in range(BATCH)]
              for _ in range(count)]
    return prompts, draws, drafts


def run_steps(server, prompts, draws, drafts, launch):
    """Drives the server; yields each step's lengths, tokens and results."""
    lengths = [0] * BATCH
    # the prompts but for their last token, from which the drafts go on
    tokens = [t[:-1] for t in prompts]
    for i, ((accept, sample), draft) in enumerate(zip(draws, drafts)):
        if i == 0:
            now = tokens
        elif i == 1:
            now = [[t[-1]] + d for t, d in zip(prompts, draft)]
        else:
            now = [[nxt] + d for nxt, d in zip(following, draft)]
        server.set(lengths, now, accept, sample)
        launch()
        got = server.read()
        yield i, lengths, now, got
        server.turn ^= 1
        if i == 0:
            lengths = [len(t) for t in now]
            kept = [list(t) for t in now]
            continue
        following = []
        for b in range(BATCH):
            n = int(got["counts"][b])
            kept[b] += now[b][:n]
            lengths[b] = len(kept[b])
            following.append(int(got["ids"][b, n - 1]))


def test_steps_of_a_small_model(lcr, gpu):
    """Logits of every row near the 64-bit forward of its request alone; ids
    exactly what the device's own logits say."""
    w = Weights(rng(31))
    server = Server(lcr, w, 32)
    prompts, draws, drafts = steps(rng(33), 6)
    texts = [[] for _ in range(BATCH)]
    for i, lengths, now, got in run_steps(server, prompts, draws, drafts, server.launch):
        starts = got["starts"]
        assert starts.tolist() == np.concatenate([[0], np.cumsum([len(t) for t in now])]).tolist()
        assert got["lengths"].tolist() == [a + len(t) for a, t in zip(lengths, now)]
        for b in range(BATCH):
            texts[b] = texts[b][: lengths[b]] + now[b]
            if not now[b]:
                continue
            want = forward64(w, texts[b])[lengths[b]:]
            ours = got["logits"][starts[b]:starts[b + 1]]
            # A row's activations are rounded to bf16 at six places a layer (x,
            # projection, head, weights, mixed, delta), each by 2^-8 of its size,
            # and pass two products of gain below 2 (0.08 sqrt(256) = 1.3): well
            # within 12 roundings of the logits' size.
            size = np.sqrt((want ** 2).mean())
            assert np.sqrt(((ours - want) ** 2).mean()) <= 12 * 2.0 ** -8 * size, (i, b)
        ids = np.zeros(MAX_ROWS, np.int64)
        flat = [x for t in now for x in t]
        ids[: len(flat)] = flat
        drafted = np.concatenate([ids[1:], [0]])
        want_ids, want_counts = batch_reference.verify(got["logits"], None, drafted, starts, host(server.heat, np.float32),
                                                       *draws[i], MAX_DRAFT)
        if i > 0:  # the prompts' chunk is longer than the drafts that are taken
            assert got["counts"].tolist() == want_counts.tolist() and got["ids"].tolist() == want_ids.tolist()


def test_captured_step_replays_for_other_lengths(lcr, gpu):
    """One captured step (two graphs: the page counts alternate between two
    buffers), replayed for prompts and drafts of other lengths with eager work
    between, gives the eager steps' bits each time."""
    w = Weights(rng(41))
    prompts, draws, drafts = steps(rng(42), 5)
    eager = Server(lcr, w, 43)
    want = [(got["ids"].copy(), got["counts"].copy(), got["logits"], got["starts"])
            for _, _, _, got in run_steps(eager, prompts, draws, drafts, eager.launch)]
    server, stream, api = Server(lcr, w, 43), Stream(), hip()
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

    for (_, _, now, got), (ids, counts, logits, starts) in zip(run_steps(server, prompts, draws, drafts, replay), want):
        rows = int(starts[-1])
        expect_bits_equal(got["starts"], starts, "row starts")
        expect_bits_equal(got["logits"][:rows].view(np.uint32), logits[:rows].view(np.uint32), "logits")
        assert got["counts"].tolist() == counts.tolist() and got["ids"].tolist() == ids.tolist()
    for graph, runner in graphs:
        api.hipGraphExecDestroy(runner)
        api.hipGraphDestroy(graph)
    stream.close()


def test_two_steps_at_once(lcr, gpu):
    """Two servers, a stream and workspaces each, launched without waiting for
    each other: each gives what it gives alone."""
    w = Weights(rng(51))
    plans = [steps(rng(52 + i), 4) for i in range(2)]
    alone = []
    for i, plan in enumerate(plans):
        server = Server(lcr, w, 60 + i)
        alone.append([(g["ids"].copy(), g["counts"].copy(), g["logits"][: g["starts"][-1]].copy())
                      for _, _, _, g in run_steps(server, *plan, server.launch)])
    servers, streams = [Server(lcr, w, 60 + i) for i in range(2)], [Stream(), Stream()]

    def together(i):
        # the other server's step is on its stream at the same time, again and
        # again on the same inputs (a step's outputs do not feed the same step)
        def launch():
            other = servers[1 - i]
            for _ in range(3):
                other.launch(streams[1 - i])
                servers[i].launch(streams[i])
            for s in streams:
                s.wait()
        return launch

    for i, plan in enumerate(plans):
        other_prompts, other_draws, _ = plans[1 - i]
        servers[1 - i].set([0] * BATCH, [t[:-1] for t in other_prompts], *other_draws[0])
        for (_, _, _, got), (ids, counts, logits) in zip(run_steps(servers[i], *plan, together(i)), alone[i]):
            rows = int(got["starts"][-1])
            expect_bits_equal(got["logits"][:rows].view(np.uint32), logits.view(np.uint32), "logits")
            assert got["counts"].tolist() == counts.tolist() and got["ids"].tolist() == ids.tolist()
        servers = [Server(lcr, w, 60 + k) for k in range(2)]
    for s in streams:
        s.close()
