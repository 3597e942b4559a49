"""lcr_batch_logprobs against its definition in 64 bits. Whole numbers are equal.

Allowed, with e = 2^-24 and d = l - max: a weight exp(d) takes its argument from two
fp32 roundings and a rounded constant, and the exponential's own two: 4 e |d| + 4 e
of its size. Up to 64 factors and terms of such an error lead to a sum (16 are added
in fp32, and a lane's largest rises a few times): 64 e. So the sum
S is off by S_rel = e (4 E|d| + 68) of its size, and log S by as much; a log
probability by that, d's rounding and its own. The entropy log S - E d: by S_rel,
by the weights' errors in the weighted sum, sum p |d| (4 e |d| + 5 e) + 64 e E|d|, and
by E|d| S_rel for the division, and its own rounding."""

import numpy as np
import pytest

from helpers import dev, expect_bits_equal, host, p, rng, sync, zeros_dev

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
MARK = 0x5A5A5A5A


def definition(row, token, top):
    """(logprob, rank, entropy, ids, logprobs), and what the three may be off by."""
    x = np.where(np.isnan(row), -np.inf, row).astype(np.float64)
    vocab = x.size
    order = np.argsort(-x, kind="stable")
    most = x[order[0]]
    if np.isfinite(most):
        with np.errstate(invalid="ignore"):
            d = np.where(x == -np.inf, -np.inf, x - most)
        w = np.exp(d)
        s = w.sum()
        lp = d - np.log(s)
        mean = lambda f: (w[w > 0] * f(d[w > 0])).sum() / s  # noqa: E731
        size, square = mean(np.abs), mean(np.square)
        entropy = np.log(s) + size
        s_rel = E * (4 * size + 68)
        allow_lp = s_rel + 3 * E * np.abs(lp)
        allow_entropy = s_rel + E * (4 * square + 5 * size) + 64 * E * size + size * s_rel + E * entropy + 1e-37
    else:
        lp = np.where(np.arange(vocab) == order[0], 0.0, -np.inf)
        entropy, allow_lp, allow_entropy = 0.0, np.zeros(vocab), 0.0
    ids = np.full(top, -1, np.int64)
    tops = np.full(top, -np.inf)
    n = min(top, int((x > -np.inf).sum()))
    ids[:n], tops[:n] = order[:n], lp[order[:n]]
    inside = 0 <= token < vocab
    return dict(logprob=lp[token] if inside else -np.inf, rank=int((x > x[token]).sum()) if inside else vocab,
                entropy=entropy, ids=ids, tops=tops, allow=allow_lp[token] if inside else 0.0,
                allow_entropy=allow_entropy, allow_tops=np.concatenate([allow_lp[ids[:n]], np.zeros(top - n)]))


def near(got, want, allow, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    # fp32 ends at FLT_MAX = (2 - 2^-23) 2^127 = 3.40e38: a log probability below
    # -(2 - 2^-24) 2^127, such as FLT_MAX's negative less FLT_MAX, rounds to -inf
    want = np.where(want <= -(2 - 2.0 ** -24) * 2.0 ** 127, -np.inf, want)
    infinite = ~np.isfinite(want)
    assert (got[infinite] == want[infinite]).all(), (what, got, want)
    off = np.abs(got[~infinite] - want[~infinite])
    assert (off <= np.asarray(allow)[~infinite]).all(), (what, got, want, allow)


class Call:
    def __init__(self, lcr, logits, tokens, top, *, vocab=None, shift=0, workspace=True):
        """logits [rows][stride] of which the first `vocab` count."""
        self.lcr, self.lib = lcr, lcr.load_library()
        self.logits, self.tokens, self.top = logits, tokens, top
        self.rows, self.stride = logits.shape
        self.vocab = self.stride if vocab is None else vocab
        self.shift = shift
        self.src = dev(np.concatenate([np.zeros(shift, np.float32), logits.ravel().astype(np.float32)]))
        self.ids = None if tokens is None else dev(np.asarray(tokens, np.int32))
        size = self.lib.lcr_batch_logprobs_workspace_bytes(self.rows, top, self.vocab) if workspace else 0
        self.ws = (dev(np.full(size // 4 + 4, np.nan, np.float32)), size) if size else (None, 0)
        mark = lambda n: dev(np.full(n + 4, MARK, np.int32))  # noqa: E731
        self.out = dict(logprobs=mark(self.rows), ranks=mark(self.rows), entropies=mark(self.rows),
                        top_ids=mark(self.rows * top), top_logprobs=mark(self.rows * top))
        if tokens is None:
            self.out["logprobs"] = self.out["ranks"] = None

    def run(self, stream=None, **without):
        arg = [None if b is None or name in without else p(b) for name, b in self.out.items()]
        if not self.top:
            arg[3] = arg[4] = None
        ws, size = self.ws
        status = self.lib.lcr_batch_logprobs(*arg, p(self.src) + 4 * self.shift, None if self.ids is None else p(self.ids),
                                             self.rows, self.top, self.vocab, self.stride,
                                             None if ws is None else p(ws), size, stream)
        assert status == 0, self.lib.lcr_last_error_message()
        return self

    def outputs(self):
        return {k: None if b is None else host(b, np.int32) for k, b in self.out.items()}

    def check(self):
        got = self.outputs()
        for name, b in got.items():
            if b is not None:
                n = self.rows * self.top if name.startswith("top") else self.rows
                assert (b[n:] == MARK).all(), name
        f = lambda name: got[name].view(np.float32)  # noqa: E731
        for t in range(self.rows):
            token = -1 if self.tokens is None else int(self.tokens[t])
            at = slice(t * self.top, (t + 1) * self.top)
            if self.tokens is not None and token < 0:
                for name, b in got.items():
                    assert (b[at if name.startswith("top") else slice(t, t + 1)] == MARK).all(), (name, t)
                continue
            want = definition(self.logits[t, : self.vocab], token, self.top)
            near(f("entropies")[t], want["entropy"], np.array(want["allow_entropy"]), ("entropy", t))
            assert (got["top_ids"][at] == want["ids"]).all(), (t, got["top_ids"][at], want["ids"])
            near(f("top_logprobs")[at], want["tops"], want["allow_tops"], ("top", t))
            if self.tokens is not None:
                assert got["ranks"][t] == want["rank"], (t, got["ranks"][t], want["rank"])
                near(f("logprobs")[t], want["logprob"], np.array(want["allow"]), ("logprob", t))
        return got


def both(lcr, logits, tokens, top, **more):
    """With a workspace and without."""
    Call(lcr, logits, tokens, top, **more).run().check()
    Call(lcr, logits, tokens, top, workspace=False, **more).run().check()


def normal(r, rows, vocab, std=3.0):
    return r.normal(0, std, (rows, vocab)).astype(np.float32)


@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
@pytest.mark.parametrize("vocab", [1, 2, 5, 31, 32, 33, 63, 64, 65, 100, 255, 256, 257, 1000, 1023, 1025, 4095, 4096, 4097, 8191, 8200,
                                   16385, 50001])
def test_vocabularies(lcr, gpu, vocab, top):
    r = rng(vocab + top)
    rows = 3
    both(lcr, normal(r, rows, vocab), r.integers(0, vocab, rows), top)


@pytest.mark.parametrize("top", [0, 3, 32])
@pytest.mark.parametrize("rows", [1, 2, 17, 64, 255, 256, 257, 700])
def test_rows(lcr, gpu, rows, top):
    r = rng(rows)
    vocab = 6007
    both(lcr, normal(r, rows, vocab), r.integers(0, vocab, rows), top)


@pytest.mark.parametrize("top", [0, 7, 20])
def test_whole_vocabulary(lcr, gpu, top):
    r = rng(top)
    x = normal(r, 5, 128256, 2.5)
    x[1, 77777] += 25.0
    x[2] *= 8.0
    both(lcr, x, [0, 77777, int(x[2].argmax()), 128255, 5], top)


@pytest.mark.parametrize("top", [1, 20, 32])
@pytest.mark.parametrize("vocab", [70, 5000, 40000])
def test_equal_logits(lcr, gpu, vocab, top):
    """Ties go to the lowest id: few values, one value, ties only at the cut."""
    r = rng(vocab * top)
    x = np.zeros((6, vocab), np.float32)
    x[0] = r.integers(0, 3, vocab)
    x[1] = r.integers(0, 200, vocab) / 8
    x[2] = 1.5
    x[3] = -0.0
    x[3, ::2] = 0.0  # zeros of both signs are equal
    x[4, r.permutation(vocab)[:10]] = 4.0
    x[5] = np.repeat(r.normal(0, 1, vocab // 10 + 1), 10)[:vocab]
    both(lcr, x, r.integers(0, vocab, 6), top)


@pytest.mark.parametrize("top", [1, 20, 32])
@pytest.mark.parametrize("vocab", [100, 5000, 66000])
def test_orders(lcr, gpu, vocab, top):
    """The largest last, first, all in one lane's or one part's ids, one after another."""
    x = np.zeros((6, vocab), np.float32)
    up = np.arange(vocab, dtype=np.float32) / 64
    x[0], x[1] = up, up[::-1]
    x[2, ::64] = up[::64] + 1
    x[3, : vocab // 2] = 3.0 + up[: vocab // 2] / 100
    x[4] = np.where(np.arange(vocab) % 256 < 4, up + 5, -up)
    x[5, -40:] = up[:40] + 9
    both(lcr, x, [vocab - 1, 0, 0, 1, vocab // 2, vocab - 3], top)


@pytest.mark.parametrize("vocab", [9, 300, 5000, 20000])
def test_masked_and_special(lcr, gpu, vocab):
    """Masks of -inf and of the type's lowest value, rows that leave nothing, NaN,
    infinities."""
    r = rng(vocab)
    low = np.finfo(np.float32).min
    x = normal(r, 14, vocab)
    x[0, r.random(vocab) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, vocab // 2] = 3.0
    x[3, r.random(vocab) < 0.9] = low
    x[4] = low
    x[5, r.random(vocab) < 0.5] = np.nan
    x[6] = np.nan
    x[7, vocab // 3] = np.inf
    x[8, [vocab // 3, vocab - 1]] = np.inf
    x[9] = np.inf
    x[10, : vocab // 2] = np.nan
    x[10, vocab // 2:] = -np.inf
    x[11] = np.where(np.arange(vocab) % 2, low, -low)
    x[12, 0], x[12, vocab - 1] = np.inf, np.nan
    x[13, 1:] = -np.inf
    x[5].view(np.uint32)[np.isnan(x[5])] = 0x7F800001  # signalling
    for top in (0, 1, 8, 32):
        both(lcr, x, r.integers(0, vocab, 14), top)
        both(lcr, x, [0] * 14, top)
        both(lcr, x, [vocab // 3] * 14, top)


@pytest.mark.parametrize("vocab", [1000, 33333])
def test_large_and_far_logits(lcr, gpu, vocab):
    r = rng(vocab)
    x = normal(r, 8, vocab)
    x[0] += 1000.0
    x[1] -= 30000.0
    x[2] *= 1e4
    x[3] *= 1e30
    x[4] *= 1e-30
    x[5] *= 1e-42
    x[6, 5] += 80.0
    x[7] += 3e38 * 0.9
    both(lcr, x, r.integers(0, vocab, 8), 12)


@pytest.mark.parametrize("changed", [dict(stride=1), dict(stride=3), dict(stride=4), dict(stride=5000), dict(shift=1),
                                     dict(shift=2), dict(shift=3, stride=2), dict(shift=4)], ids=str)
@pytest.mark.parametrize("vocab", [1000, 8193, 20004])
def test_strides_and_alignment(lcr, gpu, vocab, changed):
    """What lies between the rows counts for nothing."""
    r = rng(vocab)
    x = np.full((7, vocab + changed.get("stride", 0)), np.inf, np.float32)
    x[:, :vocab] = normal(r, 7, vocab)
    both(lcr, x, r.integers(0, vocab, 7), 9, vocab=vocab, shift=changed.get("shift", 0))


@pytest.mark.parametrize("rows", [5, 400])
def test_rows_left_out(lcr, gpu, rows):
    r = rng(rows)
    vocab = 9001
    tokens = r.integers(0, vocab, rows)
    tokens[::3] = -1
    tokens[1] = -2 ** 31
    tokens[4] = vocab          # past the vocabulary: no row is left out for it
    tokens[2] = 2 ** 31 - 1
    both(lcr, normal(r, rows, vocab), tokens, 6)
    both(lcr, normal(r, rows, vocab), [-1] * rows, 6)


@pytest.mark.parametrize("vocab", [100, 30000])
def test_without_tokens(lcr, gpu, vocab):
    both(lcr, normal(rng(1), 6, vocab), None, 4)
    both(lcr, normal(rng(2), 600, vocab // 10), None, 0)


def test_outputs_not_wanted(lcr, gpu):
    x, tokens = normal(rng(3), 4, 20000), [5, 6, 7, 8]
    for name in ("logprobs", "ranks", "entropies"):
        for workspace in (True, False):
            whole = Call(lcr, x, tokens, 3, workspace=workspace).run().check()
            got = Call(lcr, x, tokens, 3, workspace=workspace).run(**{name: 0}).outputs()
            assert (got[name] == MARK).all()
            for other in set(whole) - {name}:
                expect_bits_equal(got[other], whole[other], other)


def test_rows_past_32_bits(lcr, gpu):
    """Rows that lie 2^28 floats apart."""
    r, vocab, stride, rows = rng(6), 3001, 1 << 28, 10
    x = normal(r, rows, vocab)
    buf = lcr.DeviceBuffer(4 * ((rows - 1) * stride + vocab), np.dtype(np.float32), 0, zero=False)
    for t in range(rows):
        lcr.check(gpu, gpu.lcr_memcpy_htod(buf.ptr + 4 * t * stride, np.ascontiguousarray(x[t]).ctypes.data, 4 * vocab))
    for workspace in (True, False):
        call = Call(lcr, x, r.integers(0, vocab, rows), 5, workspace=workspace)
        call.src, call.stride = buf, stride
        call.run().check()


def test_same_bits_again(lcr, gpu):
    x = normal(rng(8), 40, 128256)
    tokens = rng(9).integers(0, 128256, 40)
    first = Call(lcr, x, tokens, 20).run().outputs()
    again = Call(lcr, x, tokens, 20)
    for _ in range(3):
        got = again.run().outputs()
        for name in first:
            expect_bits_equal(got[name], first[name], name)


def test_a_smaller_workspace(lcr, gpu):
    """One that does not suffice is not used."""
    call = Call(lcr, normal(rng(10), 2, 50000), [1, 2], 5)
    need = gpu.lcr_batch_logprobs_workspace_bytes(2, 5, 50000)
    ws = zeros_dev(max(need, 64) // 4, np.int32)
    call.ws = (ws, max(need - 16, 0)) if need else (None, 0)
    call.run().check()
    sync()


@pytest.mark.parametrize("rows,vocab,top", [(1, 128256, 32), (100, 30000, 5), (128, 9000, 20)])
def test_a_workspace_keeps_what_lies_behind_it(lcr, gpu, rows, vocab, top):
    call = Call(lcr, normal(rng(rows), rows, vocab), rng(1).integers(0, vocab, rows), top)
    size = call.ws[1]
    assert size > 0
    guard = np.full(size + 4096, 0x5A, np.uint8)
    call.ws = (dev(guard), size)
    call.run().check()
    expect_bits_equal(host(call.ws[0], np.uint8)[size:], guard[size:], "behind the workspace")
