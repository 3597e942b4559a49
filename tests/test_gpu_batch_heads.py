"""lcr_batch_norm_rope_write_kv against its definition in 64 bits: every
compiled head_dim and the generic kernel, norms and none, strides, skipped rows.

Allowed: half a step of the output's rounding, and fp32's own roundings: the
mean square's sum (d terms), the reciprocal root, two products and the rotation,
at most (d + 12) 2^-24 of the two products whose difference an element is."""

import ctypes

import numpy as np
import pytest

import batch_reference
from helpers import BF16, FP16, dev, elems, expect_bits_equal, host, p, random_elems, rng, to_f32

pytestmark = pytest.mark.gpu

KINDS = {"bf16": BF16, "fp16": FP16}


def run_case(lcr, variant, *, tokens, heads, kv, d, page=16, norm=True, skip=(), extra_stride=0, shift=0, page_pad=0,
             head_pad=0, x_scale=1.0, far=0):
    gpu = lcr.load_library(variant)
    kind = KINDS[variant]
    r = rng(tokens * 7 + heads * 3 + d)
    stride = (heads + 2 * kv) * d + extra_stride
    qkv = random_elems(r, (tokens, stride), x_scale, kind)
    pool = -(-tokens // page) + 2
    slots = r.permutation(pool * page)[:tokens].astype(np.int32)
    positions = (far + r.integers(0, 50, tokens)).astype(np.int32)
    table_positions = far + 50
    for row, (slot, position) in dict(skip).items():
        slots[row] = slots[row] if slot is None else slot
        positions[row] = positions[row] if position is None else position
    live = (slots >= 0) & (slots < pool * page) & (positions >= 0) & (positions < table_positions)
    angle = np.arange(table_positions)[:, None] * 10000.0 ** (-np.arange(d // 2) / (d // 2))
    table = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    q_norm, k_norm = ((random_elems(r, d, 0.3, kind), random_elems(r, d, 0.3, kind)) if norm else (None, None))
    head_stride = page * d + head_pad
    page_stride = kv * head_stride + page_pad
    cache = [random_elems(r, pool * page_stride + 8, 1.0, kind) for _ in range(2)]
    q_before = random_elems(r, tokens * heads * d + 8, 1.0, kind)
    # `shift` elements into each buffer: rows off the 16-byte grid
    src = dev(np.concatenate([np.zeros(shift, np.uint16), qkv.ravel()]))
    bufs = [dev(c) for c in cache]
    q_out = dev(q_before)
    view = lcr.KvView(p(bufs[0]) + 2 * shift, p(bufs[1]) + 2 * shift, None, page, page_stride, head_stride, kv, d)
    base = p(src) + 2 * shift
    w = [p(dev(x)) if x is not None else None for x in (q_norm, k_norm)]
    status = gpu.lcr_batch_norm_rope_write_kv(p(q_out), ctypes.byref(view), base, base + 2 * heads * d,
                                              base + 2 * (heads + kv) * d, *w, 1e-5, p(dev(table)), table_positions,
                                              p(dev(positions)), p(dev(slots)), tokens, heads, pool, stride, None)
    assert status == 0, gpu.lcr_last_error_message()

    x = to_f32(qkv, kind).astype(np.float64)
    angles = table.astype(np.float64)[np.where(live, positions, 0)]
    wide = lambda a: None if a is None else to_f32(a, kind).astype(np.float64)  # noqa: E731

    def close(got, want, size, what):
        half = batch_reference.HALF_STEP[variant]
        # fp16 below its normal range: half of the smallest subnormal
        allow = half * np.abs(want) * (1 + half) + (d + 12) * 2.0 ** -24 * size
        allow += 2.0 ** -25 if variant == "fp16" else 1e-38
        off = np.abs(got.astype(np.float64) - want)
        worst = np.unravel_index(np.argmax(off - allow), off.shape) if off.size else None
        assert off.size == 0 or (off <= allow).all(), (what, worst, got[worst], want[worst], allow[worst])

    got_q = host(q_out)
    expect_bits_equal(got_q[tokens * heads * d:], q_before[tokens * heads * d:], "behind the queries")
    got_q = got_q[: tokens * heads * d].reshape(tokens, heads, d)
    before = q_before[: tokens * heads * d].reshape(tokens, heads, d)
    expect_bits_equal(got_q[~live], before[~live], "a skipped row's queries")
    want, size = batch_reference.rotate_heads(x[:, : heads * d].reshape(tokens, heads, d), wide(q_norm), 1e-5, angles)
    close(to_f32(got_q[live], kind), want[live], size[live], "queries")

    keys = x[:, heads * d : (heads + kv) * d].reshape(tokens, kv, d)
    want, size = batch_reference.rotate_heads(keys, wide(k_norm), 1e-5, angles)
    rows = np.nonzero(live)[0]
    at = shift + (slots[rows, None, None] // page * page_stride + np.arange(kv)[:, None] * head_stride
                  + slots[rows, None, None] % page * d + np.arange(d))
    got_k, got_v = host(bufs[0]), host(bufs[1])
    if kv:
        close(to_f32(got_k[at], kind), want[rows], size[rows], "keys")
        expect_bits_equal(got_v[at], qkv[rows][:, (heads + kv) * d : (heads + 2 * kv) * d], "values")
    for got, was in ((got_k, cache[0]), (got_v, cache[1])):
        rest = np.ones(got.size, bool)
        rest[at.ravel()] = False
        expect_bits_equal(got[rest], was[rest], "the rest of the cache")


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("tokens,heads,kv,d", [
    (1, 32, 8, 64), (1, 1, 1, 64), (7, 32, 8, 64), (77, 16, 8, 128), (33, 4, 4, 256), (5, 3, 1, 128), (130, 8, 1, 64),
    (9, 4, 2, 96), (4, 2, 2, 2), (6, 5, 5, 80), (3, 2, 1, 512), (2, 1, 1, 34), (300, 32, 8, 64),
])
def test_heads(lcr, gpu, variant, norm, tokens, heads, kv, d):
    run_case(lcr, variant, tokens=tokens, heads=heads, kv=kv, d=d, norm=norm)


@pytest.mark.parametrize("variant", ["bf16", "fp16"])
@pytest.mark.parametrize("changed", [
    dict(extra_stride=8), dict(extra_stride=3), dict(shift=1), dict(shift=4), dict(page_pad=24, head_pad=8),
    dict(page_pad=5), dict(page=1), dict(page=7), dict(kv=0), dict(heads=0), dict(x_scale=50.0), dict(x_scale=1e-3),
    dict(far=131000),
], ids=str)
def test_heads_layouts(lcr, gpu, variant, changed):
    run_case(lcr, variant, **{**dict(tokens=21, heads=8, kv=4, d=64), **changed})


@pytest.mark.parametrize("d", [64, 128, 48])
def test_heads_skips_rows(lcr, gpu, d):
    """Slots and positions outside the pool and the table leave their rows alone."""
    skip = {0: (-1, -1), 3: (None, -1), 4: (-1, None), 9: (10 ** 6, None), 10: (None, 50), 11: (2 ** 31 - 1, 2 ** 31 - 1),
            19: (-2 ** 31, None)}
    run_case(lcr, "bf16", tokens=20, heads=6, kv=2, d=d, skip=tuple(skip.items()))
    run_case(lcr, "bf16", tokens=3, heads=6, kv=2, d=d, skip=tuple({i: (-1, -1) for i in range(3)}.items()))


@pytest.mark.parametrize("d", [64, 80])
def test_heads_special_values(lcr, gpu, d):
    """An infinite or NaN element spoils its own head alone (its pair alone
    without a norm), and zeros stay zeros."""
    r = rng(5)
    heads, kv, tokens = 4, 1, 6
    x = to_f32(random_elems(r, (tokens, (heads + 2 * kv) * d)))
    x[0, 0], x[1, d + 3], x[2, 2 * d : 3 * d] = np.inf, np.nan, 0.0
    qkv = elems(x)
    table = np.stack([np.full((1, d // 2), 0.6), np.full((1, d // 2), 0.8)], -1).astype(np.float32)
    for norm in (True, False):
        keys, values, q_out = dev(np.zeros(16 * d, np.uint16)), dev(np.zeros(16 * d, np.uint16)), \
            dev(np.zeros(tokens * heads * d, np.uint16))
        view = lcr.KvView(p(keys), p(values), None, 16, 16 * d, 16 * d, kv, d)
        src = dev(qkv)
        w = p(dev(elems(np.ones(d, np.float32)))) if norm else None
        status = gpu.lcr_batch_norm_rope_write_kv(
            p(q_out), ctypes.byref(view), p(src), p(src) + 2 * heads * d, p(src) + 2 * (heads + kv) * d, w, w, 1e-5,
            p(dev(table)), 1, p(dev(np.zeros(tokens, np.int32))), p(dev(np.arange(tokens, dtype=np.int32))), tokens,
            heads, 1, (heads + 2 * kv) * d, None)
        assert status == 0
        got = to_f32(host(q_out)).reshape(tokens, heads, d)
        spoilt = ~np.isfinite(got)
        assert (got[2, 2] == 0).all()
        if norm:
            assert spoilt[1, 1].all() and not np.isfinite(got[0, 0, [0, d // 2]]).any()
        else:
            assert spoilt[0, 0].nonzero()[0].tolist() == [0, d // 2]
            assert spoilt[1, 1].nonzero()[0].tolist() == [3, 3 + d // 2]
        spoilt[0, 0] = spoilt[1, 1] = False
        assert not spoilt.any()
