"""lcr_batch_attention_kv8 with pages of more than 2^31 and 2^32 bytes a head."""

import ctypes

import numpy as np
import pytest

import batch_reference
import kv8_reference as ref
from helpers import BF16, dev, elems, host, p, random_elems, rng, to_f32

pytestmark = pytest.mark.gpu


def encoded(rows, before, which):
    """Blocks' bytes and scales of `rows`, with `before` positions of zeros ahead of
    them, and the values that they stand for."""
    late, d = rows.shape
    blocks = np.zeros(((before + late + 15) // 16 * 16, d))
    blocks[before : before + late] = rows
    blocks = blocks.reshape(-1, 16, d)
    scales = np.array([ref.scale_for(np.abs(b).max(), "bf16") for b in blocks])
    codes = ref.encode(blocks / scales[:, None, None])
    stand_for = (ref.NUMBERS[codes] * scales[:, None, None]).reshape(-1, d)[before : before + late]
    flat = codes.reshape(len(codes), -1) if which == "keys" else ref.values_from_blocks(codes)
    return np.ascontiguousarray(flat), scales.astype(np.float32), stand_for


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("new", [[2], [8], [40, 1]], ids=str)
@pytest.mark.parametrize("past", [1 << 31, 1 << 32])
@pytest.mark.parametrize("d", [64, 128])
def test_pages_past_31_and_32_bits(lcr, gpu, d, past, new, workspace):
    """One page of every sequence (its stride counts for nothing), whose last keys lie
    `past` bytes into it. Every key before them is zero and so are its values: its
    weight beside theirs is e^-60 at most, of all of them together under 1e-17, far
    under the allowance for the last keys alone."""
    r = rng(d + sum(new))
    late, heads, tokens, batch = 1500, 4, sum(new), len(new)
    page = past // d + 4096
    first = past // d + 103              # position of the first of them, within a block
    length = first + late
    assert first * d > past and length <= page
    # 8 * k * d^-0.5 is 80, give or take the other elements' share
    q = random_elems(r, (tokens, heads, d), 1.0, BF16)
    q[..., 0] = elems(np.array([8.0], np.float32))
    k, v = r.normal(0, 1, (late, d)), r.normal(0, 1, (late, d))
    k[:, 0] = 10.0 * d ** 0.5
    lib = lcr.load_library("bf16")
    pools, scales, wide = [], [], []
    for which, rows in (("keys", k), ("values", v)):
        codes, block_scales, stand_for = encoded(rows, first % 16, which)
        pool = lcr.DeviceBuffer(page * d, zero=True)
        lcr.check(lib, lib.lcr_memcpy_htod(pool.ptr + first // 16 * 16 * d, codes.ctypes.data, codes.nbytes))
        all_scales = np.ones(page // 16, np.float32)
        all_scales[first // 16 : first // 16 + len(block_scales)] = block_scales
        pools.append(pool)
        scales.append(dev(all_scales))
        wide.append(stand_for)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    out = dev(np.zeros(tokens * heads * d + 16, np.uint16))
    view = lcr.Kv8View(pools[0].ptr, pools[1].ptr, p(scales[0]), p(scales[1]), p(dev(np.zeros(batch, np.int32))), page,
                       0, 0, 0, 0, 1, d)
    size = lib.lcr_batch_attention_kv8_workspace_bytes(batch, tokens, max(new), heads, heads, d) if workspace else 0
    ws = dev(np.full(size // 4 + 4, np.nan, np.float32)) if size else None
    status = lib.lcr_batch_attention_kv8(
        p(out), p(dev(q)), ctypes.byref(view), p(dev(starts)), p(dev(np.full(batch, length, np.int32))), batch, tokens,
        max(new), heads, heads, 1, 1, heads * d, d ** -0.5, p(ws) if ws else None, size, None)
    assert status == 0, lib.lcr_last_error_message()
    got = host(out)
    for pool in pools:
        pool.free()
    assert (got[tokens * heads * d:] == 0).all()
    want, allow = batch_reference.attention(
        to_f32(q).astype(np.float64), wide[0][None, None], wide[1][None, None], np.zeros((batch, 1), np.int32), starts,
        np.full(batch, late, np.int32), late, d ** -0.5, "bf16")
    assert (np.abs(to_f32(got[: tokens * heads * d]).reshape(want.shape) - want) <= allow).all()
