"""lcr_batch_attention with pages of more than 2^31 elements a head."""

import ctypes

import numpy as np
import pytest

import batch_reference
from helpers import BF16, dev, elems, host, p, random_elems, rng, to_f32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("new", [2, 40])
@pytest.mark.parametrize("d,page", [(128, (1 << 24) + 4096), (64, (1 << 25) + 4096), (128, (1 << 24) + 4097)])
def test_pages_past_31_bits(lcr, gpu, d, page, new, workspace):
    """One page of the whole sequence (its stride counts for nothing), whose last
    keys lie 2^31 elements into it. Every key before them is zero and so are its
    values: its weight beside theirs is e^-60 at most, of all of them together
    under 1e-18, far under the allowance for the last keys alone."""
    r = rng(d + new)
    late, heads = 1500, 4
    first = (1 << 31) // d + 100            # position of the first of them
    length = first + late
    assert first * d > 1 << 31 and length <= page
    # 8 * k * d^-0.5 is 80, give or take the other elements' share
    q = random_elems(r, (new, heads, d), 1.0, BF16)
    k, v = random_elems(r, (late, d), 1.0, BF16), random_elems(r, (late, d), 1.0, BF16)
    q[..., 0], k[:, 0] = elems(np.array([8.0, 10.0 * d ** 0.5], np.float32))
    pools = [lcr.DeviceBuffer(2 * page * d, zero=True) for _ in range(2)]
    lib = lcr.load_library("bf16")
    for pool, part in zip(pools, (k, v)):
        part = np.ascontiguousarray(part)
        lcr.check(lib, lib.lcr_memcpy_htod(pool.ptr + 2 * first * d, part.ctypes.data, part.nbytes))
    starts, lengths = np.array([0, new], np.int32), np.array([length], np.int32)
    out = dev(np.zeros(new * heads * d + 16, np.uint16))
    view = lcr.KvView(pools[0].ptr, pools[1].ptr, p(dev(np.zeros(1, np.int32))), page, 0, 0, 1, d)
    size = lib.lcr_batch_attention_workspace_bytes(1, new, new, heads, heads, d) if workspace else 0
    ws = dev(np.full(size // 4 + 4, np.nan, np.float32)) if size else None
    status = lib.lcr_batch_attention(p(out), p(dev(q)), ctypes.byref(view), p(dev(starts)), p(dev(lengths)), 1, new, new,
                                     heads, heads, 1, 1, heads * d, d ** -0.5, p(ws) if ws else None, size, None)
    assert status == 0, lib.lcr_last_error_message()
    got = host(out)
    for pool in pools:
        pool.free()
    assert (got[new * heads * d:] == 0).all()
    wide = lambda a: to_f32(a).astype(np.float64)  # noqa: E731
    want, allow = batch_reference.attention(
        wide(q), wide(k)[None, None], wide(v)[None, None], np.zeros((1, 1), np.int32), starts,
        np.array([late], np.int32), late, d ** -0.5, "bf16")
    assert (np.abs(to_f32(got[: new * heads * d]).reshape(want.shape) - want) <= allow).all()
