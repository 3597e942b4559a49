"""lcr_batch_norm_rope_write_kv8 into pages of more than 2^31 and 2^32 bytes a head."""

import ctypes

import numpy as np
import pytest

import kv8_reference as ref
from helpers import dev, host, p, sync, to_f32
from test_gpu_batch_kv8_heads import Writer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("past", [1 << 31, 1 << 32])
@pytest.mark.parametrize("d", [64, 128, 48])
def test_blocks_past_31_and_32_bits(lcr, gpu, d, past):
    """Two blocks that lie `past` bytes into the one page, begun by one call, and the
    second's last row by another with larger values: it rounds the block anew."""
    w = Writer(lcr, "bf16", heads=1, kv=1, d=d, norm=False, pool=1, seed=d)
    w.table[:] = [1.0, 0.0]
    block = past // (16 * d) + 5
    page = 16 * (block + 2)
    pools = [lcr.DeviceBuffer(page * d, np.dtype(np.uint8), page * d) for _ in range(2)]
    scales = [dev(np.full(page // 16, 0.25, np.float32)) for _ in range(2)]
    view = lcr.Kv8View(p(pools[0]), p(pools[1]), p(scales[0]), p(scales[1]), None, page, 0, 0, 0, 0, 1, d)
    first, second = w.rows(31), w.rows(1, 300.0)
    for qkv, slots in ((first, 16 * block + np.arange(31)), (second, 16 * block + np.array([31]))):
        src, q_out = dev(qkv), dev(np.zeros(len(qkv) * d, np.uint16))
        status = w.lib.lcr_batch_norm_rope_write_kv8(
            p(q_out), ctypes.byref(view), p(src), p(src) + 2 * d, p(src) + 4 * d, None, None, 1e-5, p(dev(w.table)), 64,
            p(dev(np.zeros(len(qkv), np.int32))), p(dev(slots.astype(np.int32))), len(qkv), 1, 1, w.stride, None)
        assert status == 0, w.lib.lcr_last_error_message()
        assert (host(q_out) == qkv[:, :d].ravel()).all()
    sync()
    x = to_f32(np.concatenate([first, second]), w.kind).astype(np.float64).reshape(2, 16, 3, d)
    for which, part, blocks_of in ((0, 1, ref.to_blocks), (1, 2, ref.values_to_blocks)):
        got = np.empty(32 * d, np.uint8)
        lcr.check(w.lib, w.lib.lcr_memcpy_dtoh(got.ctypes.data, p(pools[which]) + 16 * d * block, got.size))
        got = blocks_of(got.reshape(2, -1))
        got_scales = host(scales[which], np.float32)
        rows = x[:, :, part]
        whole, begun, risen = (ref.scale_for(np.abs(r).max(), "bf16") for r in (rows[0], rows[1, :15], rows[1]))
        assert risen > begun
        assert got_scales[block] == whole and got_scales[block + 1] == risen and (got_scales[:block] == 0.25).all()
        assert (got[0] == ref.encode(rows[0] / whole)).all()
        held = ref.NUMBERS[ref.encode(rows[1, :15] / begun)]
        assert (got[1, :15] == ref.encode(held * (begun / risen))).all()
        assert (got[1, 15] == ref.encode(rows[1, 15] / risen)).all()
        # where an offset of 32 bits would lead
        head = np.empty(1 << 16, np.uint8)
        lcr.check(w.lib, w.lib.lcr_memcpy_dtoh(head.ctypes.data, p(pools[which]), head.size))
        assert (head == 0).all()
    for pool in pools:
        pool.free()
