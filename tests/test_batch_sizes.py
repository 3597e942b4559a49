"""Sizes of the batched entries at the end of what 32 bits count."""

import ctypes

import numpy as np
import pytest

from test_batch_refusals import lib, refused, verify_call  # noqa: F401  (a fixture)


def test_verify_refuses_drafts_past_2_to_30(lib):  # noqa: F811
    refused(lib, verify_call(lib, max_draft=(1 << 30) + 1), "up to 2^30 drafts")
    refused(lib, verify_call(lib, max_draft=2 ** 31 - 2), "up to 2^30 drafts, got 2147483646")


@pytest.mark.gpu
def test_map_of_nearly_2_to_31_pages(lcr, gpu):
    """Pages of one position: 4096 sequences whose tables lack all of theirs."""
    from helpers import dev, host, p
    batch, stride = 4096, 1 << 19
    lengths = np.full(batch, stride, np.int32)
    lengths[-1] -= 1000
    total = int(lengths.sum(dtype=np.int64))
    assert total == 2 ** 31 - 1000
    free = lcr.DeviceBuffer(4 * total, zero=True)
    ends = np.array([7, 5], np.int32)  # the first and the last page of the list
    for at, value in ((0, ends[:1]), (total - 1, ends[1:])):
        lcr.check(gpu, gpu.lcr_memcpy_htod(free.ptr + 4 * at, value.ctypes.data, 4))
    tables = lcr.DeviceBuffer(4 * batch * stride, zero=False)
    lcr.check(gpu, gpu.lcr_device_memset(tables.ptr, 0xff, tables.nbytes))
    zeros = dev(np.zeros(batch, np.int32))
    outs = [dev(np.zeros(n, np.int32)) for n in (batch + 1, 131072, 131072, batch, batch, 2)]
    status = gpu.lcr_batch_map(*[p(o) for o in outs], tables.ptr, p(dev(lengths)), p(zeros), p(zeros), free.ptr,
                               p(dev(np.array([total], np.int32))), batch, 131072, stride, 1, 8, total, None)
    assert status == 0, gpu.lcr_last_error_message()
    assert host(outs[5], np.int32).tolist() == [batch, 0]
    assert (host(outs[4], np.int32) == lengths).all()
    got = np.zeros(2000, np.int32)

    def read(at, n):
        lcr.check(gpu, gpu.lcr_memcpy_dtoh(got.ctypes.data, ctypes.c_void_p(tables.ptr + 4 * at), 4 * n))
        return got[:n].tolist()

    assert read(0, 3) == [5, 0, 0]
    assert read(2 ** 30, 3) == [0, 0, 0]
    assert read(total - 3, 1003) == [0, 0, 7] + [-1] * 1000
    free.free()
    tables.free()
