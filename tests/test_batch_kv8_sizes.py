"""Calls of the 8-bit cache's attention whose launch would have more than 2^32 threads:
refused on the host, whichever of its kernels takes them."""

import pytest

from test_batch_kv8_refusals import attention_call, lib, refused  # noqa: F401  (a fixture)


@pytest.mark.parametrize("d,kv,max_new", [
    # a block of 512 threads a sequence and head, 4096 of 2048 heads and more
    (64, 2048, 1), (64, 2048, 16), (128, 2048, 1), (128, 2048, 33),
    # of 256 threads
    (64, 4096, 17), (64, 4096, 33), (128, 4096, 17),
])
def test_attention_refuses_more_than_2_to_32_threads(lcr, lib, d, kv, max_new):  # noqa: F811
    view = dict(num_kv_heads=kv, head_dim=d, page_stride=0, head_stride=0)
    refused(lib, attention_call(lcr, lib, view, batch=4096, tokens=4096, max_new=max_new, num_heads=kv, heads_per_kv=1,
                                q_row_stride=kv * d), "needs more than 2^32 threads")
