"""What the batched entry points (include/lcr_batch.h) refuse on the host, with
their messages, and the calls that have nothing to do. No kernel is launched, so
this runs without a GPU."""

import ctypes

import pytest

A = 1 << 20  # stands for a device pointer: 16-byte aligned, never followed


@pytest.fixture(params=["bf16", "fp16"])
def lib(request, lcr):
    return lcr.load_library(request.param)


def refused(lib, status, text):
    assert status == -1, status
    message = lib.lcr_last_error_message().decode()
    assert text in message, message


def map_call(lib, **changed):
    args = dict(row_starts=A, positions=2 * A, slots=3 * A, lengths_out=4 * A, mapped_out=5 * A, counts=6 * A,
                page_tables=7 * A, lengths=8 * A, new_tokens=9 * A, mapped=10 * A, free_pages=11 * A,
                free_count=12 * A, batch=2, max_rows=8, table_stride=4, page_size=16, pool_pages=9, free_capacity=3)
    assert set(changed) <= set(args)
    args.update(changed)
    return lib.lcr_batch_map(*args.values(), None)


@pytest.mark.parametrize("changed,text", [
    (dict(batch=-1), "non-negative"), (dict(max_rows=-1), "non-negative"),
    (dict(batch=4097), "up to 4096 sequences, got 4097"), (dict(page_size=0), "positive page size, got 0"),
    (dict(page_size=-16), "positive page size"), (dict(table_stride=0), "at least one page"),
    (dict(pool_pages=-1), "non-negative page counts"), (dict(free_capacity=-1), "non-negative page counts"),
    (dict(pool_pages=1 << 27, page_size=16), "slots past 32 bits"),
    (dict(table_stride=1 << 27, page_size=16), "positions past 32 bits"),
    (dict(lengths=None), "needs its arrays"), (dict(counts=None), "needs its arrays"),
    (dict(free_count=None), "needs its arrays"), (dict(slots=None), "positions and slots"),
    (dict(free_pages=None), "has no pointer"), (dict(lengths_out=8 * A), "beside its inputs"),
    (dict(mapped_out=10 * A), "beside its inputs"), (dict(counts=12 * A), "beside its inputs"),
    (dict(free_count=6 * A + 4), "beside its inputs"),
])
def test_map_refuses(lib, changed, text):
    refused(lib, map_call(lib, **changed), text)


def test_map_of_no_sequences(lib):
    assert map_call(lib, batch=0, lengths=None) == 0


def heads_call(lcr, lib, view=None, **changed):
    v = lcr.KvView(A, 2 * A, None, 16, 16 * 2 * 64, 16 * 64, 2, 64)
    for name, value in (view or {}).items():
        setattr(v, name, value)
    args = dict(q_out=3 * A, q=4 * A, k=5 * A, v=6 * A, q_norm=7 * A, k_norm=8 * A, eps=1e-5, rope_table=9 * A,
                table_positions=64, positions=10 * A, slots=11 * A, tokens=3, num_heads=4, pool_pages=7,
                src_row_stride=512)
    assert set(changed) <= set(args)
    args.update(changed)
    values = list(args.values())
    return lib.lcr_batch_norm_rope_write_kv(values[0], ctypes.byref(v), *values[1:], None)


@pytest.mark.parametrize("view,changed,text", [
    ({}, dict(tokens=-1), "non-negative sizes"), ({}, dict(num_heads=-1), "non-negative sizes"),
    (dict(num_kv_heads=-1), {}, "non-negative sizes"), (dict(head_dim=0), {}, "positive and even"),
    (dict(head_dim=63), {}, "positive and even"), (dict(head_dim=514), {}, "up to 512"),
    (dict(page_size=0), {}, "positive page size"), ({}, dict(pool_pages=-1), "non-negative pool"),
    ({}, dict(table_positions=-1), "non-negative pool"), ({}, dict(pool_pages=1 << 28), "slots past 32 bits"),
    (dict(page_stride=-8), {}, "non-negative cache strides"), ({}, dict(src_row_stride=255), "cannot lie 255 apart"),
    ({}, dict(positions=None), "positions and slots"), ({}, dict(q=None), "its queries"),
    ({}, dict(v=None), "keys and values"), (dict(keys=None), {}, "keys and values"),
    ({}, dict(rope_table=None), "RoPE table"), ({}, dict(rope_table=9 * A + 4), "RoPE table"),
    ({}, dict(tokens=2 ** 31 - 1), "2^32 heads"),
])
def test_heads_refuses(lcr, lib, view, changed, text):
    refused(lib, heads_call(lcr, lib, view, **changed), text)


def test_heads_with_nothing_to_do(lcr, lib):
    assert heads_call(lcr, lib, tokens=0, q=None) == 0
    assert heads_call(lcr, lib, dict(num_kv_heads=0), num_heads=0) == 0
    refused(lib, lib.lcr_batch_norm_rope_write_kv(A, None, A, A, A, A, A, 1e-5, A, 4, A, A, 3, 4, 7, 512, None),
            "needs a cache view")


def attention_call(lcr, lib, view=None, **changed):
    v = lcr.KvView(A, 2 * A, 3 * A, 16, 16 * 2 * 64, 16 * 64, 2, 64)
    for name, value in (view or {}).items():
        setattr(v, name, value)
    args = dict(out=4 * A, q=5 * A, row_starts=6 * A, lengths=7 * A, batch=2, tokens=3, max_new=2, num_heads=8,
                heads_per_kv=4, table_stride=5, pool_pages=9, q_row_stride=512, scale=0.125, workspace=None,
                workspace_bytes=0)
    assert set(changed) <= set(args)
    args.update(changed)
    values = list(args.values())
    return lib.lcr_batch_attention(*values[:2], ctypes.byref(v), *values[2:], None)


@pytest.mark.parametrize("view,changed,text", [
    ({}, dict(batch=-1), "non-negative sizes"), ({}, dict(tokens=-1), "non-negative sizes"),
    ({}, dict(max_new=-1), "non-negative sizes"), ({}, dict(batch=4097), "up to 4096"),
    (dict(head_dim=0), {}, "head_dim up to 256"), (dict(head_dim=257), {}, "head_dim up to 256"),
    ({}, dict(heads_per_kv=0), "must equal num_kv_heads"), ({}, dict(heads_per_kv=3), "must equal num_kv_heads"),
    (dict(num_kv_heads=4), {}, "must equal num_kv_heads"), (dict(page_table=None), {}, "needs a page table"),
    (dict(page_size=0), {}, "positive page size"), ({}, dict(table_stride=0), "at least one page"),
    ({}, dict(pool_pages=0), "at least one page"), ({}, dict(table_stride=1 << 28), "positions past 32 bits"),
    (dict(head_stride=-8), {}, "non-negative cache strides"), ({}, dict(q_row_stride=511), "cannot lie 511"),
    ({}, dict(tokens=1 << 28), "2^31 - 1 query heads"), ({}, dict(out=None), "needs its arrays"),
    ({}, dict(lengths=None), "needs its arrays"), (dict(values=None), {}, "needs its arrays"),
    ({}, dict(workspace_bytes=64), "has no pointer"), ({}, dict(workspace=A + 8, workspace_bytes=64), "16-byte aligned"),
])
def test_attention_refuses(lcr, lib, view, changed, text):
    refused(lib, attention_call(lcr, lib, view, **changed), text)


def test_attention_with_nothing_to_do(lcr, lib):
    assert attention_call(lcr, lib, batch=0, lengths=None) == 0
    assert attention_call(lcr, lib, tokens=0, q=None) == 0
    refused(lib, lib.lcr_batch_attention(A, A, None, A, A, 1, 1, 1, 8, 4, 5, 9, 512, 0.125, None, 0, None),
            "needs a cache view")
    assert lib.lcr_batch_attention_workspace_bytes(0, 8, 1, 32, 4, 64) == 0
    assert lib.lcr_batch_attention_workspace_bytes(8, 0, 1, 32, 4, 64) == 0


def verify_call(lib, **changed):
    args = dict(out_ids=A, out_counts=2 * A, target=3 * A, draft=4 * A, draft_ids=5 * A, row_starts=6 * A,
                temperatures=7 * A, accept=8 * A, sample=9 * A, batch=2, rows=5, max_draft=3, vocab=100,
                logits_stride=100, workspace=10 * A,
                workspace_bytes=lib.lcr_batch_verify_workspace_bytes(2, 5, 100))
    assert set(changed) <= set(args)
    args.update(changed)
    return lib.lcr_batch_verify(*args.values(), None)


@pytest.mark.parametrize("changed,text", [
    (dict(batch=-1), "non-negative"), (dict(rows=-1), "non-negative"), (dict(max_draft=-1), "non-negative"),
    (dict(batch=4097), "up to 4096"), (dict(vocab=0), "empty vocabulary"), (dict(max_draft=2 ** 31 - 1), "drafts"),
    (dict(logits_stride=99), "cannot lie 99 apart"), (dict(rows=65536), "65535 rows"),
    (dict(out_ids=None), "needs its arrays"), (dict(sample=None), "needs its arrays"),
    (dict(target=None), "target's logits"), (dict(draft_ids=None), "drafted tokens"),
    (dict(accept=None), "drafted tokens"), (dict(workspace=None), "needs a workspace of"),
    (dict(workspace_bytes=64), "needs a workspace of"), (dict(workspace=10 * A + 8), "16-byte aligned"),
])
def test_verify_refuses(lib, changed, text):
    refused(lib, verify_call(lib, **changed), text)


def test_verify_of_no_sequences(lib):
    assert verify_call(lib, batch=0, temperatures=None) == 0
    assert lib.lcr_batch_verify_workspace_bytes(0, 5, 100) == 0
    assert lib.lcr_batch_verify_workspace_bytes(2, 5, 0) == 0


def test_sizes_past_a_launch(lcr, lib):
    """More than 2^32 threads: refused, by the layout that the call would use."""
    refused(lib, heads_call(lcr, lib, tokens=1 << 28), "2^32 threads")
    refused(lib, heads_call(lcr, lib, dict(head_dim=62), tokens=1 << 23), "2^32 threads")
    refused(lib, attention_call(lcr, lib, dict(head_dim=72), tokens=1 << 23, q_row_stride=576), "2^32 threads")
    refused(lib, attention_call(lcr, lib, dict(num_kv_heads=1), tokens=1 << 24, num_heads=80, heads_per_kv=80,
                                q_row_stride=5120), "2^32 threads")


def test_attention_refuses_positions_past_2_to_30(lcr, lib):
    refused(lib, attention_call(lcr, lib, table_stride=(1 << 26) + 1), "up to 2^30 positions")
