"""What the entry points of the 8-bit cache and of log probabilities refuse on the
host, with their messages, and the calls that have nothing to do. No kernel is
launched, so this runs without a GPU."""

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


def view_of(lcr, changed):
    v = lcr.Kv8View(A, 2 * A, 3 * A, 4 * A, 5 * A, 32, 2 * 32 * 64, 32 * 64, 4, 2, 2, 64)
    for name, value in changed.items():
        assert hasattr(v, name)
        setattr(v, name, value)
    return v


def write_call(lcr, lib, view=None, **changed):
    v = view_of(lcr, view or {})
    args = dict(q_out=6 * A, q=7 * A, k=8 * A, v=9 * A, q_norm=10 * A, k_norm=11 * A, eps=1e-5, rope_table=12 * A,
                table_positions=64, positions=13 * A, slots=14 * A, tokens=3, num_heads=4, pool_pages=7,
                src_row_stride=512)
    assert set(changed) <= set(args)
    args.update(changed)
    values = list(args.values())
    return lib.lcr_batch_norm_rope_write_kv8(values[0], ctypes.byref(v), *values[1:], None)


VIEWS = [
    (dict(head_dim=0), "multiple of 16 up to 256, got 0"), (dict(head_dim=-16), "multiple of 16"),
    (dict(head_dim=72), "multiple of 16 up to 256, got 72"), (dict(head_dim=272), "multiple of 16 up to 256"),
    (dict(page_size=0), "multiple of 16 positions, got 0"), (dict(page_size=24), "multiple of 16 positions, got 24"),
    (dict(page_size=-16), "multiple of 16 positions"), (dict(page_stride=-16), "non-negative strides"),
    (dict(head_stride=-16), "non-negative strides"), (dict(scale_page_stride=-1), "non-negative strides"),
    (dict(scale_head_stride=-1), "non-negative strides"), (dict(page_stride=4104), "multiples of 16 bytes"),
    (dict(head_stride=2052), "multiples of 16 bytes"), (dict(keys=A + 8), "16-byte aligned"),
    (dict(values=2 * A + 4), "16-byte aligned"),
]


@pytest.mark.parametrize("view,changed,text", [(v, {}, t) for v, t in VIEWS] + [
    ({}, dict(tokens=-1), "non-negative sizes"), ({}, dict(num_heads=-1), "non-negative sizes"),
    (dict(num_kv_heads=-1), {}, "non-negative sizes"), ({}, dict(pool_pages=-1), "non-negative pool"),
    ({}, dict(table_positions=-1), "non-negative pool"), ({}, dict(pool_pages=1 << 27), "slots past 32 bits"),
    ({}, dict(src_row_stride=255), "cannot lie 255 apart"), ({}, dict(positions=None), "positions and slots"),
    ({}, dict(slots=None), "positions and slots"), ({}, dict(q=None), "its queries"), ({}, dict(q_out=None), "its queries"),
    ({}, dict(k=None), "a cache with scales"), ({}, dict(v=None), "a cache with scales"),
    (dict(keys=None), {}, "a cache with scales"), (dict(value_scales=None), {}, "a cache with scales"),
    (dict(key_scales=None), {}, "a cache with scales"), ({}, dict(rope_table=None), "RoPE table"),
    ({}, dict(rope_table=12 * A + 4), "RoPE table"), ({}, dict(tokens=2 ** 31 - 1), "heads in all"),
])
def test_write_refuses(lcr, lib, view, changed, text):
    refused(lib, write_call(lcr, lib, view, **changed), text)


def test_write_of_nothing(lcr, lib):
    assert write_call(lcr, lib, tokens=0) == 0
    assert write_call(lcr, lib, dict(num_kv_heads=0), num_heads=0) == 0
    assert write_call(lcr, lib, tokens=0, q=None, slots=None) == 0
    refused(lib, lib.lcr_batch_norm_rope_write_kv8(A, None, A, A, A, A, A, 1e-5, A, 1, A, A, 1, 1, 1, 64, None),
            "needs a cache view")


def attention_call(lcr, lib, view=None, **changed):
    v = view_of(lcr, view or {})
    args = dict(out=6 * A, q=7 * A, row_starts=8 * A, lengths=9 * A, batch=2, tokens=3, max_new=2, num_heads=4,
                heads_per_kv=2, table_stride=5, pool_pages=7, q_row_stride=256, scale=0.125, workspace=None,
                workspace_bytes=0)
    assert set(changed) <= set(args)
    args.update(changed)
    a = list(args.values())
    return lib.lcr_batch_attention_kv8(a[0], a[1], ctypes.byref(v), *a[2:], None)


@pytest.mark.parametrize("view,changed,text", [(v, {}, t) for v, t in VIEWS] + [
    ({}, dict(batch=-1), "non-negative sizes"), ({}, dict(tokens=-1), "non-negative sizes"),
    ({}, dict(max_new=-1), "non-negative sizes"), ({}, dict(num_heads=-4), "non-negative sizes"),
    ({}, dict(batch=4097), "up to 4096 sequences, got 4097"), ({}, dict(heads_per_kv=0), "must equal"),
    ({}, dict(heads_per_kv=4), "must equal"), ({}, dict(num_heads=5), "must equal"),
    (dict(num_kv_heads=3), {}, "must equal"), (dict(page_table=None), {}, "needs a page table"),
    ({}, dict(table_stride=0), "at least one page"), ({}, dict(pool_pages=0), "at least one page"),
    ({}, dict(table_stride=(1 << 25) + 1), "up to 2^30 positions"),
    ({}, dict(q_row_stride=255), "cannot lie 255 elements apart"), ({}, dict(tokens=(1 << 30) + 1), "up to 2^30 rows"),
    ({}, dict(tokens=1 << 29), "2^31 - 1 query heads"), ({}, dict(out=None), "needs its arrays"),
    ({}, dict(q=None), "needs its arrays"), (dict(values=None), {}, "needs its arrays"),
    (dict(key_scales=None), {}, "needs its arrays"), (dict(value_scales=None), {}, "needs its arrays"),
    ({}, dict(row_starts=None), "needs its arrays"), ({}, dict(lengths=None), "needs its arrays"),
    ({}, dict(workspace_bytes=64), "has no pointer"), ({}, dict(workspace=10 * A + 8, workspace_bytes=64), "16-byte aligned"),
    (dict(head_dim=48), dict(tokens=1 << 28), "more than 2^32 threads"),
])
def test_attention_refuses(lcr, lib, view, changed, text):
    refused(lib, attention_call(lcr, lib, view, **changed), text)


def test_attention_of_nothing(lcr, lib):
    for nothing in (dict(batch=0), dict(tokens=0), dict(num_heads=0)):
        assert attention_call(lcr, lib, q=None, out=None, **nothing) == 0
    assert lib.lcr_batch_attention_kv8(A, A, None, A, A, 1, 1, 1, 1, 1, 1, 1, 64, 0.1, None, 0, None) == -1
    for args in ((0, 1, 1, 1, 1, 64), (1, 0, 1, 1, 1, 64), (1, 1, 0, 1, 1, 64), (1, 1, 1, 0, 1, 64), (1, 1, 1, 1, 0, 64),
                 (1, 1, 1, 1, 1, 48), (-1, -1, -1, -1, -1, -1)):
        assert lib.lcr_batch_attention_kv8_workspace_bytes(*args) == 0


def logprobs_call(lib, **changed):
    args = dict(logprobs=A, ranks=2 * A, entropies=3 * A, top_ids=4 * A, top_logprobs=5 * A, logits=6 * A,
                token_ids=7 * A, rows=3, top=5, vocab=1000, logits_stride=1000, workspace=None, workspace_bytes=0)
    assert set(changed) <= set(args)
    args.update(changed)
    return lib.lcr_batch_logprobs(*args.values(), None)


@pytest.mark.parametrize("changed,text", [
    (dict(rows=-1), "non-negative sizes"), (dict(top=-1), "non-negative sizes"),
    (dict(top=33), "up to 32 alternatives, got 33"), (dict(vocab=0), "a vocabulary, got 0"),
    (dict(vocab=-5), "a vocabulary"), (dict(vocab=(1 << 30) + 1, logits_stride=2 ** 31 - 1), "up to 2^30 ids"),
    (dict(logits=6 * A + 2), "4-byte boundaries"), (dict(logits_stride=999), "cannot lie 999 apart"),
    (dict(logits=None), "needs logits"), (dict(top_ids=None), "room for its alternatives"),
    (dict(top_logprobs=None), "room for its alternatives"), (dict(token_ids=None), "needs the tokens"),
    (dict(token_ids=None, logprobs=None), "needs the tokens"), (dict(workspace_bytes=16), "has no pointer"),
    (dict(workspace=8 * A + 4, workspace_bytes=64), "16-byte aligned"), (dict(rows=2 ** 31 - 1), "2^32 threads"),
])
def test_logprobs_refuses(lib, changed, text):
    refused(lib, logprobs_call(lib, **changed), text)


def test_logprobs_of_nothing(lib):
    assert logprobs_call(lib, rows=0) == 0
    assert logprobs_call(lib, rows=0, logits=None, vocab=0) == 0
    for args in ((0, 1, 10), (-1, 1, 10), (1, -1, 10), (1, 1, 0), (1, 1, -1)):
        assert lib.lcr_batch_logprobs_workspace_bytes(*args) == 0
