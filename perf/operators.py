"""One step of serving many requests over a paged cache, operator by operator.

  map     block tables, row positions and cache slots from the requests' lengths
  heads   per-head norm of queries and keys, rotation, and the cache write by slot
  attend  attention of each request's new tokens over its pages
  verify  drafted tokens against the target's distribution, from given draws

Head layouts, vocabulary and page size are those of this repository's
configuration (32 query heads of 64 on 8, or 16 of 128 on 8; 128256 ids; pages
of 16) and variations of them. A request's lengths follow from its case alone;
its contents from the seed.
"""

import importlib
import math
import random

import torch

own = False

DEVICE = "cuda:0"
ELEM = {"bf16": torch.bfloat16, "fp16": torch.float16}
VOCAB = 128256
EPS = 1e-5
ROPE_THETA = 500000.0


def listed():
    return [
        # one token each for a handful of chats: the smallest step, all latency
        {"name": "map_decode_8", "kind": "map", "batch": 8, "chunks": 0, "new": 1, "context": 900, "page": 16},
        # a busy server's step of verified drafts with some prompts among them
        {"name": "map_mixed_256", "kind": "map", "batch": 256, "chunks": 40, "new": 129, "context": 8000, "page": 16},
        # many prompts admitted at once
        {"name": "map_prompts_1024", "kind": "map", "batch": 1024, "chunks": 1024, "new": 60, "context": 0, "page": 32},

        # the same handful of chats
        {"name": "heads_decode_8", "kind": "heads", "batch": 8, "chunks": 0, "new": 1, "context": 900, "page": 16,
         "heads": 32, "kv_heads": 8, "head_dim": 64, "norm": True, "dtype": "bf16"},
        # four drafts and a token for each of 64 requests, wide heads, fp16
        {"name": "heads_drafts_64_fp16", "kind": "heads", "batch": 64, "chunks": 64, "new": 5, "context": 3000,
         "page": 16, "heads": 16, "kv_heads": 8, "head_dim": 128, "norm": True, "dtype": "fp16"},
        # prompts of several requests in one pass, as many rows as fit a step
        {"name": "heads_prompts", "kind": "heads", "batch": 11, "chunks": 11, "new": 800, "context": 500, "page": 16,
         "heads": 32, "kv_heads": 8, "head_dim": 64, "norm": True, "dtype": "bf16"},

        # two chats, one token each: latency
        {"name": "attend_decode_2", "kind": "attend", "batch": 2, "chunks": 0, "new": 1, "context": 300, "page": 16,
         "heads": 32, "kv_heads": 8, "head_dim": 64, "dtype": "bf16"},
        # a full server's decode step: the cache's bytes
        {"name": "attend_decode_64", "kind": "attend", "batch": 64, "chunks": 0, "new": 1, "context": 8000,
         "page": 16, "heads": 32, "kv_heads": 8, "head_dim": 64, "dtype": "bf16"},
        # verified drafts over long documents, wide heads, fp16
        {"name": "attend_drafts_24_fp16", "kind": "attend", "batch": 24, "chunks": 24, "new": 5, "context": 5000,
         "page": 16, "heads": 16, "kv_heads": 8, "head_dim": 128, "dtype": "fp16"},
        # chunks of two long prompts beside the running requests' tokens
        {"name": "attend_mixed_18", "kind": "attend", "batch": 18, "chunks": 2, "new": 1000, "context": 4000,
         "page": 16, "heads": 32, "kv_heads": 8, "head_dim": 64, "dtype": "bf16"},

        # one request's drafts: latency
        {"name": "verify_1", "kind": "verify", "batch": 1, "draft": 4, "vocab": VOCAB, "model_draft": True},
        # a full server's drafts
        {"name": "verify_64", "kind": "verify", "batch": 64, "draft": 4, "vocab": VOCAB, "model_draft": True},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["map", "heads", "attend", "attend", "verify"])
    page = rng.choice([8, 16, 16, 32, 64])
    if kind == "map":
        batch = _spread(rng, 1, 1024)
        return {"kind": kind, "batch": batch, "chunks": rng.randint(0, batch), "new": _spread(rng, 1, 60),
                "context": rng.choice([0, _spread(rng, 16, 8000)]), "page": page}
    if kind == "verify":
        batch = _spread(rng, 1, 64)
        return {"kind": kind, "batch": batch, "draft": rng.randint(1, 4),
                "vocab": rng.choice([VOCAB, _spread(rng, 1000, VOCAB)]), "model_draft": rng.random() < 0.7}
    head_dim = rng.choice([64, 64, 128])
    kv_heads = rng.choice([8, 8, 4, 2])
    case = {"kind": kind, "page": page, "heads": kv_heads * rng.choice([1, 2, 4, 4, 8] if head_dim == 64 else [1, 2, 4]),
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind == "heads":
        batch = _spread(rng, 1, 64)
        tokens = 24576000 // ((case["heads"] + 2 * kv_heads) * head_dim)  # as many values as the listed prompts
        case.update(batch=batch, chunks=rng.randint(0, batch), new=_spread(rng, 1, max(2, min(8000, tokens) // batch)),
                    context=rng.choice([0, _spread(rng, 16, 8000)]), norm=rng.random() < 0.7)
        return case
    shape = rng.choice(["tokens", "drafts", "mixed"])
    if shape == "tokens":
        batch = _spread(rng, 1, 64)
        positions = 300000 * 64 * 8 // (head_dim * kv_heads)
        case.update(batch=batch, chunks=0, new=1, context=_spread(rng, 16, min(100000, positions // batch)))
    elif shape == "drafts":
        batch = _spread(rng, 1, 32)
        case.update(batch=batch, chunks=batch, new=rng.randint(2, 9), context=_spread(rng, 16, min(30000, 160000 // batch)))
    else:
        batch = _spread(rng, 1, 16)
        new = _spread(rng, 16, 1000 * 2048 // max(2048, case["heads"] * head_dim))
        case.update(batch=batch, chunks=rng.randint(1, min(batch, 2)), new=new,
                    context=rng.choice([0, _spread(rng, 16, 4000)]))
    return case


# ---------------------------------------------------------------------------
# inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(gen, shape, std, dtype):
    return (torch.randn(shape, device=DEVICE, generator=gen) * std).to(ELEM[dtype])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _lengths(case):
    """Per request: positions already cached, and new tokens. `chunks` of them
    have up to `new` tokens, the first exactly that many; the rest have one."""
    rng = random.Random("%(batch)d %(chunks)d %(new)d %(context)d" % case)
    past = [rng.randint((case["context"] + 1) // 3, case["context"]) for _ in range(case["batch"])]
    new = [rng.randint((case["new"] + 1) // 2, case["new"]) for _ in range(case["chunks"])]
    new[:1] = [case["new"]] * min(1, case["chunks"])
    new += [1] * (case["batch"] - case["chunks"])
    order = list(range(case["batch"]))
    rng.shuffle(order)
    return [past[i] for i in order], [new[i] for i in order]


def _rows(case):
    """Rows of the step's buffers: the requests' tokens, and room behind them
    as a captured step keeps it."""
    return -(-sum(_lengths(case)[1]) // 8) * 8


def _pages_for(case, count):
    return -(-count // case["page"])


def _starts(new):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return starts


def _tables(gen, case):
    """Page tables of the requests, past and new positions mapped, pages in
    random order; the pool holds an eighth more. Unused entries are -1."""
    past, new = _lengths(case)
    need = [_pages_for(case, p + n) for p, n in zip(past, new)]
    total, width = sum(need), max(need)
    pool = total + total // 8 + 1
    pages = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
    need_t, first = _ints(need), _ints(_starts(need)[:-1])
    column = torch.arange(width, device=DEVICE, dtype=torch.int32)
    at = (first[:, None] + column).clamp(max=total - 1).long()
    return torch.where(column < need_t[:, None], pages[at], -1).contiguous(), pool


def _prepare_map(case, seed):
    gen = _generator(seed)
    past, new = _lengths(case)
    page, batch, rows = case["page"], case["batch"], _rows(case)
    mapped = [_pages_for(case, p) for p in past]
    # tables as wide as the longest request a server of this kind takes
    width = _pages_for(case, max(8192, max(p + n for p, n in zip(past, new))))
    needed = sum(_pages_for(case, p + n) - m for p, n, m in zip(past, new, mapped))
    held, spare = sum(mapped), max(4, needed // 8)
    pool = held + needed + spare
    pages = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
    column = torch.arange(width, device=DEVICE, dtype=torch.int32)
    at = (_ints(_starts(mapped)[:-1])[:, None] + column).clamp(max=max(held - 1, 0)).long()
    i32 = {"device": DEVICE, "dtype": torch.int32}
    return {
        "tables": torch.where(column < _ints(mapped)[:, None], pages[at], -1).contiguous(),
        "lengths": _ints(past), "new": _ints(new), "mapped": _ints(mapped),
        "free": pages[held:].contiguous(), "free_count": _ints([needed + spare]),
        "pool": pool, "rows": rows,
        "row_starts": torch.empty(batch + 1, **i32), "positions": torch.empty(rows, **i32),
        "slots": torch.empty(rows, **i32), "lengths_out": torch.empty(batch, **i32),
        "mapped_out": torch.empty(batch, **i32), "counts": torch.empty(2, **i32),
    }


def _rope_table(positions, head_dim):
    """[positions][head_dim / 2][cos, sin]"""
    freq = ROPE_THETA ** (-torch.arange(0, head_dim, 2, device=DEVICE, dtype=torch.float64) / head_dim)
    angle = torch.arange(positions, device=DEVICE, dtype=torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def _row_places(case, tables):
    """position and slot of every row, -1 behind the last."""
    past, new = _lengths(case)
    rows, starts = _rows(case), _ints(_starts(new))
    row = torch.arange(rows, device=DEVICE, dtype=torch.int32)
    seq = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=len(new) - 1)
    position = _ints(past)[seq] + row - starts[seq]
    inside = row < starts[-1]
    column = (position // case["page"]).clamp(max=tables.shape[1] - 1).long()
    slot = tables[seq, column] * case["page"] + position % case["page"]
    return torch.where(inside, position, -1).contiguous(), torch.where(inside, slot, -1).contiguous()


def _prepare_heads(case, seed):
    gen = _generator(seed)
    H, K, d, page, dtype = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["dtype"]
    rows = _rows(case)
    tables, pool = _tables(gen, case)
    positions, slots = _row_places(case, tables)
    past, new = _lengths(case)
    limit = max(p + n for p, n in zip(past, new))
    qkv = _normal(gen, (rows, (H + 2 * K) * d), 1.0, dtype)
    weight = lambda: (1.0 + 0.2 * torch.randn(d, device=DEVICE, generator=gen)).to(ELEM[dtype])  # noqa: E731
    return {
        "qkv": qkv, "q": qkv[:, : H * d], "k": qkv[:, H * d : (H + K) * d], "v": qkv[:, (H + K) * d :],
        "q_norm": weight() if case["norm"] else None, "k_norm": weight() if case["norm"] else None,
        "rope": _rope_table(limit, d), "positions": positions, "slots": slots, "pool": pool, "rows": rows,
        "keys": torch.zeros(pool, K, page, d, device=DEVICE, dtype=ELEM[dtype]),
        "values": torch.zeros(pool, K, page, d, device=DEVICE, dtype=ELEM[dtype]),
        "q_out": torch.zeros(rows, H, d, device=DEVICE, dtype=ELEM[dtype]),
    }


def _prepare_attend(case, seed):
    gen = _generator(seed)
    H, K, d, page, dtype = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["dtype"]
    rows = _rows(case)
    tables, pool = _tables(gen, case)
    past, new = _lengths(case)
    state = {
        "q": _normal(gen, (rows, H, d), 1.5, dtype), "tables": tables, "pool": pool, "rows": rows,
        "keys": _normal(gen, (pool, K, page, d), 1.5, dtype), "values": _normal(gen, (pool, K, page, d), 1.0, dtype),
        "row_starts": _ints(_starts(new)), "lengths": _ints([p + n for p, n in zip(past, new)]), "max_new": max(new),
        "out": torch.zeros(rows, H, d, device=DEVICE, dtype=ELEM[dtype]), "workspace": None,
    }
    return state


def _drafts(case):
    """Drafted tokens of each request; the first has as many as any."""
    rng = random.Random("%(batch)d %(draft)d %(vocab)d" % case)
    return [case["draft"]] + [rng.randint(0, case["draft"]) for _ in range(case["batch"] - 1)]


def _temperatures(case):
    """Every fourth request asks for the likeliest token, the first samples."""
    return [(0.0 if b % 4 == 3 else 0.6 + 0.1 * (b % 6)) for b in range(case["batch"])]


def _prepare_verify(case, seed):
    gen = _generator(seed)
    drafts, V = _drafts(case), case["vocab"]
    starts = _starts([d + 1 for d in drafts])
    rows = starts[-1]
    target = 2.5 * torch.randn(rows, V, device=DEVICE, generator=gen)
    draft = target + 0.4 * torch.randn(rows, V, device=DEVICE, generator=gen)
    seq = torch.repeat_interleave(torch.arange(case["batch"], device=DEVICE), _ints([d + 1 for d in drafts]))
    heat = torch.tensor(_temperatures(case), device=DEVICE)[seq]
    noise = -torch.log(-torch.log(torch.rand(rows, V, device=DEVICE, generator=gen).clamp(1e-9, 1 - 1e-7)))
    ids = (draft + heat[:, None] * noise).argmax(-1).to(torch.int32)
    del noise
    if not case["model_draft"]:
        draft = None  # tokens copied from the text: no distribution behind them
    i32 = {"device": DEVICE, "dtype": torch.int32}
    return {
        "target": target, "draft": draft, "ids": ids, "row_starts": _ints(starts),
        "temperatures": torch.tensor(_temperatures(case), device=DEVICE),
        "accept": torch.rand(rows, device=DEVICE, generator=gen),
        "sample": torch.rand(case["batch"], device=DEVICE, generator=gen), "rows": rows,
        "out_ids": torch.empty(case["batch"], case["draft"] + 1, **i32),
        "out_counts": torch.empty(case["batch"], **i32), "workspace": None,
    }


def prepare(case, seed):
    state = {"map": _prepare_map, "heads": _prepare_heads, "attend": _prepare_attend,
             "verify": _prepare_verify}[case["kind"]](case, seed)
    state["case"] = dict(case)
    return state


# ---------------------------------------------------------------------------
# one pass through the framework


def _library(case):
    lcr = importlib.import_module("llama-cuda-runtime_amd")
    return lcr, lcr.load_library(case.get("dtype", "bf16"))


def _view(lcr, s):
    if "view" not in s:
        v = lcr.KvView()
        pool, K, page, d = s["keys"].shape
        v.keys, v.values = s["keys"].data_ptr(), s["values"].data_ptr()
        v.page_table = s["tables"].data_ptr() if "tables" in s else None
        v.page_size, v.page_stride, v.head_stride = page, K * page * d, page * d
        v.num_kv_heads, v.head_dim = K, d
        s["view"] = v
    return s["view"]


def _workspace(s, size):
    """A program's own workspace, kept from call to call."""
    if s["workspace"] is None:
        s["workspace"] = torch.empty(max(size, 16), device=DEVICE, dtype=torch.uint8)
    return s["workspace"].data_ptr(), s["workspace"].numel()


def _own_map(lcr, lib, s, c, stream):
    p = torch.Tensor.data_ptr
    lcr.check(lib, lib.lcr_batch_map(
        p(s["row_starts"]), p(s["positions"]), p(s["slots"]), p(s["lengths_out"]), p(s["mapped_out"]), p(s["counts"]),
        p(s["tables"]), p(s["lengths"]), p(s["new"]), p(s["mapped"]), p(s["free"]), p(s["free_count"]), c["batch"],
        s["rows"], s["tables"].shape[1], c["page"], s["pool"], s["free"].numel(), stream), "batch_map")
    return {k: s[k] for k in ("row_starts", "positions", "slots", "lengths_out", "mapped_out", "counts", "tables")}


def _own_heads(lcr, lib, s, c, stream):
    p = torch.Tensor.data_ptr
    norms = (p(s["q_norm"]), p(s["k_norm"])) if c["norm"] else (None, None)
    lcr.check(lib, lib.lcr_batch_norm_rope_write_kv(
        p(s["q_out"]), _view(lcr, s), p(s["q"]), p(s["k"]), p(s["v"]), *norms, EPS, p(s["rope"]), s["rope"].shape[0],
        p(s["positions"]), p(s["slots"]), s["rows"], c["heads"], s["pool"], s["qkv"].stride(0), stream),
        "batch_norm_rope_write_kv")
    return {"q": s["q_out"], "keys": s["keys"], "values": s["values"]}


def _own_attend(lcr, lib, s, c, stream):
    p = torch.Tensor.data_ptr
    group = c["heads"] // c["kv_heads"]
    if s["workspace"] is None:
        _workspace(s, lib.lcr_batch_attention_workspace_bytes(c["batch"], s["rows"], s["max_new"], c["heads"], group,
                                                              c["head_dim"]))
    lcr.check(lib, lib.lcr_batch_attention(
        p(s["out"]), p(s["q"]), _view(lcr, s), p(s["row_starts"]), p(s["lengths"]), c["batch"], s["rows"],
        s["max_new"], c["heads"], group, s["tables"].shape[1], s["pool"], s["q"].stride(0), c["head_dim"] ** -0.5,
        *_workspace(s, 0), stream), "batch_attention")
    return s["out"]


def _own_verify(lcr, lib, s, c, stream):
    p = torch.Tensor.data_ptr
    if s["workspace"] is None:
        _workspace(s, lib.lcr_batch_verify_workspace_bytes(c["batch"], s["rows"], c["vocab"]))
    lcr.check(lib, lib.lcr_batch_verify(
        p(s["out_ids"]), p(s["out_counts"]), p(s["target"]), p(s["draft"]) if c["model_draft"] else None, p(s["ids"]),
        p(s["row_starts"]), p(s["temperatures"]), p(s["accept"]), p(s["sample"]), c["batch"], s["rows"], c["draft"],
        c["vocab"], s["target"].stride(0), *_workspace(s, 0), stream), "batch_verify")
    return {"ids": s["out_ids"], "counts": s["out_counts"]}


# ---------------------------------------------------------------------------
# one pass in plain operations


def _plain_map(s, c):
    page, batch, rows = c["page"], c["batch"], s["rows"]
    past, new, mapped, tables = s["lengths"], s["new"], s["mapped"], s["tables"]
    total = past + new
    need = (-(-total // page) - mapped).clamp(min=0)
    free = s["free_count"].clamp(max=s["free"].numel())
    fits = (new >= 0) & (past >= 0) & (total <= tables.shape[1] * page)
    fits &= (need.cumsum(0) <= free) & (new.cumsum(0) <= rows)
    placed = fits.int().cumprod(0).bool()
    zero = torch.zeros(1, device=DEVICE, dtype=torch.int32)
    given = torch.where(placed, new, 0)
    pages = torch.where(placed, need, 0)
    starts = torch.cat([zero, given.cumsum(0).int()])
    first = pages.cumsum(0).int() - pages
    # new entries come off the free list's end, in the requests' order
    column = torch.arange(tables.shape[1], device=DEVICE, dtype=torch.int32)
    rank = first[:, None] + column - mapped[:, None]
    fresh = (column >= mapped[:, None]) & (column < (mapped + pages)[:, None])
    tables = torch.where(fresh, s["free"][(free - 1 - rank).clamp(0, s["free"].numel() - 1).long()], tables)
    row = torch.arange(rows, device=DEVICE, dtype=torch.int32)
    seq = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=batch - 1)
    inside = row < starts[-1]
    position = past[seq] + row - starts[seq]
    at = (position // page).clamp(max=tables.shape[1] - 1).long()
    slot = tables[seq, at] * page + position % page
    return {
        "row_starts": starts, "positions": torch.where(inside, position, -1), "slots": torch.where(inside, slot, -1),
        "lengths_out": torch.where(placed, total, past), "mapped_out": mapped + pages,
        "counts": torch.cat([placed.sum().int()[None], free - pages.sum().int()]), "tables": tables,
    }


def _plain_rotate(x, weight, c, cos, sin):
    """[rows][heads][d] in 32 bits: norm over d, then the half-split rotation."""
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain_heads(s, c):
    H, K, d, page, elem = c["heads"], c["kv_heads"], c["head_dim"], c["page"], ELEM[c["dtype"]]
    rows, inside = s["rows"], s["slots"] >= 0
    cs = s["rope"][s["positions"].clamp(min=0).long()]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    q = _plain_rotate(s["q"].reshape(rows, H, d).float(), s["q_norm"], c, cos, sin).to(elem)
    k = _plain_rotate(s["k"].reshape(rows, K, d).float(), s["k_norm"], c, cos, sin).to(elem)
    slot = torch.where(inside, s["slots"], 0).long()
    # rows without a slot go to one row behind the pool
    at = torch.where(inside, slot // page, s["pool"])
    pools = []
    for pool, new in ((s["keys"], k), (s["values"], s["v"].reshape(rows, K, d))):
        wide = torch.cat([pool, pool[:1]])
        wide[at, :, slot % page] = new
        pools.append(wide[:-1])
    return {"q": torch.where(inside[:, None, None], q, s["q_out"]), "keys": pools[0], "values": pools[1]}


def _plain_attend(s, c):
    H, K, d, page, batch = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["batch"]
    group, rows, longest = H // K, s["rows"], s["max_new"]
    starts, lengths, tables = s["row_starts"], s["lengths"], s["tables"]
    new = starts[1:] - starts[:-1]
    span = tables.shape[1] * page
    pages = tables.clamp(min=0).long()
    gather = lambda pool: pool[pages].permute(0, 2, 1, 3, 4).reshape(batch, K, span, d).float()  # noqa: E731
    step = torch.arange(longest, device=DEVICE)
    row = (starts[:-1, None] + step).clamp(max=rows - 1).long()
    q = s["q"][row].float().reshape(batch, longest, K, group, d).permute(0, 2, 1, 3, 4).reshape(batch, K, -1, d)
    scores = torch.matmul(q, gather(s["keys"]).transpose(-1, -2).contiguous()) * d ** -0.5
    position = (lengths - new)[:, None] + step
    seen = torch.arange(span, device=DEVICE) <= position[:, :, None]
    scores = scores.reshape(batch, K, longest, group, span).masked_fill_(~seen[:, None, :, None], -math.inf)
    weights = torch.softmax(scores, -1).reshape(batch, K, -1, span)
    del scores
    out = torch.matmul(weights, gather(s["values"])).reshape(batch, K, longest, group, d)
    out = out.permute(0, 2, 1, 3, 4).reshape(batch, longest, H, d).to(s["out"].dtype)
    every = torch.arange(rows, device=DEVICE, dtype=torch.int32)
    seq = (torch.searchsorted(starts, every, right=True) - 1).clamp(max=batch - 1)
    inside = every < starts[-1]
    picked = out[seq, (every - starts[seq]).clamp(0, longest - 1).long()]
    return torch.where(inside[:, None, None], picked, s["out"])


def _plain_first(logits):
    """The lowest index of the largest value of each row."""
    at = torch.arange(logits.shape[-1], device=DEVICE)
    return torch.where(logits == logits.amax(-1, keepdim=True), at, logits.shape[-1]).amin(-1)


def _plain_verify(s, c):
    # 64 bits: which id a draw falls on hangs on intervals of the running sum
    # that are 1e-5 wide or less
    batch, D, rows = c["batch"], c["draft"], s["rows"]
    starts, target = s["row_starts"], s["target"]
    row = torch.arange(rows, device=DEVICE, dtype=torch.int32)
    seq = torch.searchsorted(starts, row, right=True) - 1
    heat = s["temperatures"].double()[seq]
    greedy = heat <= 0
    heat = torch.where(greedy, 1.0, heat)[:, None]
    p = torch.softmax(target.double() / heat, -1)
    x = s["ids"].long()[:, None]
    p_x = p.gather(1, x)[:, 0]
    if s["draft"] is not None:
        q = torch.softmax(s["draft"].double() / heat, -1)
    else:
        q = torch.zeros_like(p).scatter_(1, x, 1.0)
    best = _plain_first(target)
    taken = torch.where(greedy, best == x[:, 0], s["accept"].double() * q.gather(1, x)[:, 0] < p_x)
    count = starts[1:] - starts[:-1] - 1
    step = torch.arange(D + 1, device=DEVICE)
    at = (starts[:-1, None] + step).clamp(max=rows - 1).long()
    drafted = step < count[:, None]
    kept = (taken[at] & drafted).int().cumprod(1).sum(1)
    last = starts[:-1].long() + kept
    rest = p[last]
    left = (rest - q[last]).clamp(min=0)
    left = torch.where((kept < count)[:, None] & (left.sum(-1, keepdim=True) > 0), left, rest)
    run_up = left.cumsum(-1)
    goal = s["sample"].double()[:, None] * run_up[:, -1:]
    drawn = (run_up <= goal).sum(-1).clamp(max=c["vocab"] - 1)
    final = torch.where(s["temperatures"] <= 0, best[last], drawn)
    ids = torch.where(step < kept[:, None], s["ids"].long()[at], torch.where(step == kept[:, None], final[:, None], -1))
    return {"ids": ids.int(), "counts": (kept + 1).int()}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        lcr, lib = _library(case)
        stream = torch.cuda.current_stream().cuda_stream
        return {"map": _own_map, "heads": _own_heads, "attend": _own_attend, "verify": _own_verify}[kind](
            lcr, lib, state, case, stream)
    return {"map": _plain_map, "heads": _plain_heads, "attend": _plain_attend, "verify": _plain_verify}[kind](
        state, case)


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits


def _exact_heads(s, c):
    H, K, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    qkv, half = s["qkv"].double(), d // 2
    keys, values, q_out = s["keys"].double(), s["values"].double(), s["q_out"].double()
    live = torch.nonzero(s["slots"] >= 0)[:, 0]
    slot, position = s["slots"][live].long(), s["positions"][live].long()
    table = s["rope"].double()[position]
    for h in range(H + 2 * K):
        x = qkv[live, h * d : (h + 1) * d]
        if h >= H + K:
            values[slot // page, h - H - K, slot % page] = x
            continue
        w = s["q_norm"] if h < H else s["k_norm"]
        if w is not None:
            x = x / torch.sqrt((x * x).sum(1, keepdim=True) / d + EPS) * w.double()
        turned = torch.empty_like(x)
        turned[:, :half] = x[:, :half] * table[:, :, 0] - x[:, half:] * table[:, :, 1]
        turned[:, half:] = x[:, half:] * table[:, :, 0] + x[:, :half] * table[:, :, 1]
        if h < H:
            q_out[live, h] = turned
        else:
            keys[slot // page, h - H, slot % page] = turned
    return {"q": q_out, "keys": keys, "values": values}


def _exact_attend(s, c):
    H, K, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    out = s["out"].double()
    starts, lengths = s["row_starts"].tolist(), s["lengths"].tolist()
    for b, length in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        pages = s["tables"][b, : -(-length // page)].long()
        last = torch.arange(length - (hi - lo), length, device=DEVICE)
        hidden = torch.arange(length, device=DEVICE) > last[:, None]
        for k in range(K):
            keys = s["keys"][pages, k].reshape(-1, d)[:length].double()
            values = s["values"][pages, k].reshape(-1, d)[:length].double()
            for h in range(k * (H // K), (k + 1) * (H // K)):
                x = (s["q"][lo:hi, h].double() @ keys.t()) / math.sqrt(d)
                x = torch.exp(x.masked_fill(hidden, -math.inf) - x.masked_fill(hidden, -math.inf).amax(1, keepdim=True))
                out[lo:hi, h] = (x @ values) / x.sum(1, keepdim=True)
    return out


def exact(case, seed):
    if case["kind"] == "heads":
        return _exact_heads(prepare(case, seed), case)
    if case["kind"] == "attend":
        return _exact_attend(prepare(case, seed), case)
    return None  # whole numbers


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    kind, e = case["kind"], 2
    if kind == "verify":
        drafts = _drafts(case)
        rows = sum(drafts) + len(drafts)
        values = case["vocab"] * (rows + (sum(drafts) if case["model_draft"] else 0))
        return {"bytes": 4 * values + 8 * rows, "flops": 4.0 * values}
    past, new = _lengths(case)
    tokens = sum(new)
    if kind == "map":
        fresh = sum(_pages_for(case, p + n) - _pages_for(case, p) for p, n in zip(past, new))
        return {"bytes": 4 * (6 * case["batch"] + 2 * fresh + 2 * _rows(case)), "flops": 4.0 * tokens}
    H, K, d = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "heads":
        return {"bytes": tokens * (2 * e * (H + 2 * K) * d + 4 * d + 8), "flops": 8.0 * tokens * (H + K) * d}
    seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
    cached = sum(p + n for p, n in zip(past, new))
    return {"bytes": 2 * e * K * d * cached + 2 * e * tokens * H * d, "flops": 4.0 * H * d * seen}
