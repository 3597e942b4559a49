"""Plain 64-bit restatements of the batched operators (include/lcr_batch.h),
written from their definitions, one sequence and one row at a time."""

from __future__ import annotations

import numpy as np

# half a step of a rounding to the element type, relative to the value
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def batch_map(lengths, new_tokens, mapped, tables, free_pages, free_count, max_rows, page_size, pool_pages):
    """What lcr_batch_map writes, as a dict of int32 arrays."""
    batch, stride = tables.shape
    tables = tables.copy()
    free = [int(x) for x in free_pages[: max(0, min(int(free_count), len(free_pages)))]]
    row_starts = [0]
    positions = np.full(max_rows, -1, np.int32)
    slots = np.full(max_rows, -1, np.int32)
    lengths_out, mapped_out = lengths.copy(), mapped.copy()
    placed, open_ = 0, True
    for b in range(batch):
        length, new, have = int(lengths[b]), int(new_tokens[b]), int(mapped[b])
        start = row_starts[-1]
        if open_:
            total = length + new
            need = max(0, -(-total // page_size) - have)
            if (min(length, new, have) < 0 or total > stride * page_size or start + new > max_rows or need > len(free)):
                open_ = False
        if not open_:
            row_starts.append(start)
            continue
        for j in range(need):
            tables[b, have + j] = free.pop()
        for i in range(new):
            position = length + i
            page = int(tables[b, position // page_size])
            positions[start + i] = position
            if 0 <= page < pool_pages:
                slots[start + i] = page * page_size + position % page_size
        row_starts.append(start + new)
        lengths_out[b], mapped_out[b] = total, have + need
        placed += 1
    return {"row_starts": np.array(row_starts, np.int32), "positions": positions, "slots": slots,
            "lengths_out": lengths_out, "mapped_out": mapped_out, "tables": tables,
            "counts": np.array([placed, len(free)], np.int32)}


def rotate_heads(x, weight, eps, angles):
    """x [rows][heads][d] in 64 bits, angles [rows][d/2][2]; the result, and the
    size of the two products whose difference each element is."""
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    c, s = angles[:, None, :, 0], angles[:, None, :, 1]
    out = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    size = np.concatenate([np.abs(lo * c) + np.abs(hi * s), np.abs(hi * c) + np.abs(lo * s)], -1)
    return out, size


def attention(q, keys, values, tables, row_starts, lengths, page_size, scale, kind):
    """q [tokens][heads][d], caches [pages][kv][page][d], all 64-bit. Returns
    the rows' outputs (NaN behind the last sequence) and the error allowed.

    Counted: the probabilities' rounding (half a step each, and for fp16 half of
    the smallest subnormal, taken against a largest probability of 1), the
    output's rounding, and fp32 scores: a dot product of d terms is off by up to
    (d + 2) 2^-24 of the sum of its terms' sizes, the exponent's argument by
    2^-22 of its size, which moves each weight by that much, relatively, and the
    normaliser as well; the value sum's fp32 terms (one per key) add 2^-24 each
    of the weighted sizes, as does the weights' sum."""
    tokens, heads, d = q.shape
    kv = keys.shape[1]
    half_step = HALF_STEP[kind]
    out = np.full((tokens, heads, d), np.nan)
    allow = np.full((tokens, heads, d), np.nan)
    for b, length in enumerate(lengths):
        lo, hi = int(row_starts[b]), int(row_starts[b + 1])
        length = min(int(length), tables.shape[1] * page_size)
        at = np.arange(max(length, 0))
        pages = tables[b, at // page_size]
        k = keys[pages, :, at % page_size]
        v = values[pages, :, at % page_size]
        for row in range(lo, hi):
            seen = min(int(lengths[b]) - (hi - row) + 1, length)
            for h in range(heads):
                if seen <= 0:
                    out[row, h], allow[row, h] = 0.0, 0.0
                    continue
                kh, vh = k[:seen, h // (heads // kv)], v[:seen, h // (heads // kv)]
                s = kh @ q[row, h] * scale
                w = np.exp(s - s.max())
                total = w.sum()
                o = w @ vh / total
                mean_size = w @ np.abs(vh) / total
                score_off = (d + 2) * 2.0 ** -24 * (np.abs(kh) @ np.abs(q[row, h])).max() * scale \
                    + 2.0 ** -22 * np.abs(s).max()
                weight_off = half_step + 2 * score_off + 2 * seen * 2.0 ** -24
                tiny = (2.0 ** -25 if kind == "fp16" else 0.0) * np.abs(vh).sum(0) / total
                out[row, h] = o
                allow[row, h] = half_step * np.abs(o) + 1.01 * weight_off * mean_size + tiny + 1e-30
    return out, allow


def distribution(logits, temperature, hot=None):
    """softmax(logits / temperature) in 64 bits; where the largest is not
    finite, one at `hot`, or at that value's lowest index."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    top = x.max()
    if not np.isfinite(top):
        p = np.zeros_like(x)
        p[int(np.argmax(x == top)) if hot is None else hot] = 1.0
        return p
    with np.errstate(invalid="ignore"):
        z = np.where(x == -np.inf, -np.inf, (x - top) / np.float64(temperature))
    p = np.exp(z)
    return p / p.sum()


def verify(target, draft, draft_ids, row_starts, temperatures, accept, sample, max_draft):
    """What lcr_batch_verify writes: ids [batch][max_draft + 1] and counts."""
    batch, vocab = len(row_starts) - 1, target.shape[1]
    ids = np.full((batch, max_draft + 1), -1, np.int32)
    counts = np.zeros(batch, np.int32)
    for b in range(batch):
        first, n = int(row_starts[b]), int(row_starts[b + 1] - row_starts[b])
        if n <= 0:
            continue
        drafts = min(n - 1, max_draft)
        t = np.float32(temperatures[b])
        kept, last = 0, None
        while True:
            row = first + kept
            clean = np.where(np.isnan(target[row]), -np.inf, target[row])
            best = int(np.argmax(clean))
            if kept == drafts:
                p, last = (best if not t > 0 else distribution(target[row], t)), None
                break
            x = int(draft_ids[row])
            if not t > 0:
                if x != best:
                    p = best
                    break
                kept += 1
                continue
            p = distribution(target[row], t)
            inside = 0 <= x < vocab
            if draft is None or not np.isfinite(np.where(np.isnan(draft[row]), -np.inf, draft[row]).max()):
                q = np.zeros(vocab)
                if inside:
                    q[x] = 1.0
            else:
                q = distribution(draft[row], t)
            if not (inside and np.float64(np.float32(accept[row])) * q[x] < p[x]):
                last = q
                break
            kept += 1
        ids[b, :kept] = draft_ids[first:first + kept]
        if not t > 0:
            ids[b, kept] = p
        else:
            w = p if last is None else np.maximum(p - last, 0.0)
            if not w.sum() > 0:
                w = p
            run = np.cumsum(w)
            goal = np.float64(np.float32(sample[b])) * run[-1]
            ids[b, kept] = int(np.searchsorted(run, goal, side="right"))
        counts[b] = kept + 1
    return ids, counts
