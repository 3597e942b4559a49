"""Plain restatements of the 8-bit cache (include/lcr_batch.h): its numbers, its
layout, and what appending to it leaves, one block and one number at a time."""

from __future__ import annotations

import numpy as np

BLOCK = 16
LEAST = {"bf16": 2.0 ** -117, "fp16": 2.0 ** -15}
LARGEST = {"bf16": 1.875 * 2.0 ** 127, "fp16": 61440.0}
NAN = 0x7F


def _number(code):
    sign = -1.0 if code & 0x80 else 1.0
    exponent, mantissa = (code >> 3) & 15, code & 7
    if exponent == 15 and mantissa == 7:
        return np.nan
    return sign * (mantissa * 2.0 ** -9 if exponent == 0 else (1 + mantissa / 8) * 2.0 ** (exponent - 7))


NUMBERS = np.array([_number(c) for c in range(256)])
_POSITIVE = NUMBERS[:127]


def encode(x):
    """The nearest numbers, ties to the even mantissa; NaN for what is not finite."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    finite = np.isfinite(a)
    assert (a[finite] <= 448).all()
    with np.errstate(divide="ignore"):
        exponent = np.maximum(np.floor(np.log2(np.where(finite & (a > 0), a, 1.0))), -6)
    step = 2.0 ** (exponent - 3)
    near = np.rint(np.where(finite, a, 0) / step) * step
    code = np.searchsorted(_POSITIVE, near).astype(np.uint8)
    assert (_POSITIVE[code] == near).all()
    return np.where(finite, code | (np.signbit(x).astype(np.uint8) << 7), NAN).astype(np.uint8)


def scale_for(largest, variant):
    """The least power of two with which `largest` is at most 448."""
    s = LEAST[variant]
    while largest > 448 * s:
        s *= 2
    return s


def clamp(x, variant):
    with np.errstate(over="ignore", invalid="ignore"):
        x = np.asarray(x).astype(np.float32).astype(np.float64)
        return np.where(np.isfinite(x), np.clip(x, -LARGEST[variant], LARGEST[variant]), np.nan)


def to_blocks(numbers):
    """Keys' bytes [..., 16 d] of blocks as [..., 16, d]."""
    return numbers.reshape(*numbers.shape[:-1], BLOCK, -1)


def values_to_blocks(numbers):
    """Values' bytes [..., 16 d] as [..., 16, d]: four positions lie side by side."""
    x = numbers.reshape(*numbers.shape[:-1], 4, -1, 4)
    return np.swapaxes(x, -1, -2).reshape(*numbers.shape[:-1], BLOCK, -1)


def values_from_blocks(blocks):
    d = blocks.shape[-1]
    x = blocks.reshape(*blocks.shape[:-2], 4, 4, d)
    return np.swapaxes(x, -1, -2).reshape(*blocks.shape[:-2], BLOCK * d)


def append(block, scale, new, variant):
    """A head's block [16][d] of codes and its scale after positions new = {t: row}
    (in 64 bits) were written. Returns the scale, the codes of the positions not
    written, and the rows as they are to be held, clamped and over the scale."""
    rows = {t: clamp(x, variant) for t, x in new.items()}
    largest = max(np.abs(np.where(np.isnan(x), 0, x)).max() for x in rows.values())
    need = scale_for(largest, variant)
    after = need if 0 in new else max(need, float(scale))
    kept = block.copy()
    if 0 not in new and after > scale:
        others = [t for t in range(BLOCK) if t not in new]
        kept[others] = encode(NUMBERS[block[others]] * (float(scale) / after))
    return after, kept, {t: x / after for t, x in rows.items()}


class Cache8:
    """Host arrays of a paged 8-bit cache with any strides; every byte and scale
    that no page covers holds a mark."""

    def __init__(self, pool, kv, page, d, head_pad=0, page_pad=0, scale_head_pad=0, scale_page_pad=0, seed=0):
        assert page % BLOCK == 0
        r = np.random.default_rng(seed)
        self.pool, self.kv, self.page, self.d = pool, kv, page, d
        self.blocks = page // BLOCK
        self.head_stride = page * d + head_pad
        self.page_stride = kv * self.head_stride + page_pad
        self.scale_head_stride = self.blocks + scale_head_pad
        self.scale_page_stride = kv * self.scale_head_stride + scale_page_pad
        # any bytes at all, as memory that was never written
        self.keys, self.values = (r.integers(0, 256, pool * self.page_stride + 16).astype(np.uint8) for _ in range(2))
        self.key_scales, self.value_scales = (
            (2.0 ** r.integers(-9, -4, pool * self.scale_page_stride + 4)).astype(np.float32) for _ in range(2))
        page_, head, n = np.arange(pool)[:, None, None], np.arange(kv)[:, None], np.arange(self.blocks)
        self.at = (page_ * self.page_stride + head * self.head_stride + n * BLOCK * d)[..., None] + np.arange(BLOCK * d)
        self.scales_at = page_ * self.scale_page_stride + head * self.scale_head_stride + n

    def wide(self):
        """Keys and values [pool][kv][page][d] in 64 bits, as they stand for."""
        k = NUMBERS[to_blocks(self.keys[self.at])] * self.key_scales[self.scales_at].astype(np.float64)[..., None, None]
        v = NUMBERS[values_to_blocks(self.values[self.at])] \
            * self.value_scales[self.scales_at].astype(np.float64)[..., None, None]
        return tuple(x.reshape(self.pool, self.kv, self.page, self.d) for x in (k, v))

    def fill(self, r, variant, key_std=1.0, value_std=1.0):
        """Every block full of normal values."""
        for which, std in (("keys", key_std), ("values", value_std)):
            x = r.normal(0, std, self.at.shape[:-1] + (BLOCK, self.d))
            largest = np.abs(x).max((-1, -2))
            scale = np.maximum(2.0 ** np.ceil(np.log2(largest / 448)), LEAST[variant])
            codes = encode(x / scale[..., None, None])
            flat = codes.reshape(*codes.shape[:-2], -1) if which == "keys" else values_from_blocks(codes)
            getattr(self, which)[self.at] = flat
            getattr(self, which[:-1] + "_scales")[self.scales_at] = scale

    def set_position(self, which, page, head, slot, dims, codes):
        """Codes of some dims of a position."""
        n, t = divmod(slot, BLOCK)
        base = page * self.page_stride + head * self.head_stride + n * BLOCK * self.d
        dims = np.arange(self.d)[dims]
        at = t * self.d + dims if which == "keys" else t // 4 * 4 * self.d + 4 * dims + t % 4
        getattr(self, which)[base + at] = codes

    def upload(self, dev):
        self.on_device = [dev(x) for x in (self.keys, self.values, self.key_scales, self.value_scales)]
        return self.on_device

    def view(self, lcr, p, table=None):
        k, v, ks, vs = self.on_device
        return lcr.Kv8View(p(k), p(v), p(ks), p(vs), table, self.page, self.page_stride, self.head_stride,
                           self.scale_page_stride, self.scale_head_stride, self.kv, self.d)
