"""The 8-bit paged key/value cache in 64 bits: append, norm and rotation, attention, written from their definitions."""
import math

import numpy as np

PAGE = 16
UNASSIGNED = 0xFFFFFFFF


def round_e4m3(values):
    """Nearest E4M3 value (ties to the even one) of |values| <= 448; infinities go to 448, NaN stays."""
    values = np.asarray(values, dtype=np.float64)
    clipped = np.clip(values, -448.0, 448.0)
    _, exponent = np.frexp(np.where(clipped == 0, 2.0 ** -20, clipped))
    step = np.exp2(np.maximum(exponent - 1, -6) - 3.0)
    return np.where(np.isnan(values), np.nan, np.round(clipped / step) * step)


# value of every code, NaN at 0x7f and 0xff
_CODES = np.arange(256)
_SIGN = np.where(_CODES & 0x80, -1.0, 1.0)
_FIELD, _FRACTION = (_CODES >> 3) & 15, _CODES & 7
CODE_VALUES = _SIGN * np.where(_FIELD == 0, _FRACTION * 2.0 ** -9, (8 + _FRACTION) * np.exp2(_FIELD - 10.0))
CODE_VALUES[0x7F] = CODE_VALUES[0xFF] = np.nan


def scale_of(largest):
    """Least 2^e, e >= -126, with largest <= 448 * 2^e."""
    if largest == 0:
        return 2.0 ** -126
    return 2.0 ** max(-126, math.ceil(math.log2(largest / 448.0) - 1e-12))


class Cache:
    """values [pages, heads, 16, dim] before their scale, and scales [pages, heads], for keys or for values."""

    def __init__(self, codes, scales):
        self.values = CODE_VALUES[codes]
        self.scales = np.asarray(scales, dtype=np.float64).copy()

    def append(self, rows, slots):
        """rows [tokens, heads, dim] at slots [tokens]."""
        pages = len(self.values)
        token = 0
        while token < len(slots):
            if slots[token] < 0 or slots[token] // PAGE >= pages:
                token += 1
                continue
            end = token + 1
            while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % PAGE:
                end += 1
            page, offset = slots[token] // PAGE, slots[token] % PAGE
            for head in range(rows.shape[1]):
                run = rows[token:end, head]
                finite = np.abs(run[np.isfinite(run)])
                scale = scale_of(finite.max() if finite.size else 0.0)
                if offset:
                    old = max(self.scales[page, head], 2.0 ** -126)
                    scale = max(scale, old)
                    self.values[page, head, :offset] = round_e4m3(self.values[page, head, :offset] * (old / scale))
                self.scales[page, head] = scale
                self.values[page, head, offset:offset + end - token] = round_e4m3(run / scale)
            token = end

    def full(self):
        return self.values * self.scales[:, :, None, None]


def norm_rope(x, weight, inv_freq, positions, eps):
    x = np.asarray(x, dtype=np.float64)
    x = x / np.sqrt(np.mean(x * x, axis=2, keepdims=True) + eps) * weight
    angle = (np.asarray(positions, dtype=np.float64)[:, None] * np.asarray(inv_freq, dtype=np.float64))[:, None]
    half = x.shape[2] // 2
    low, high = x[:, :, :half], x[:, :, half:]
    return np.concatenate((low * np.cos(angle) - high * np.sin(angle), high * np.cos(angle) + low * np.sin(angle)), axis=2)


def attend(query, key, value, tables, rows, positions, window=0, sinks=0, scale=None):
    """Exact outputs [tokens, heads, dim], and for each the sum of weight * |value| and the largest sum |q k| * scale, which
    rounding errors are proportional to.  key / value are full() caches."""
    tokens, heads, dim = query.shape
    group = heads // key.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, magnitude, score = (np.full((tokens, heads, dim), np.nan), np.zeros((tokens, heads, dim)), np.zeros((tokens, heads, 1)))
    for token in range(tokens):
        if rows[token] >= len(tables):
            continue
        last = int(positions[token])
        index = np.arange(last + 1)
        if window:
            index = index[(index > last - window) | (index < sinks)]
        pages, offsets = tables[rows[token]][index // PAGE], index % PAGE
        if (pages >= len(key)).any():
            continue
        for head in range(heads):
            k, v = key[pages, head // group, offsets], value[pages, head // group, offsets]
            s = k @ query[token, head] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[token, head], magnitude[token, head] = w @ v, w @ np.abs(v)
            score[token, head] = (np.abs(k) @ np.abs(query[token, head])).max() * scale
    return out, magnitude, score


def tolerance(exact, magnitude, score, dim, weight_rounding):
    """A weight is rounded by at most `weight_rounding`, the result by 2^-8.  A score has dim products of f32 size, each added
    with an error of 2^-23 at most of the largest partial sum, and a handful of scalings; it moves numerator and denominator."""
    scores = 2 * (dim + 8) * 2.0 ** -23 * score
    return 2.0 ** -8 * np.abs(exact) + (1 + 2.0 ** -8) * (weight_rounding + scores + 2.0 ** -20) * magnitude + 1e-37
