"""Rotary positions and the 8-bit key / value cache stated plainly, in 64-bit numpy: what tests/cache_cases.py holds the oracle and the HIP
library to.  (include/catgrad_hip.h has the definitions.)"""
import numpy as np

# what the codes 0 .. 126 stand for (127: NaN; 128 + c: minus c)
VALUES = np.array([(c & 7) / 512 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10) for c in range(127)])


def decode(codes):
    codes = np.asarray(codes, np.uint8)
    v = np.where(codes & 127 == 127, np.nan, VALUES[np.minimum(codes & 127, 126)])
    return np.where(codes & 128, -v, v)


def nearest(x):
    """The values of the nearest codes (ties to the even code; the largest beyond the range; NaN stays)."""
    a = np.minimum(np.abs(x), 448.0)
    hi = np.minimum(np.searchsorted(VALUES, np.where(np.isnan(a), 0, a)), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = VALUES[hi] - a, a - VALUES[lo]
    c = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.where(np.isnan(x), np.nan, np.copysign(VALUES[c], x))


def exponent(size):
    e = -117
    while e < 119 and size > 448.0 * 2.0 ** e:
        e += 1
    return e


def rotate(x, position, turns, magnitude, interleaved):
    """x [.., heads, dim] at whole-number positions [..]."""
    n = 2 * len(turns)
    angle = (np.asarray(position, np.float64)[..., None] * np.asarray(turns, np.float64)) % 1.0 * 2 * np.pi
    z = magnitude * np.exp(1j * angle)[..., None, :]
    out = np.array(x, np.float64)
    if interleaved:
        w = (out[..., 0:n:2] + 1j * out[..., 1:n:2]) * z
        out[..., 0:n:2], out[..., 1:n:2] = w.real, w.imag
    else:
        w = (out[..., :n // 2] + 1j * out[..., n // 2:n]) * z
        out[..., :n // 2], out[..., n // 2:n] = w.real, w.imag
    return out


class Head:
    """The keys or the values of one head: values [positions, width] and a scale's exponent for each block."""

    def __init__(self, capacity, width, block):
        self.x, self.e, self.block = np.zeros((capacity, width)), np.full(capacity // block, -117), block

    def append(self, held, new):
        """new [tokens, width] at held, held + 1, ..; what does not fit is left out."""
        new = np.asarray(new, np.float64)[: max(0, len(self.x) - held)]
        if not len(new):
            return
        end = held + len(new)
        for j in range(held // self.block, -(-end // self.block)):
            first, p0, p1 = j * self.block, max(held, j * self.block), min(end, (j + 1) * self.block)
            here = new[p0 - held: p1 - held]
            e = exponent(np.abs(here[np.isfinite(here)]).max(initial=0.0))
            if p0 > first:
                e = max(e, self.e[j])
                self.x[first:p0] = nearest(self.x[first:p0] * 2.0 ** -float(e)) * 2.0 ** float(e)
            self.x[p0:p1] = nearest(here * 2.0 ** -float(e)) * 2.0 ** float(e)
            self.e[j] = e


def attend(q, position, k, v, scale, window):
    """q [rows, dim] at one position over keys and values [positions, ..] -> (result, the sum of weight times |value|, the largest |score|
    term: what rounding errors of a row are in proportion to)."""
    end = min(position + 1, len(k))
    lo = min(end, max(0, position + 1 - window) if window else 0)
    k, v = k[lo:end], v[lo:end]
    if lo == end:
        return np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros((len(q), 1))
    with np.errstate(invalid="ignore"):
        s = q @ k.T * scale
        w = np.exp(s - s.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        terms = abs(scale) * np.abs(q).max(-1, keepdims=True) * np.abs(k).sum(-1).max()
        return w @ v, w @ np.abs(v), terms
