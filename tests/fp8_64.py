"""Rows in 8-bit floating point, products with them, an encoder's stored states and the
attention over them, in float64 numpy (test reference)."""
import math

import numpy as np


def e4m3_values():
    """The value of each of the 256 codes."""
    v = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v[c] = math.ldexp(8 + m, e - 10) if e else math.ldexp(m, -9)
        if c & 127 == 127:
            v[c] = np.nan
    v[128:] = -v[128:]
    return v


VALUES = e4m3_values()


def e4m3(y):
    """Codes of float64 values of at most 448: nearest, half to the even code; NaN to 0x7f."""
    y = np.asarray(y, np.float64)
    a = np.abs(np.where(np.isnan(y), 0.0, y))
    grid = VALUES[:127]
    hi = np.clip(np.searchsorted(grid, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(a == grid[hi], hi, code)
    code = code | np.where(np.signbit(y), 128, 0)
    return np.where(np.isnan(y), 127, code).astype(np.uint8)


def blocks(k):
    return -(-k // 128)


def quantise(x):
    """(codes [rows, k], exponents + 127 [rows, blocks]) of float32 rows."""
    rows, k = x.shape
    nb = blocks(k)
    p = np.zeros((rows, nb * 128))
    p[:, :k] = x
    p = np.where(np.isfinite(p), p, np.nan).reshape(rows, nb, 128)
    amax = np.nanmax(np.concatenate([np.abs(p), np.zeros((rows, nb, 1))], -1), -1)
    m, e = np.frexp(amax)  # 448 = 0.875 * 2^9
    e = np.where(amax == 0, -127, np.where(m > 0.875, e - 8, e - 9)).clip(-127, 127)
    codes = e4m3(p * np.ldexp(1.0, -e)[..., None]).reshape(rows, nb * 128)[:, :k]
    return np.ascontiguousarray(codes), (e + 127).astype(np.uint8)


def values(codes, exps):
    k = codes.shape[1]
    return VALUES[codes] * np.repeat(np.ldexp(1.0, exps.astype(int) - 127), 128, 1)[:, :k]


def block_values(codes, scales):
    """[N, K] codes with a scale for each 128 x 128."""
    n, k = codes.shape
    s = np.asarray(scales, np.float64).reshape(blocks(n), blocks(k))
    return VALUES[codes] * np.repeat(np.repeat(s, 128, 0)[:n], 128, 1)[:, :k]


def gelu(x):
    return x * 0.5 * np.vectorize(math.erfc)(-x * math.sqrt(0.5))


# ---- an encoder's states --------------------------------------------------------------


def halves(x, amax, parts):
    """x as `parts` binary16 halves of x 2^-e hold it, amax 2^-e in [2^14, 2^15)."""
    _, e = np.frexp(amax.astype(np.float64))
    e = np.where(amax == 0, 0, e - 15)
    s = np.ldexp(np.asarray(x, np.float64), -e)
    hi = s.astype(np.float16).astype(np.float64)
    lo = (s - hi).astype(np.float32).astype(np.float16).astype(np.float64) if parts == 2 else 0.0
    return np.ldexp(hi + lo, e)


def stored(k, v, kind, seen=None):
    """K and V [tokens, heads, dim] of one image as its states hold them: the seen tokens."""
    if seen is not None:
        k, v = k[seen != 0], v[seen != 0]
    if not len(k):
        return k.astype(np.float64), v.astype(np.float64)
    parts = 2 if kind == "f32" else 1
    top = lambda x, axis: np.max(np.where(np.isfinite(x), np.abs(x), 0), axis, keepdims=True)  # noqa: E731
    return halves(k, top(k, (0, 2)), parts), halves(v, top(v, 0), parts)


def attention(q, k, v):
    """One image: q [n, heads, d], k and v [tokens, kv_heads, d] -> [n, heads, d]."""
    n, heads, d = q.shape
    out = np.zeros(q.shape)
    for h in range(heads if len(k) else 0):
        one = h // (heads // k.shape[1])
        s = q[:, h].astype(np.float64) @ k[:, one].T / np.sqrt(d)
        p = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = p @ v[:, one] / p.sum(1, keepdims=True)
    return out
