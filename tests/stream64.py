"""The operators of a stream of frames in float64 numpy: rotary positions, what a
cache holds, page tables, and attention over a cache (test reference)."""
import numpy as np


def rotate(x, pos, pairs, frequency, shared):
    """x [tokens, heads, d] float, pos [tokens, axes]."""
    x = np.asarray(x, np.float64)
    out = x.copy()
    o, i, n = 0, 0, sum(pairs)
    for a, s in enumerate(pairs):
        for j in range(s):
            e, u, w = (i / n, i, n + i) if shared else (j / s, o + j, o + s + j)
            t = (pos[:, a].astype(np.float64) * float(frequency) ** -e)[:, None]
            out[..., u] = x[..., u] * np.cos(t) - x[..., w] * np.sin(t)
            out[..., w] = x[..., w] * np.cos(t) + x[..., u] * np.sin(t)
            i += 1
        o += 2 * s
    return out


def q8_0(x):
    """quantize_row_q8_0 of float32 rows, as the values it stands for (float32 products of a value
    and a binary16 scale are exact)."""
    a = np.ascontiguousarray(x, np.float32).reshape(-1, 32)
    # A quotient rounded from float64 is the correctly rounded float32 one.
    d = (np.abs(a).max(1, keepdims=True).astype(np.float64) / 127.0).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(d != 0, (1.0 / d.astype(np.float64)).astype(np.float32), np.float32(0))
    y = (a * inv).astype(np.float64)
    q = np.clip(np.copysign(np.floor(np.abs(y) + 0.5), y), -127, 127)
    with np.errstate(over="ignore", invalid="ignore"):  # scales past binary16 are infinite
        return (q * d.astype(np.float16).astype(np.float64)).astype(np.float32).reshape(x.shape)


def bf16(x):
    """float32 values rounded to bfloat16, half to even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((b + (0x7FFF + ((b >> 16) & 1))) & 0xFFFF0000).astype(np.uint32)
    return r.view(np.float32).reshape(np.shape(x))


def stored(x, kind):
    return {"f32": lambda v: np.asarray(v, np.float32), "bf16": bf16, "q8_0": q8_0}[kind](x)


def pages(cached, added, free, free_start, page, table, tokens):
    """(starts, lens, slots, table, free_next) by walking the requests and their tokens."""
    table = np.array(table)
    slots = np.full(tokens, -1, np.int64)
    starts, lens, taken, t = [0], [], int(free_start), 0
    for r, (c, n) in enumerate(zip(cached, added)):
        c, n = max(int(c), 0), min(max(int(n), 0), tokens - t)
        for p in range(c, c + n):
            col = p // page
            if p % page == 0:
                got = int(free[taken]) if 0 <= taken < len(free) else -1
                taken += 1
                if col < table.shape[1]:
                    table[r, col] = got
            held = int(table[r, col]) if col < table.shape[1] else -1
            slots[t] = held * page + p % page if held >= 0 else -1
            t += 1
        starts.append(t)
        lens.append(c + n)
    return np.array(starts), np.array(lens), slots, table, taken


def seen(length, n, block=0, window=0):
    """[n, length]: whether a new token sees a key."""
    pos = np.arange(length - n, length)
    hi = np.full(n, length) if not block else np.where(pos < 0, 0, np.minimum(length, (pos // block + 1) * block))
    lo = np.maximum(0, hi - window) if window else np.zeros(n, int)
    j = np.arange(length)
    return (j[None] >= lo[:, None]) & (j[None] < hi[:, None])


def attention(q, k, v, starts, lens, heads, block=0, window=0, absent=None, dtype=np.float64):
    """q [tokens, heads, d]; k, v: per request [len, kv_heads, d]; absent: per request [len], keys that are not there.
    Rows behind the last request are zeros.  An unseen key or value counts for nothing, whatever it holds; a seen
    value that is not finite makes its dim NaN, a seen key that is not the row infinite (no defined row)."""
    q = np.asarray(q, dtype)
    out = np.zeros(q.shape, dtype)
    for r in range(len(lens)):
        n, length = int(starts[r + 1] - starts[r]), int(lens[r])
        if n <= 0 or length <= 0:
            continue
        group = heads // k[r].shape[1]
        mask = seen(length, n, block, window)
        if absent is not None:
            mask &= ~absent[r][None]
        for h in range(heads):
            kk, vv = k[r][:, h // group].astype(dtype), v[r][:, h // group].astype(dtype)
            with np.errstate(invalid="ignore"):
                s = (q[starts[r]:starts[r + 1], h] @ kk.T) * dtype(1 / np.sqrt(q.shape[-1]))
            s = np.where(mask, s, -np.inf)
            bad_key = (mask & ~np.isfinite(kk).all(1)[None]).any(1)
            s[:, ~np.isfinite(kk).all(1)] = -np.inf
            top = s.max(1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(top), top, 0))
            total = p.sum(1, keepdims=True)
            o = p @ np.where(np.isfinite(vv), vv, 0) / np.where(total > 0, total, 1)
            o[(mask.astype(np.float32) @ (~np.isfinite(vv)).astype(np.float32)) > 0] = np.nan
            o[bad_key] = np.inf
            out[starts[r]:starts[r + 1], h] = o
    return out
