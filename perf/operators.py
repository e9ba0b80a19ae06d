"""Operators of a stream of frames: rotary positions of several axes, a paged cache
of keys and values with its page tables, and the attention of new tokens over it.

A program that feeds the encoder frame after frame (or token after token) rotates
the new queries and keys, writes the keys and values to pages of a cache, and lets
the new queries attend to what the cache holds.  A case is a dict of plain values;
``kind`` selects the operator.  ``run`` makes the framework's calls where ``own`` is
true and computes the same in elementary torch operations where it is false.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
MAX_LEN = 16384


def listed():
    return [
        # One 504 x 336 frame (24 x 36 patches and the CLS token), head-major as the QKV
        # projection writes it: time, height and width positions.
        {"name": "rope_frame", "kind": "rope", "heads": 12, "frames": 1, "rows": 24, "cols": 36,
         "head_dim": 64, "pairs": "8,12,12", "shared": False, "token_major": False},
        # Sixteen 1008 x 672 frames of a video at once, token-major, one spectrum shared by the axes.
        {"name": "rope_video", "kind": "rope", "heads": 12, "frames": 16, "rows": 48, "cols": 72,
         "head_dim": 64, "pairs": "10,10,10", "shared": True, "token_major": True},
        # Eight streams that get a token each: the tables of one decoding step.
        {"name": "pages_step", "kind": "pages", "requests": 8, "most_new": 1, "most_cached": 4000,
         "page": 64, "spare": 0},
        # A thousand ragged requests admitted together on small pages, in a padded batch.
        {"name": "pages_batch", "kind": "pages", "requests": 1024, "most_new": 300,
         "most_cached": 2000, "page": 16, "spare": 1001},
        # Single tokens of sixteen streams, grouped heads, bfloat16 cache: launch latency.
        {"name": "append_tokens", "kind": "append", "tokens": 16, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "type": "bf16", "page": 64, "axes": 1, "spare": 0},
        # One frame's QKV rows into a Q8_0 cache (quantised weights' companion).
        {"name": "append_frame_q8", "kind": "append", "tokens": 865, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "type": "q8_0", "page": 32, "axes": 3, "spare": 3},
        # Four 1008 x 672 frames into a float cache: the bandwidth case.
        {"name": "append_video", "kind": "append", "tokens": 13828, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "type": "f32", "page": 128, "axes": 3, "spare": 0},
        # One new token against four cached frames: the smallest call.
        {"name": "attn_token", "kind": "attention", "requests": 1, "most_new": 1, "least_new": 1,
         "most_len": 3461, "least_len": 3461, "heads": 12, "kv_heads": 12, "head_dim": 64,
         "type": "f32", "page": 64, "block": 0, "window": 0},
        # Sixty-four streams of very different lengths, a token each, grouped heads: cache bandwidth.
        {"name": "attn_tokens_64", "kind": "attention", "requests": 64, "most_new": 1,
         "least_new": 1, "most_len": MAX_LEN, "least_len": 130, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "type": "bf16", "page": 64, "block": 1, "window": 0},
        # A frame against itself and seven earlier ones, full precision.
        {"name": "attn_frame", "kind": "attention", "requests": 1, "most_new": 865,
         "least_new": 865, "most_len": 6920, "least_len": 6920, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "type": "f32", "page": 32, "block": 865, "window": 0},
        # Ragged causal chunks of a batch over a Q8_0 cache, with a sliding window.
        {"name": "attn_chunks_q8", "kind": "attention", "requests": 6, "most_new": 701,
         "least_new": 33, "most_len": 4099, "least_len": 800, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "type": "q8_0", "page": 16, "block": 1, "window": 2048},
        # A 1008 x 672 frame against itself and five earlier ones: the largest product.
        {"name": "attn_video", "kind": "attention", "requests": 1, "most_new": 3457,
         "least_new": 3457, "most_len": 20742, "least_len": 20742, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "type": "bf16", "page": 256, "block": 0, "window": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "pages", "append", "append", "attention", "attention", "attention",
                       "attention"])
    heads, kv_heads = rng.choice([(12, 12), (12, 12), (6, 6), (32, 8), (16, 2), (12, 4), (9, 3), (8, 1)])
    head_dim = rng.choice([64, 64, 128, 32, 96])
    kind_of_cache = rng.choice(["f32", "bf16", "q8_0"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "rope":
        half = head_dim // 2
        axes = rng.randint(1, 4)
        pairs = [rng.randint(1, half // axes) for _ in range(axes)]
        rows, cols = _log_int(rng, 1, 48), _log_int(rng, 1, 72)
        return {"kind": "rope", "heads": heads, "frames": rng.randint(1, 8), "rows": rows, "cols": cols,
                "head_dim": head_dim, "pairs": ",".join(map(str, pairs)),
                "shared": rng.random() < 0.5, "token_major": rng.random() < 0.5}
    if kind == "pages":
        return {"kind": "pages", "requests": _log_int(rng, 1, 1024), "most_new": _log_int(rng, 1, 300),
                "most_cached": _log_int(rng, 1, 8000), "page": page, "spare": rng.choice([0, 1, 77])}
    if kind == "append":
        return {"kind": "append", "tokens": _log_int(rng, 1, 6000), "heads": heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "type": kind_of_cache, "page": page, "axes": rng.randint(0, 3),
                "spare": rng.choice([0, 0, 5])}
    if rng.random() < 0.5:  # single tokens
        return {"kind": "attention", "requests": _log_int(rng, 1, 64), "most_new": rng.choice([1, 1, 4]),
                "least_new": 1, "most_len": _log_int(rng, 64, 8000), "least_len": rng.randint(4, 64),
                "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "type": kind_of_cache,
                "page": page, "block": 1, "window": rng.choice([0, 0, 1000])}
    most_new = _log_int(rng, 5, 1500)
    case = {"kind": "attention", "requests": rng.randint(1, 4), "most_new": most_new,
            "least_new": rng.randint(1, most_new), "most_len": most_new + _log_int(rng, 1, 6000),
            "least_len": most_new, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "type": kind_of_cache, "page": page, "block": rng.choice([0, 1, 1, 865, 100]),
            "window": rng.choice([0, 0, 700])}
    while case["requests"] > 1 and work(case)["flops"] > 1e11:
        case["requests"] -= 1
    return case


# ---- inputs ----------------------------------------------------------------------


def _lens(case):
    """(new tokens, lengths with them) of each request: of the case alone, so that work() knows them."""
    r = random.Random("%(requests)d %(most_new)d %(most_len)d %(heads)d" % case)
    new = [r.randint(case["least_new"], case["most_new"]) for _ in range(case["requests"])]
    lens = [max(n, _log_int(r, case["least_len"], case["most_len"])) for n in new]
    new[0], lens[-1] = case["most_new"], case["most_len"]
    lens[0] = max(lens[0], new[0])
    return new, lens


def _pages_lens(case):
    r = random.Random("%(requests)d %(most_new)d %(most_cached)d" % case)
    cached = [r.randint(0, case["most_cached"]) for _ in range(case["requests"])]
    new = [r.randint(0, case["most_new"]) if case["most_new"] > 1 else 1 for _ in range(case["requests"])]
    new[-1] = case["most_new"]
    return cached, new


def _rng(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) + 101)


def _normal(rng, *shape, std=1.0):
    return torch.randn(*shape, generator=rng, device=DEV, dtype=torch.float32) * std


def _i32(values):
    return torch.as_tensor(np.asarray(values), device=DEV).to(torch.int32)


def _q8(x):
    """(values, scales) of Q8_0 blocks of 32: d = amax / 127, values round(x (1 / d)) half away
    from zero, d kept in 16 bits; the two quotients correctly rounded to 32 bits."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    d = (amax.double() / 127.0).float()
    inv = torch.where(d != 0, 1.0 / d.double(), 0.0).float()
    y = (b * inv).double()
    q = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-127, 127).to(torch.int8)
    return q.reshape(x.shape), d[..., 0].to(torch.float16)


def _q8_values(q, d):
    return (q.reshape(*q.shape[:-1], -1, 32).float() * d.float()[..., None]).reshape(q.shape)


def _stored(x, kind):
    return x if kind == "f32" else x.to(torch.bfloat16) if kind == "bf16" else _q8(x)


def _values(s, kind):
    return _q8_values(*s) if kind == "q8_0" else s.float()


def _axis_of(pairs):
    return [a for a, s in enumerate(pairs) for _ in range(s)]


def _rope_plan(pairs, shared, base):
    """Of each rotated pair: its two dims, its axis and its frequency."""
    first, second, axis, freq, o, n = [], [], _axis_of(pairs), [], 0, sum(pairs)
    for s in pairs:
        for j in range(s):
            if shared:
                i = len(first)
                first.append(i), second.append(n + i), freq.append(base ** (-i / n))
            else:
                first.append(o + j), second.append(o + s + j), freq.append(base ** (-j / s))
        o += 2 * s
    to = dict(device=DEV, dtype=torch.int64)
    return {"first": torch.tensor(first, **to), "second": torch.tensor(second, **to),
            "axis": torch.tensor(axis, **to),
            "freq": torch.tensor(freq, device=DEV, dtype=torch.float64)}


def _rope_inputs(case, seed):
    rng = _rng(seed)
    f, r, c = case["frames"], case["rows"], case["cols"]
    pairs = [int(v) for v in case["pairs"].split(",")]
    t = torch.arange(f, device=DEV)[:, None].expand(f, r * c + 1) + 1000 * (int(seed) % 97)
    p = torch.arange(r * c, device=DEV)
    y = torch.cat([torch.zeros(1, device=DEV, dtype=torch.int64), p // c + 1])[None].expand(f, -1)
    x = torch.cat([torch.zeros(1, device=DEV, dtype=torch.int64), p % c + 1])[None].expand(f, -1)
    axes = [t, y, x, t + y][: len(pairs)]
    pos = torch.stack([a.reshape(-1) for a in axes], 1).to(torch.int32).contiguous()
    n = pos.shape[0]
    shape = (n, case["heads"], case["head_dim"]) if case["token_major"] else (case["heads"], n, case["head_dim"])
    return {"x": _normal(rng, *shape), "pos": pos, "tokens": n, "pairs": pairs,
            "base": 10000.0 if case["shared"] else 100.0}


def _pages_inputs(case, seed):
    cached, new = _pages_lens(case)
    page = case["page"]
    held = [-(-c // page) for c in cached]
    need = [-(-(c + n) // page) for c, n in zip(cached, new)]
    width = max(need) + 2
    total = sum(need) + 40
    order = torch.randperm(total, generator=_rng(seed), device=DEV).to(torch.int32).cpu().numpy()
    table = np.full((case["requests"], width), -1, np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at: at + h]
        at += h
    return {"cached": _i32(cached), "new": _i32(new), "table": _i32(table), "width": width,
            "free": _i32(order[at - 7 if at >= 7 else 0:]), "free_start": _i32([min(7, at)]),
            "tokens": sum(new) + case["spare"]}


def _append_inputs(case, seed):
    rng = _rng(seed)
    n, h, g, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    pages = -(-n // case["page"]) + 3
    slots = torch.randperm(pages * case["page"], generator=rng, device=DEV)[: n + case["spare"]].to(torch.int32)
    if case["page"] > 1 and n > case["page"]:  # whole pages in any order, as a table gives them
        order = torch.randperm(pages, generator=rng, device=DEV)
        t = torch.arange(n + case["spare"], device=DEV)
        slots = (order[t // case["page"]] * case["page"] + t % case["page"]).to(torch.int32)
    if case["spare"]:
        slots[n:] = -1
    n += case["spare"]
    pairs = [[], [d // 2], [d // 4, d // 4], [d // 2 - 2 * (d // 6), d // 6, d // 6]][case["axes"]]
    pos = torch.randint(0, 5000, (n, max(1, len(pairs))), generator=rng, device=DEV, dtype=torch.int32)
    return {"qkv": _normal(rng, n, (h + 2 * g) * d), "slots": slots, "pos": pos, "pairs": pairs,
            "pages": pages, "base": 10000.0, "tokens": n}


def _attention_inputs(case, seed):
    """Queries, the rows of the cache by slot ([pages * page] rows of which the requests own some) and
    the tables.  Rows that no request owns hold what was left there."""
    rng = _rng(seed)
    new, lens = _lens(case)
    page, g, d = case["page"], case["kv_heads"], case["head_dim"]
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=rng, device=DEV).to(torch.int32).cpu().numpy()
    table = np.full((case["requests"], max(held)), -1, np.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at: at + n]
        at += n
    k, v = (_normal(rng, pages, page, g, d) for _ in range(2))
    k[..., 3] += 2.0  # a channel that all keys share, as trained ones do
    starts = np.concatenate([[0], np.cumsum(new)])
    return {"q": _normal(rng, sum(new), case["heads"], d, std=1.5), "k": k, "v": v,
            "table": _i32(table), "starts": _i32(starts), "lens": _i32(lens), "pages": pages,
            "width": max(held), "tokens": sum(new), "most_new": max(new), "most_len": max(lens)}


# ---- the framework's side ----------------------------------------------------------

_runtime = None


def _rt():
    global _runtime
    if _runtime is None:
        for p in (os.path.join(os.getcwd(), "vestra-kernels_amd"),
                  os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vestra-kernels_amd")):
            if os.path.isdir(p) and p not in sys.path:
                sys.path.append(p)
        import vestra_hip

        _runtime = vestra_hip.Runtime(0)
    return _runtime


class _Device:
    """A device buffer of the framework as torch sees it."""

    def __init__(self, owner, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": kind, "version": 3,
                                         "data": (owner.device_ptr, False)}


def _floats(*shape):
    """A float tensor of the framework, and torch's view of it."""
    t = _rt().alloc_f32(math.prod(shape))
    return t, torch.as_tensor(_Device(t, shape, "<f4"), device=DEV)


def _ints(*shape):
    t = _rt().alloc_i32(math.prod(shape))
    return t, torch.as_tensor(_Device(t, shape, "<i4"), device=DEV)


def _given(x):
    t, view = _ints(*x.shape) if x.dtype == torch.int32 else _floats(*x.shape)
    view.copy_(x)
    return t


# ---- prepare -------------------------------------------------------------------------


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case, "kind": kind}
    if kind == "rope":
        i = _rope_inputs(case, seed)
        if own:
            out, view = _floats(*i["x"].shape)
            s |= {"x": _given(i["x"]), "pos": _given(i["pos"]), "tokens": i["tokens"], "out": out, "view": view,
                  "rope": _rt().prepare_rope_axes(case["head_dim"], i["pairs"], i["base"], shared=case["shared"])}
        else:
            s |= i | {"plan": _rope_plan(i["pairs"], case["shared"], i["base"])}
    elif kind == "pages":
        i = _pages_inputs(case, seed)
        if own:
            n, r = i["tokens"], case["requests"]
            s |= {k: _given(i[k]) for k in ("cached", "new", "free", "free_start")} | {"width": i["width"]}
            for name, shape in (("table", (r, i["width"])), ("starts", (r + 1,)), ("lens", (r,)),
                                ("slots", (n,)), ("free_next", (1,))):
                s[name], s[name + "_view"] = _ints(*shape)
            s["table_view"].copy_(i["table"])
        else:
            s |= i
    elif kind == "append":
        i = _append_inputs(case, seed)
        n, g, d = i["tokens"], case["kv_heads"], case["head_dim"]
        if own:
            rt = _rt()
            s |= {k: _given(i[k]) for k in ("qkv", "slots", "pos")} | {"tokens": n}
            s["cache"] = rt.kv_cache(case["type"], i["pages"], case["page"], g, d)
            s["rope"] = rt.prepare_rope_axes(d, i["pairs"], i["base"]) if i["pairs"] else None
            s["q"], s["q_view"] = _floats(n, case["heads"], d)
            s["k"], s["k_view"] = _floats(n, g, d)
            s["v"], s["v_view"] = _floats(n, g, d)
        else:
            s |= i | {"plan": _rope_plan(i["pairs"], False, i["base"]) if i["pairs"] else None}
            rows = i["pages"] * case["page"]
            t = {"f32": torch.float32, "bf16": torch.bfloat16, "q8_0": torch.int8}[case["type"]]
            s["cache"] = [torch.zeros(rows, g, d, device=DEV, dtype=t) for _ in range(2)]
            s["scales"] = [torch.zeros(rows, g, d // 32, device=DEV, dtype=torch.float16)
                           for _ in range(2)] if case["type"] == "q8_0" else [None, None]
    else:
        i = _attention_inputs(case, seed)
        if own:
            rt = _rt()
            g, d, rows = case["kv_heads"], case["head_dim"], i["pages"] * case["page"]
            s |= {k: _given(i[k]) for k in ("q", "table", "starts", "lens")}
            s |= {k: i[k] for k in ("tokens", "width")}
            s["cache"] = rt.kv_cache(case["type"], i["pages"], case["page"], g, d)
            s["out"], s["view"] = _floats(i["tokens"], case["heads"], d)
            step = max(1, (1 << 28) // (g * d))
            every = torch.arange(rows, device=DEV, dtype=torch.int32)
            for a in range(0, rows, step):
                b = min(rows, a + step)
                k, v, at = (_given(x[a:b].contiguous())
                            for x in (i["k"].reshape(rows, -1), i["v"].reshape(rows, -1), every))
                torch.cuda.synchronize()
                s["cache"].append(k, v, b - a, at, token_major=True)
                rt.synchronize()
        else:
            s |= i | {"k": _stored(i["k"], case["type"]), "v": _stored(i["v"], case["type"])}
    return s


# ---- one pass ------------------------------------------------------------------------


def _rotate(x, pos, plan):
    """Rows x [tokens, heads, d] rotated by the angles of their positions [tokens, axes]."""
    angle = pos.to(torch.float64)[:, plan["axis"]] * plan["freq"]
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., plan["first"]], x[..., plan["second"]]
    out = x.clone()
    out[..., plan["first"]] = a * c - b * s
    out[..., plan["second"]] = b * c + a * s
    return out


def _rope_plain(s):
    x = s["x"] if s["case"]["token_major"] else s["x"].transpose(0, 1)
    y = _rotate(x, s["pos"], s["plan"])
    return y if s["case"]["token_major"] else y.transpose(0, 1).contiguous()


def _pages_plain(s):
    page, n = s["case"]["page"], s["tokens"]
    c, a = s["cached"].long(), s["new"].long()
    held, need = (c + page - 1) // page, (c + a + page - 1) // page
    first = torch.cumsum(need - held, 0) - (need - held)
    ends = torch.cumsum(a, 0)
    starts = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(n, device=DEV)
    r = torch.searchsorted(ends, t, right=True).clamp(max=c.numel() - 1)
    pos = c[r] + t - starts[r]
    col = pos // page
    fresh = col >= held[r]
    at = (s["free_start"].long() + first[r] + col - held[r]).clamp(0, s["free"].numel() - 1)
    got = torch.where(fresh, s["free"].long()[at], s["table"].long()[r, col.clamp(max=s["width"] - 1)])
    inside = t < starts[-1]
    slots = torch.where(inside, got * page + pos % page, -1)
    table = torch.cat([s["table"].reshape(-1), s["table"].new_zeros(1)])
    table[torch.where(inside & fresh, r * s["width"] + col, table.numel() - 1)] = got.to(torch.int32)
    free_next = s["free_start"].long() + (need - held).sum()
    return {"starts": starts.to(torch.int32), "lens": (c + a).to(torch.int32), "slots": slots.to(torch.int32),
            "table": table[:-1].reshape(-1, s["width"]), "free_next": free_next.to(torch.int32)}


def _append_plain(s):
    case = s["case"]
    n, h, g, d = s["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    rows = s["qkv"].reshape(n, h + 2 * g, d)
    q, k, v = rows[:, :h], rows[:, h: h + g], rows[:, h + g:]
    if s["plan"] is not None:
        q, k = _rotate(q, s["pos"], s["plan"]), _rotate(k, s["pos"], s["plan"])
    live = s["slots"] >= 0
    at = s["slots"].long()[live]
    read = []
    for x, cache, scales in ((k, s["cache"][0], s["scales"][0]), (v, s["cache"][1], s["scales"][1])):
        if scales is None:
            cache[at] = x[live].to(cache.dtype)
            got = cache[s["slots"].long().clamp(min=0)].float()
        else:
            cache[at], scales[at] = _q8(x[live])
            m = s["slots"].long().clamp(min=0)
            got = _q8_values(cache[m], scales[m])
        read.append(torch.where(live[:, None, None], got, 0.0))
    return {"q": q.contiguous(), "k": read[0], "v": read[1]}


def _attention_plain(s):
    """Every request padded to the longest: its queries [R, N], its keys by the page table [R, L]."""
    case = s["case"]
    h, g, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    n, most = s["most_new"], s["most_len"]
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    i, j = torch.arange(n, device=DEV), torch.arange(most, device=DEV)
    slot = s["table"].long().clamp(min=0)[:, j // page] * page + j % page
    there = (j[None] < lens[:, None])[..., None, None]

    def rows(x):
        if case["type"] == "q8_0":
            got = _q8_values(x[0].reshape(-1, g, d)[slot], x[1].reshape(-1, g, d // 32)[slot])
        else:
            got = x.reshape(-1, g, d)[slot].float()
        return torch.where(there, got, 0.0).permute(0, 2, 1, 3).contiguous()

    real = i[None] < new[:, None]
    row = (starts[:-1, None] + i[None]).clamp(max=s["tokens"] - 1)
    q = s["q"][row].reshape(-1, n, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(-1, g, h // g * n, d)
    pos = (lens - new)[:, None] + i[None]
    hi = lens[:, None].expand_as(pos)
    if case["block"]:
        hi = torch.minimum(hi, (pos // case["block"] + 1) * case["block"])
    lo = (hi - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(hi)
    seen = (j >= lo[..., None]) & (j < hi[..., None])  # [R, N, L]
    x = torch.matmul(q, rows(s["k"]).transpose(-1, -2).contiguous())
    x = (x * (1.0 / math.sqrt(d))).reshape(-1, g, h // g, n, most)
    x = torch.where(seen[:, None, None], x, float("-inf"))
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(-1, g, h // g * n, most), rows(s["v"])).reshape(-1, g, h // g, n, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(-1, n, h, d)[real]


def run(s):
    kind, case = s["kind"], s["case"]
    if not own:
        return {"rope": _rope_plain, "pages": _pages_plain, "append": _append_plain,
                "attention": _attention_plain}[kind](s)
    if kind == "rope":
        s["rope"].run(s["x"], case["heads"], s["tokens"], s["pos"], s["out"], token_major=case["token_major"])
        return s["view"]
    if kind == "pages":
        _rt().kv_pages_assign(s["cached"], s["new"], s["free"], s["free_start"], case["page"], s["table"],
                              s["width"], s["starts"], s["lens"], s["slots"], s["free_next"])
        return {k: s[k + "_view"] for k in ("starts", "lens", "slots", "table", "free_next")}
    if kind == "append":
        s["cache"].append_qkv(s["qkv"], case["heads"], s["tokens"], s["slots"], s["q"], rope=s["rope"],
                              positions=s["pos"] if s["rope"] else None)
        s["cache"].gather(s["slots"], s["tokens"], s["k"], s["v"])
        return {k: s[k + "_view"] for k in "qkv"}
    s["cache"].attention(s["q"], case["heads"], s["tokens"], s["table"], s["width"], s["starts"], s["lens"],
                         s["out"], block=case["block"], window=case["window"])
    return s["view"]


# ---- what a pass cannot do without -----------------------------------------------------

_BYTES = {"f32": 4.0, "bf16": 2.0, "q8_0": 34.0 / 32.0}


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["frames"] * (case["rows"] * case["cols"] + 1)
        axes = case["pairs"].count(",") + 1
        values = n * case["heads"] * case["head_dim"]
        pairs = sum(int(v) for v in case["pairs"].split(","))
        return {"bytes": 8 * values + 4 * n * axes, "flops": 6 * pairs * n * case["heads"]}
    if kind == "pages":
        cached, new = _pages_lens(case)
        p = case["page"]
        fresh = sum(-(-(c + n) // p) - -(-c // p) for c, n in zip(cached, new))
        return {"bytes": 4 * (2 * len(new) + 2 * fresh + sum(new) + case["spare"] + 2 * len(new) + 1), "flops": 0}
    d, h, g = case["head_dim"], case["heads"], case["kv_heads"]
    if kind == "append":
        n = case["tokens"] + case["spare"]
        # The rows in, Q out, K and V written and read back as floats.
        return {"bytes": n * d * (4 * (h + 2 * g) + 4 * h + 2 * g * (2 * _BYTES[case["type"]] + 4)) +
                4 * n * (2 + max(1, case["axes"])), "flops": 3 * n * d * (h + g)}
    new, lens = _lens(case)
    pairs = rows = 0
    for n, length in zip(new, lens):
        pos = np.arange(length - n, length)
        hi = np.minimum(length, (pos // case["block"] + 1) * case["block"]) if case["block"] else np.full(n, length)
        lo = np.maximum(0, hi - case["window"]) if case["window"] else np.zeros_like(hi)
        pairs += int((hi - lo).sum())
        rows += int(hi.max() - lo.min())
    return {"bytes": rows * 2 * g * d * _BYTES[case["type"]] + 8 * sum(new) * h * d, "flops": 4 * d * h * pairs}


# ---- the definition, in 64 bits ----------------------------------------------------------


def _rotated(x, pos, pairs, shared, base):
    x = x.double().clone()
    out = x.clone()
    o, i, n = 0, 0, sum(pairs)
    for a, s in enumerate(pairs):
        for j in range(s):
            f, u, w = (base ** (-i / n), i, n + i) if shared else (base ** (-j / s), o + j, o + s + j)
            t = (pos[:, a].double() * f)[:, None]
            out[..., u] = x[..., u] * torch.cos(t) - x[..., w] * torch.sin(t)
            out[..., w] = x[..., w] * torch.cos(t) + x[..., u] * torch.sin(t)
            i += 1
        o += 2 * s
    return out


def _as_stored(x, kind):
    """What a cache of that type holds of these floats."""
    if kind == "f32":
        return x.double()
    if kind == "bf16":
        return x.bfloat16().double()
    a = x.cpu().numpy().reshape(-1, 32)
    d = (np.abs(a).max(1, keepdims=True).astype(np.float64) / 127.0).astype(np.float32)
    inv = np.zeros_like(d)
    np.divide(np.float32(1.0), d, out=inv, where=d != 0)
    y = (a * inv).astype(np.float64)
    q = np.clip(np.copysign(np.floor(np.abs(y) + 0.5), y), -127, 127)
    return torch.from_numpy(q * d.astype(np.float16).astype(np.float64)).to(DEV).reshape(x.shape)


def exact(case, seed):
    kind = case["kind"]
    if kind == "pages":
        return None  # whole numbers
    if kind == "rope":
        i = _rope_inputs(case, seed)
        x = i["x"] if case["token_major"] else i["x"].transpose(0, 1)
        y = _rotated(x, i["pos"], i["pairs"], case["shared"], i["base"])
        return y if case["token_major"] else y.transpose(0, 1).contiguous()
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        i = _append_inputs(case, seed)
        rows = i["qkv"].reshape(-1, h + 2 * g, d)
        q, k = (_rotated(x, i["pos"], i["pairs"], False, i["base"]) if i["pairs"] else x.double()
                for x in (rows[:, :h], rows[:, h: h + g]))
        live = (i["slots"] >= 0)[:, None, None]
        # A rotated key next to a border of fewer bits has no one value.
        k = torch.where(live, k, 0.0) if case["type"] == "f32" else None
        v = torch.where(live, _as_stored(rows[:, h + g:].contiguous(), case["type"]), 0.0)
        return {"q": q, "k": k, "v": v}
    i = _attention_inputs(case, seed)
    k = _as_stored(i["k"], case["type"]).reshape(-1, g, d)
    v = _as_stored(i["v"], case["type"]).reshape(-1, g, d)
    out = torch.zeros(i["tokens"], h, d, device=DEV, dtype=torch.float64)
    starts, lens, table = i["starts"].tolist(), i["lens"].tolist(), i["table"].long()
    for r, length in enumerate(lens):
        n = starts[r + 1] - starts[r]
        key = torch.arange(length, device=DEV)
        slot = table[r, key // case["page"]] * case["page"] + key % case["page"]
        pos = torch.arange(length - n, length, device=DEV)
        hi = torch.full_like(pos, length)
        if case["block"]:
            hi = torch.clamp((pos // case["block"] + 1) * case["block"], max=length)
        lo = torch.clamp(hi - case["window"], min=0) if case["window"] else torch.zeros_like(hi)
        hidden = (key[None] < lo[:, None]) | (key[None] >= hi[:, None])
        for head in range(h):
            kh, vh = k[slot, head // (h // g)], v[slot, head // (h // g)]
            score = i["q"][starts[r]: starts[r + 1], head].double() @ kh.T / math.sqrt(d)
            out[starts[r]: starts[r + 1], head] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ vh
    return out
