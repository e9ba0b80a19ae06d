"""Operators of a decoder behind the encoder: projections in 8-bit floating point and
attention over the encoder's states.

A program that hangs a decoder behind the encoder quantises the encoder's states once,
projects them to the keys and values of each decoder layer, keeps those, and lets the
layer's queries attend to them, a token or a frame at a time.  A case is a dict of plain
values; ``kind`` selects the operator.  ``run`` makes the framework's calls where ``own``
is true and computes the same in elementary torch operations where it is false.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
BLOCK = 128  # values that share a scale


def listed():
    return [
        # The tokens of one 504 x 336 frame, as a layer norm leaves them: quantised, and read back.
        {"name": "quant_frame", "kind": "quantise", "rows": 865, "k": 768, "spread": 1.0},
        # Sixteen 1008 x 672 frames' states of an odd width: the bandwidth case, short last block.
        {"name": "quant_video", "kind": "quantise", "rows": 55312, "k": 1100, "spread": 6.0},
        # One token's projection to Q, K and V: latency.
        {"name": "linear_token", "kind": "linear", "rows": 1, "k": 768, "n": 2304, "input": "floats",
         "weights": "rows", "epilogue": "store"},
        # One frame's tokens through the MLP's first layer, with its GELU.
        {"name": "linear_frame", "kind": "linear", "rows": 865, "k": 768, "n": 3072, "input": "floats",
         "weights": "rows", "epilogue": "gelu"},
        # A checkpoint's weights with a float scale for each 128 x 128 block, odd sizes.
        {"name": "linear_blocks", "kind": "linear", "rows": 4001, "k": 2200, "n": 5001, "input": "floats",
         "weights": "blocks", "epilogue": "store"},
        # Encoder states, quantised once, through the K and V projection of one wide decoder layer.
        {"name": "linear_states", "kind": "linear", "rows": 13828, "k": 4096, "n": 8192, "input": "rows",
         "weights": "rows", "epilogue": "store"},
        # K and V of one frame, as floats, some tokens masked: stored, and read back.
        {"name": "states_frame", "kind": "states", "images": 1, "tokens": 865, "kv_heads": 12, "head_dim": 64,
         "type": "f32", "token_major": False, "seen": 0.9, "empty": False},
        # Sixteen 1008 x 672 frames' rows of a KV projection, as halves.
        {"name": "states_video", "kind": "states", "images": 16, "tokens": 3457, "kv_heads": 8, "head_dim": 128,
         "type": "f16", "token_major": True, "seen": 1.0, "empty": False},
        # One new token against the states of four frames: the smallest call.
        {"name": "cross_token", "kind": "attention", "images": 1, "queries": 1, "tokens": 3460, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "type": "f16", "token_major": True, "seen": 1.0, "empty": False},
        # A padded batch of single tokens with grouped heads, one image with nothing to see: bandwidth.
        {"name": "cross_tokens_48", "kind": "attention", "images": 48, "queries": 1, "tokens": 6000, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "type": "f16", "token_major": True, "seen": 0.7, "empty": True},
        # One frame's tokens against four other frames' states, as floats, head-major.
        {"name": "cross_frame", "kind": "attention", "images": 1, "queries": 865, "tokens": 3460, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "type": "f32", "token_major": False, "seen": 0.9, "empty": False},
        # A 1008 x 672 frame against six frames' states as halves: the largest product.
        {"name": "cross_video", "kind": "attention", "images": 1, "queries": 3457, "tokens": 20742, "heads": 12,
         "kv_heads": 12, "head_dim": 64, "type": "f16", "token_major": True, "seen": 1.0, "empty": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "linear", "states", "attention", "attention", "attention"])
    if kind == "quantise":
        return {"kind": kind, "rows": _log_int(rng, 1, 20000), "k": _log_int(rng, 1, 3000),
                "spread": rng.choice([1.0, 6.0, 20.0])}
    if kind == "linear":
        case = {"kind": kind, "rows": _log_int(rng, 1, 8000), "k": _log_int(rng, 16, 6000),
                "n": _log_int(rng, 1, 8000), "input": rng.choice(["floats", "floats", "rows"]),
                "weights": rng.choice(["rows", "blocks"]), "epilogue": rng.choice(["store", "store", "gelu"])}
        if rng.random() < 0.3:  # few tokens
            case["rows"] = rng.randint(1, 64)
        return case
    heads, kv_heads, head_dim = rng.choice([(12, 12, 64), (12, 12, 64), (6, 6, 64), (32, 8, 128), (16, 2, 128),
                                            (12, 4, 64), (8, 1, 32), (9, 3, 96), (5, 5, 52), (40, 10, 100)])
    case = {"kind": kind, "images": rng.randint(1, 6), "tokens": _log_int(rng, 1, 8000), "kv_heads": kv_heads,
            "head_dim": head_dim, "type": rng.choice(["f32", "f16"]), "token_major": rng.random() < 0.5,
            "seen": rng.choice([1.0, 1.0, 0.9, 0.3]), "empty": rng.random() < 0.2}
    if kind == "states":
        return case
    case |= {"heads": heads, "queries": _log_int(rng, 1, 3000) if rng.random() < 0.6 else rng.randint(1, 16)}
    if case["queries"] <= 16:
        case["images"] = rng.randint(1, 64)
    while case["images"] > 1 and (work(case)["flops"] > 1e11 or work(case)["bytes"] > 8e8):
        case["images"] -= 1
    while work(case)["flops"] > 2e11:
        case["queries"] = max(1, case["queries"] // 2)
    return case


# ---- inputs ----------------------------------------------------------------------


def _rng(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) + 77)


def _normal(rng, *shape, std=1.0):
    return torch.randn(*shape, generator=rng, device=DEV, dtype=torch.float32) * std


def _quantise_inputs(case, seed):
    """Rows whose sizes differ by 2^spread and more, a block of zeros among them."""
    rng = _rng(seed)
    x = _normal(rng, case["rows"], case["k"]) * torch.exp2(_normal(rng, case["rows"], 1, std=case["spread"]))
    if case["rows"] > 1:
        x[case["rows"] // 2, : BLOCK] = 0.0
    return {"x": x}


def _linear_inputs(case, seed):
    rng = _rng(seed)
    m, k, n = case["rows"], case["k"], case["n"]
    x = _normal(rng, m, k)
    x[:, k // 3] *= 8.0  # a channel of large values, as trained ones have
    w = _normal(rng, k, n, std=1.0 / math.sqrt(k))
    i = {"x": x, "w": w, "bias": _normal(rng, n, std=0.1)}
    if case["weights"] == "blocks":
        nb, kb = -(-n // BLOCK), -(-k // BLOCK)
        i["codes"] = (w.T.contiguous() * (100.0 * math.sqrt(k))).clamp(-448, 448).to(torch.float8_e4m3fn)
        i["scales"] = torch.exp(_normal(rng, nb, kb, std=0.3)) / (100.0 * math.sqrt(k))
        del i["w"]
    return i


def _seen_of(case):
    """Of each image, how many of its tokens there are to see: of the case alone, so that work() knows them."""
    r = random.Random("%(images)d %(tokens)d %(kv_heads)d %(seen)f" % case)
    n = []
    for i in range(case["images"]):
        n.append(case["tokens"] if case["seen"] == 1.0 else
                 min(case["tokens"], max(1, round(case["tokens"] * r.uniform(case["seen"], 1.0)))))
    if case["empty"] and case["images"] > 1:
        n[1] = 0
    return n


def _states_inputs(case, seed):
    """K and V [images, tokens, kv_heads, head_dim] and the mask of the tokens."""
    rng = _rng(seed)
    shape = (case["images"], case["tokens"], case["kv_heads"], case["head_dim"])
    k, v = _normal(rng, *shape), _normal(rng, *shape)
    k[..., 3] += 2.0  # a channel that all keys share, as trained ones do
    counts = torch.tensor(_seen_of(case), device=DEV)
    order = torch.rand(case["images"], case["tokens"], generator=rng, device=DEV).argsort(1).argsort(1)
    seen = (order < counts[:, None]).to(torch.int32)
    return {"k": k, "v": v, "seen": None if case["seen"] == 1.0 and not case["empty"] else seen,
            "lens": _seen_of(case)}


def _attention_inputs(case, seed):
    i = _states_inputs(case, seed)
    i["q"] = _normal(_rng(seed + 5000), case["images"], case["queries"], case["heads"], case["head_dim"], std=1.5)
    return i


def _head_major(x):
    return x.transpose(1, 2).contiguous()


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
    if x is None:
        return None
    t, view = _ints(*x.shape) if x.dtype == torch.int32 else _floats(*x.shape)
    view.copy_(x)
    return t


# ---- prepare -------------------------------------------------------------------------


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case, "kind": kind}
    if kind == "quantise":
        i = _quantise_inputs(case, seed)
        if own:
            s["x"] = _given(i["x"])
            s["rows"] = _rt().alloc_fp8(case["rows"], case["k"])
            s["out"], s["view"] = _floats(case["rows"], case["k"])
        else:
            s |= i
    elif kind == "linear":
        i = _linear_inputs(case, seed)
        m, k, n = case["rows"], case["k"], case["n"]
        if own:
            rt = _rt()
            if case["weights"] == "blocks":
                s["linear"] = rt.prepare_linear_fp8_blocks(k, n, i["codes"].view(torch.uint8).cpu().numpy(),
                                                           i["scales"].cpu().numpy(), i["bias"].cpu().numpy())
            else:
                s["linear"] = rt.prepare_linear_fp8(k, n, i["w"].cpu().numpy(), i["bias"].cpu().numpy())
            s["x"] = _given(i["x"])
            s["out"], s["view"] = _floats(m, n)
            torch.cuda.synchronize()
            if case["input"] == "rows":
                s["rows"] = rt.quantize_fp8(s["x"], m, k)
                rt.synchronize()
                del s["x"]
        else:
            s["bias"] = i["bias"]
            s["x"] = _fp8_rows(i["x"]) if case["input"] == "rows" else i["x"]
            if case["weights"] == "blocks":
                s |= {"codes": i["codes"], "scales": i["scales"]}
            else:  # [N, K] codes with a scale for 128 values of a row, laid out once
                s["codes"], s["exps"] = _fp8_rows(i["w"].T.contiguous())
    else:
        i = _attention_inputs(case, seed) if kind == "attention" else _states_inputs(case, seed)
        b, t, g, d = case["images"], case["tokens"], case["kv_heads"], case["head_dim"]
        if own:
            rt = _rt()
            s["kv"] = rt.cross_kv(case["type"], b, t, g, d)
            s["seen"] = _given(i["seen"])
            if case["token_major"]:  # rows of a projection to K and V
                s["rows"] = _given(torch.cat([i["k"].reshape(b * t, g * d), i["v"].reshape(b * t, g * d)], 1))
            else:
                s["k"], s["v"] = _given(_head_major(i["k"])), _given(_head_major(i["v"]))
            if kind == "states":
                s["k_out"], s["k_view"] = _floats(b, t, g, d)
                s["v_out"], s["v_view"] = _floats(b, t, g, d)
                s["lens"], s["lens_view"] = _ints(b)
            else:
                torch.cuda.synchronize()
                _write(s)
                rt.synchronize()
                for name in ("seen", "rows", "k", "v"):
                    s.pop(name, None)
                q = i["q"] if case["token_major"] else _head_major(i["q"])
                s["q"] = _given(q)
                s["out"], s["view"] = _floats(*q.shape)
        elif kind == "states":
            s |= {"seen": i["seen"]}
            if case["token_major"]:
                s["rows"] = torch.cat([i["k"].reshape(b * t, g * d), i["v"].reshape(b * t, g * d)], 1)
            else:
                s |= {"k": _head_major(i["k"]), "v": _head_major(i["v"])}
        else:
            k, v, lens = _stored(i["k"], i["v"], i["seen"], case["type"])
            s |= {"k": k, "v": v, "lens": lens, "q": i["q"] if case["token_major"] else _head_major(i["q"])}
    return s


# ---- one pass ------------------------------------------------------------------------


def _pow2(e):
    """2^e for -127 <= e <= 127, by its bits."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _fp8_rows(x):
    """(codes, exponents): of each 128 values of a row the least e with all of them within 448 2^e,
    and the values over 2^e rounded to e4m3.  448 is 0.875 2^9."""
    rows, k = x.shape
    nb = -(-k // BLOCK)
    b = torch.nn.functional.pad(x, (0, nb * BLOCK - k)).reshape(rows, nb, BLOCK)
    m, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(m == 0, -127, e).clamp(-127, 127)
    codes = (b * _pow2(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes.reshape(rows, nb * BLOCK)[:, :k], e


def _fp8_values(rows):
    codes, e = rows
    m, k = codes.shape
    return codes.float() * _pow2(e).repeat_interleave(BLOCK, 1)[:, :k]


def _linear_plain(s):
    case = s["case"]
    n, k = case["n"], case["k"]
    rows = s["x"] if case["input"] == "rows" else _fp8_rows(s["x"])
    if case["weights"] == "blocks":
        scale = s["scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        w = s["codes"].float() * scale
    else:
        w = _fp8_values((s["codes"], s["exps"]))
    y = torch.matmul(_fp8_values(rows), w.T.contiguous()) + s["bias"]
    if case["epilogue"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y


def _halves(x, e):
    """x as binary16 of x 2^-e."""
    return (x * _pow2(-e)).to(torch.float16).float() * _pow2(e)


def _exponent(amax):
    """The e with amax 2^-e in [2^14, 2^15)."""
    e = torch.frexp(amax)[1] - 15
    return torch.where(amax == 0, 0, e)


def _stored(k, v, seen, kind):
    """The seen tokens of each image in order, zeros behind them, as the type holds them."""
    b, t = k.shape[:2]
    if seen is None:
        lens = torch.full((b,), t, device=DEV, dtype=torch.int32)
    else:
        lens = seen.sum(1, dtype=torch.int32)
        at = torch.sort(seen, dim=1, descending=True, stable=True)[1][..., None, None].expand_as(k)
        there = (torch.arange(t, device=DEV)[None] < lens[:, None])[..., None, None]
        k, v = (torch.where(there, torch.gather(x, 1, at), 0.0) for x in (k, v))
    if kind == "f16":
        k = _halves(k, _exponent(k.abs().amax((1, 3), keepdim=True)))
        v = _halves(v, _exponent(v.abs().amax(1, keepdim=True)))
    return k, v, lens


def _states_plain(s):
    case = s["case"]
    b, t, g, d = case["images"], case["tokens"], case["kv_heads"], case["head_dim"]
    if case["token_major"]:
        k, v = (x.reshape(b, t, g, d) for x in s["rows"].split(g * d, 1))
    else:
        k, v = s["k"].transpose(1, 2), s["v"].transpose(1, 2)
    k, v, lens = _stored(k, v, s["seen"], case["type"])
    return {"k": k.contiguous(), "v": v.contiguous(), "lens": lens}


def _attention_plain(s):
    case = s["case"]
    b, n, t, g, d = (case[x] for x in ("images", "queries", "tokens", "kv_heads", "head_dim"))
    r = case["heads"] // g
    q = s["q"].transpose(1, 2) if case["token_major"] else s["q"]
    q = q.reshape(b, g, r * n, d)  # query heads that share one of K and V together
    x = torch.matmul(q, s["k"].permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(d))
    hidden = torch.arange(t, device=DEV)[None] >= s["lens"][:, None]
    x = x.masked_fill(hidden[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, s["v"].transpose(1, 2).contiguous())
    o = torch.where(total > 0, o / total, 0.0).reshape(b, g * r, n, d)
    return o.transpose(1, 2).contiguous() if case["token_major"] else o


def _write(s):
    case = s["case"]
    if case["token_major"]:
        s["kv"].write_rows(s["rows"], case["tokens"], seen=s["seen"])
    else:
        s["kv"].write(s["k"], s["v"], case["tokens"], seen=s["seen"])


def run(s):
    kind, case = s["kind"], s["case"]
    if not own:
        if kind == "quantise":
            return _fp8_values(_fp8_rows(s["x"]))
        return {"linear": _linear_plain, "states": _states_plain, "attention": _attention_plain}[kind](s)
    if kind == "quantise":
        _rt().quantize_fp8_into(s["x"], case["rows"], case["k"], s["rows"])
        _rt().dequantize_fp8_into(s["rows"], s["out"])
        return s["view"]
    if kind == "linear":
        gelu = case["epilogue"] == "gelu"
        if case["input"] == "rows":
            (s["linear"].run_rows_gelu if gelu else s["linear"].run_rows)(s["rows"], s["out"])
        else:
            (s["linear"].run_gelu if gelu else s["linear"].run)(s["x"], case["rows"], s["out"])
        return s["view"]
    if kind == "states":
        _write(s)
        s["kv"].read(s["k_out"], s["v_out"], s["lens"])
        return {"k": s["k_view"], "v": s["v_view"], "lens": s["lens_view"]}
    s["kv"].attention(s["q"], case["heads"], case["queries"], s["out"], token_major=case["token_major"])
    return s["view"]


# ---- what a pass cannot do without -----------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "quantise":
        values, blocks = case["rows"] * case["k"], case["rows"] * -(-case["k"] // BLOCK)
        # The floats in, the codes written and read back, their values out.
        return {"bytes": 10 * values + 2 * blocks, "flops": 2 * values}
    if kind == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": m * k * (4 if case["input"] == "floats" else 1) + k * n + 4 * m * n + 4 * n,
                "flops": 2 * m * k * n}
    g, d = case["kv_heads"], case["head_dim"]
    kept = sum(_seen_of(case))
    stored = 2 * g * d * kept * (4 if case["type"] == "f32" else 2)
    if kind == "states":
        rows = case["images"] * case["tokens"]
        mask = 0 if case["seen"] == 1.0 and not case["empty"] else 4 * rows
        # The seen rows in, what is stored written and read back, every row's values out.
        return {"bytes": 8 * g * d * kept + mask + 2 * stored + 8 * g * d * rows, "flops": 4 * g * d * kept}
    h, n = case["heads"], case["queries"]
    return {"bytes": stored + 8 * case["images"] * n * h * d, "flops": 4 * n * h * d * kept}


# ---- the definition, in 64 bits ----------------------------------------------------------


def _e4m3(x):
    """x (64 bits) over 2^e rounded to four significand bits, half to even, subnormal below 2^-6: the values
    that the codes of a row stand for."""
    rows, k = x.shape
    out = torch.empty_like(x)
    for at in range(0, k, BLOCK):
        b = x[:, at: at + BLOCK]
        amax = b.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(amax > 0, amax / 448.0, 1.0)))
        e += (amax > 448.0 * torch.exp2(e)).double()  # log2 next to a whole number
        e -= (amax <= 448.0 * torch.exp2(e - 1)).double()
        s = torch.exp2(e.clamp(-127, 127))
        y = b / s
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, at: at + BLOCK] = torch.round(y / step) * step * s
    return out


def _as_halves(x, amax):
    """x in binary16 of x 2^-e with amax 2^-e in [2^14, 2^15)."""
    e = torch.floor(torch.log2(torch.where(amax > 0, amax, 1.0))) - 14
    return (x * torch.exp2(-e)).to(torch.float16).double() * torch.exp2(e)


def _kept(i, image, kind):
    """K and V of an image's seen tokens [n, kv_heads, head_dim], as they are stored."""
    k, v = i["k"][image].double(), i["v"][image].double()
    if i["seen"] is not None:
        at = torch.nonzero(i["seen"][image])[:, 0]
        k, v = k[at], v[at]
    if kind == "f16" and len(k):
        k = _as_halves(k, k.abs().amax((0, 2), keepdim=True))
        v = _as_halves(v, v.abs().amax(0, keepdim=True))
    return k, v


def exact(case, seed):
    kind = case["kind"]
    if kind == "quantise":
        return _e4m3(_quantise_inputs(case, seed)["x"].double())
    if kind == "linear":
        i = _linear_inputs(case, seed)
        if case["weights"] == "blocks":
            n, k = i["codes"].shape
            r, c = torch.arange(n, device=DEV) // BLOCK, torch.arange(k, device=DEV) // BLOCK
            w = i["codes"].double() * i["scales"].double()[r][:, c]
        else:
            w = _e4m3(i["w"].T.double().contiguous())
        y = _e4m3(i["x"].double()) @ w.T.contiguous() + i["bias"].double()
        return y * torch.special.ndtr(y) if case["epilogue"] == "gelu" else y
    i = _attention_inputs(case, seed) if kind == "attention" else _states_inputs(case, seed)
    b, t, g, d = case["images"], case["tokens"], case["kv_heads"], case["head_dim"]
    if kind == "states":
        k, v = (torch.zeros(b, t, g, d, device=DEV, dtype=torch.float64) for _ in range(2))
        for j, n in enumerate(i["lens"]):
            k[j, :n], v[j, :n] = _kept(i, j, case["type"])
        return {"k": k, "v": v, "lens": None}
    out = torch.zeros(b, case["queries"], case["heads"], d, device=DEV, dtype=torch.float64)
    for j, n in enumerate(i["lens"]):
        k, v = _kept(i, j, case["type"])
        for h in range(case["heads"] if n else 0):
            one = h // (case["heads"] // g)
            score = i["q"][j, :, h].double() @ k[:, one].T / math.sqrt(d)
            out[j, :, h] = torch.softmax(score, -1) @ v[:, one]
    return out if case["token_major"] else out.transpose(1, 2).contiguous()
