"""Rotary positions of several axes, the paged cache and its page tables on the GPU,
against float64 numpy (tests/stream64.py)."""
import ctypes

import numpy as np
import pytest

import stream64 as ref
import vestra_hip as vh
from conftest import assert_bits_equal
from vestra_hip import da3, seeded

pytestmark = pytest.mark.gpu


def _pos(seed, tokens, axes, most):
    u = seeded.uniform01(seed, tokens * axes)
    return ((2 * u - 1) * most).astype(np.int32).reshape(tokens, axes)


# ---- rotary positions -----------------------------------------------------------


def _rope(rt, x, pos, pairs, freq, shared, token_major, in_place=False):
    tokens, heads, hd = x.shape
    rope = rt.prepare_rope_axes(hd, pairs, freq, shared=shared)
    src = x if token_major else x.transpose(1, 0, 2)
    xt = rt.upload_f32(src)
    out = xt if in_place else rt.upload_f32(np.full(x.size, 7.0, np.float32))
    rope.run(xt, heads, tokens, rt.upload_i32(pos), out, token_major=token_major)
    got = rt.download_f32(out)
    return got.reshape(tokens, heads, hd) if token_major else got.reshape(heads, tokens, hd).transpose(1, 0, 2)


# x0 c - x1 s in floats: sine and cosine are rounded (2^-24 of each product), then the products, then the sum, half a
# step each: 3 * 2^-24 (|x0| + |x1|) in all.  The angle of position p is off by 3 * 2^-53 p at most on top.
ROPE_TOL = 3.0 * 2.0 ** -24


@pytest.mark.parametrize("tokens, heads, hd, pairs, shared", [
    (1, 1, 4, [1], False), (1, 12, 64, [16, 16], False), (865, 12, 64, [8, 12, 12], False),
    (37, 5, 64, [3, 7, 1, 9], True), (37, 5, 64, [3, 7, 1, 9], False), (130, 3, 40, [5, 6], True),
    (17, 2, 256, [128], False), (9, 7, 96, [10, 11, 12], True), (4100, 2, 32, [5, 5, 6], False),
    (3, 70, 128, [20, 22, 22], True), (50, 1, 12, [2, 1], False)])
@pytest.mark.parametrize("token_major", [False, True])
def test_rope_axes_against_float64(rt, tokens, heads, hd, pairs, shared, token_major):
    x = seeded.normal(tokens + hd, tokens * heads * hd).reshape(tokens, heads, hd)
    pos = _pos(heads + hd, tokens, len(pairs), 100_000)
    got = _rope(rt, x, pos, pairs, 10000.0, shared, token_major)
    exp = ref.rotate(x, pos, pairs, 10000.0, shared)
    # |x0| + |x1| of a pair is at most sqrt(2) times its length, which rotation keeps.
    size = np.abs(x).max(-1, keepdims=True) * 2.0
    assert (np.abs(got - exp) <= ROPE_TOL * size).all()
    turned = 2 * sum(pairs)
    assert_bits_equal(got[..., turned:].ravel(), x[..., turned:].ravel(), "dims past the pairs")


def test_rope_axes_in_place_and_repeated(rt):
    x = seeded.normal(5, 100 * 4 * 64).reshape(100, 4, 64)
    pos = _pos(6, 100, 3, 5000)
    a = _rope(rt, x, pos, [10, 11, 11], 10000.0, True, True)
    b = _rope(rt, x, pos, [10, 11, 11], 10000.0, True, True, in_place=True)
    assert_bits_equal(a.ravel(), b.ravel(), "in place")


def test_rope_axes_of_two_axes_is_rope2d(rt):
    heads, tokens = 12, 865
    x = seeded.normal(7, heads * tokens * 64)
    pos = da3.positions_yx(24, 36)
    a = rt.upload_f32(x)
    rt.rope2d_f32_in_place(a, heads, tokens, 64, pos, 100.0)
    got = _rope(rt, x.reshape(heads, tokens, 64).transpose(1, 0, 2), pos.reshape(-1, 2).astype(np.int32), [16, 16],
                100.0, False, False)
    # rope2d forms its angles in 32 bits: up to 36 rad off by 3 * 2^-24 of themselves (the power of the frequency to
    # a last bit, the product to half of one), on pairs of length below 6.5; and both round as above.
    diff = np.abs(rt.download_f32(a).reshape(heads, tokens, 64).transpose(1, 0, 2) - got).max()
    assert diff <= (36 * 3 * 6.5 + 2 * 3 * 2 * 6.5) * 2.0 ** -24


@pytest.mark.parametrize("far", [0, 1_000_000, -1_000_000, 2**31 - 1, -2**31])
def test_rope_axes_far_positions(rt, far):
    x = seeded.normal(8, 3 * 2 * 64).reshape(3, 2, 64)
    pos = np.full((3, 2), far, np.int32)
    got = _rope(rt, x, pos, [16, 16], 10000.0, False, True)
    exp = ref.rotate(x, pos, [16, 16], 10000.0, False)
    # numpy's own float64 angle is off by 2^-53 of it as well.
    tol = ROPE_TOL + 2 * abs(far) * 2.0 ** -52
    assert (np.abs(got - exp) <= tol * 2 * np.abs(x).max(-1, keepdims=True)).all()


def test_rope_axes_passes_non_finite_values_by_pair(rt):
    x = seeded.normal(9, 2 * 64).reshape(2, 1, 64)
    x[0, 0, 3], x[1, 0, 63] = np.inf, np.nan
    got = _rope(rt, x, np.ones((2, 1), np.int32), [20], 100.0, True, True)
    bad = ~np.isfinite(got)
    exp = np.zeros_like(bad)
    exp[0, 0, [3, 23]], exp[1, 0, 63] = True, True
    assert (bad == exp).all()


def test_rope_axes_of_nothing(rt):
    rope = rt.prepare_rope_axes(64, [16, 16], 100.0)
    e, p = rt.upload_f32(np.zeros(0)), rt.upload_i32(np.zeros(0))
    rope.run(e, 12, 0, p, rt.upload_f32(np.zeros(0)))
    rope.run(e, 0, 5, rt.upload_i32(np.zeros(10)), rt.upload_f32(np.zeros(0)))


# ---- cache -------------------------------------------------------------------------


def _slots(seed, n, total):
    return np.argsort(seeded.uniform01(seed, total), kind="stable")[:n].astype(np.int32)


KINDS = ["f32", "bf16", "q8_0"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens, kvh, hd, page", [(1, 1, 64, 1), (33, 12, 64, 16), (70, 3, 32, 8), (5, 8, 128, 64),
                                                   (130, 2, 96, 4096), (4200, 1, 64, 128)])
@pytest.mark.parametrize("token_major", [False, True])
def test_append_and_gather_are_exact(rt, kind, tokens, kvh, hd, page, token_major):
    pages = -(-tokens // page) + 1
    k, v = (seeded.normal(s + hd, tokens * kvh * hd, 2.0).reshape(tokens, kvh, hd) for s in (1, 2))
    k[0, 0, :32] = 0.0
    if tokens > 1:
        # Of a wide range; the scale of a Q8_0 block stays within binary16.
        k[1, -1, :4] = [8e6, -1e-3, 1e5, -65504.0] if kind == "q8_0" else [1e30, -1e-30, 3e38, -65504.0]
    slots = _slots(tokens, tokens, pages * page)
    slots[tokens // 2] = [-1, pages * page, 2**31 - 1][tokens % 3] if tokens > 1 else slots[0]
    cache = rt.kv_cache(kind, pages, page, kvh, hd)
    assert cache.slots == pages * page
    order = (lambda x: x) if token_major else (lambda x: np.ascontiguousarray(x.transpose(1, 0, 2)))
    cache.append(rt.upload_f32(order(k)), rt.upload_f32(order(v)), tokens, rt.upload_i32(slots), token_major=token_major)
    out = [rt.upload_f32(np.full(tokens * kvh * hd, 9.0)) for _ in range(2)]
    cache.gather(rt.upload_i32(slots), tokens, *out)
    live = ((slots >= 0) & (slots < pages * page))[:, None, None]
    for x, t in zip((k, v), out):
        assert_bits_equal(rt.download_f32(t).ravel() + 0.0, np.where(live, ref.stored(x, kind), 0).ravel() + 0.0, kind)


def test_a_new_cache_holds_zeros_and_unwritten_slots_keep_theirs(rt):
    for kind in KINDS:
        cache = rt.kv_cache(kind, 3, 16, 2, 64)
        out = [rt.upload_f32(np.full(48 * 128, 9.0)) for _ in range(2)]
        every = rt.upload_i32(np.arange(48))
        one = rt.upload_f32(np.ones(128))
        cache.append(one, one, 1, rt.upload_i32([17]))
        cache.gather(every, 48, *out)
        for t in out:
            got = rt.download_f32(t).reshape(48, 128)
            assert (got[17] != 0).all() and (np.delete(got, 17, 0) == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_append_non_finite(rt, kind):
    """Infinities and NaN stay what they are in f32 and bf16; quantize_row_q8_0 has its own rule (NaN to 0)."""
    x = seeded.normal(3, 2 * 64).reshape(2, 64)
    x[0, 5], x[0, 40], x[1, 7] = np.inf, -np.inf, np.nan
    if kind == "q8_0":
        x[0, 5] = x[0, 40] = 1.0
    cache = rt.kv_cache(kind, 1, 2, 1, 64)
    t = rt.upload_f32(x)
    cache.append(t, t, 2, rt.upload_i32([0, 1]), token_major=True)
    k, v = rt.alloc_f32(128), rt.alloc_f32(128)
    cache.gather(rt.upload_i32([0, 1]), 2, k, v)
    got = rt.download_f32(k).reshape(2, 64)
    if kind == "q8_0":
        assert got[1, 7] == 0 and np.isfinite(got).all()
    else:
        assert got[0, 5] == np.inf and got[0, 40] == -np.inf and np.isnan(got[1, 7])
        assert np.isfinite(got).sum() == 125


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens, heads, kvh, hd, pairs, shared", [
    (1, 32, 8, 128, [64], True), (865, 12, 12, 64, [8, 12, 12], False), (37, 9, 3, 96, [10, 11, 12], True),
    (20, 8, 1, 32, [], False), (2500, 4, 2, 64, [15, 16], False)])
def test_append_qkv_equals_its_parts(rt, kind, tokens, heads, kvh, hd, pairs, shared):
    rows = seeded.normal(tokens + heads, tokens * (heads + 2 * kvh) * hd).reshape(tokens, heads + 2 * kvh, hd)
    pos = _pos(3, tokens, max(1, len(pairs)), 3000)
    slots = _slots(4, tokens, 2 * tokens + 64)
    slots[tokens // 3] = -1
    p, at = rt.upload_i32(pos), rt.upload_i32(slots)
    a, b = (rt.kv_cache(kind, tokens * 2 // 32 + 2, 32, kvh, hd) for _ in range(2))
    q = rt.alloc_f32(tokens * heads * hd)
    rope = rt.prepare_rope_axes(hd, pairs, 10000.0, shared=shared) if pairs else None
    a.append_qkv(rt.upload_f32(rows), heads, tokens, at, q, rope=rope, positions=p if pairs else None)

    def turned(x):
        if not pairs:
            return x
        t = rt.upload_f32(np.ascontiguousarray(x))
        rope.run(t, x.shape[1], tokens, p, t, token_major=True)
        return rt.download_f32(t).reshape(x.shape)

    qe, ke = turned(rows[:, :heads]), turned(rows[:, heads:heads + kvh])
    assert_bits_equal(rt.download_f32(q), np.ascontiguousarray(qe).ravel(), "q")
    b.append(rt.upload_f32(ke), rt.upload_f32(rows[:, heads + kvh:]), tokens, at, token_major=True)
    for cache in (a, b):
        cache.got = [rt.alloc_f32(tokens * kvh * hd) for _ in range(2)]
        cache.gather(at, tokens, *cache.got)
    for x, y, name in zip(a.got, b.got, "kv"):
        assert_bits_equal(rt.download_f32(x), rt.download_f32(y), name)
    exp = ref.stored(rows[:, heads + kvh:], kind)
    exp[(slots < 0) | (slots >= a.slots)] = 0
    assert_bits_equal(rt.download_f32(a.got[1]) + 0.0, exp.ravel() + 0.0, "v against numpy")


def _tiled(rt, n, piece):
    """n floats on the device that repeat `piece`."""
    t, p = rt.alloc_f32(n), rt.upload_f32(piece)
    for at in range(0, n, piece.size):
        rt.copy_segment_into_f32(t, at, p, 0, min(piece.size, n - at))
    return t


def test_rows_past_4_gib(rt):
    """Tensors whose bytes pass 2^32: the last tokens of a rotation in place, and of an append from QKV rows."""
    hd, tokens, tail = 64, (1 << 24) + 35, 700
    rope = rt.prepare_rope_axes(hd, [30], 10000.0, shared=True)
    piece = seeded.normal(21, (1 << 20) * hd)
    x = _tiled(rt, tokens * hd, piece)
    pos = np.arange(tokens) % 5000
    rope.run(x, 1, tokens, rt.upload_i32(pos), x)
    rows = np.arange(tokens - tail, tokens)
    src = piece.reshape(-1, 1, hd)[rows % (1 << 20)]
    exp = ref.rotate(src, pos[rows, None], [30], 10000.0, True)
    got = rt.download_f32(rt.copy_segment_f32(x, (tokens - tail) * hd, tail * hd)).reshape(exp.shape)
    assert (np.abs(got - exp) <= ROPE_TOL * 2 * np.abs(src).max(-1, keepdims=True)).all()
    del x

    heads, kvh, tokens = 12, 2, (1 << 20) + 35
    width = (heads + 2 * kvh) * hd
    piece = seeded.normal(22, (1 << 15) * width)
    qkv, q = _tiled(rt, tokens * width, piece), rt.alloc_f32(tokens * heads * hd)
    cache = rt.kv_cache("f32", 8, 128, kvh, hd)
    slots = np.full(tokens, -1)
    slots[-tail:] = _slots(3, tail, 1024)
    cache.append_qkv(qkv, heads, tokens, rt.upload_i32(slots), q)
    rows = np.arange(tokens - tail, tokens)
    exp = piece.reshape(-1, heads + 2 * kvh, hd)[rows % (1 << 15)]
    got = rt.download_f32(rt.copy_segment_f32(q, (tokens - tail) * heads * hd, tail * heads * hd))
    assert_bits_equal(got, exp[:, :heads].ravel(), "q")
    k, v = rt.alloc_f32(tail * kvh * hd), rt.alloc_f32(tail * kvh * hd)
    cache.gather(rt.upload_i32(slots[-tail:]), tail, k, v)
    assert_bits_equal(rt.download_f32(k), exp[:, heads:heads + kvh].ravel(), "k")
    assert_bits_equal(rt.download_f32(v), exp[:, heads + kvh:].ravel(), "v")


# ---- page tables ---------------------------------------------------------------------


def _assign(rt, cached, added, free, free_start, page, table, tokens):
    r = len(cached)
    table_t = rt.upload_i32(table)
    out = {"starts": rt.alloc_i32(r + 1), "lens": rt.alloc_i32(r), "slots": rt.alloc_i32(tokens),
           "free_next": rt.alloc_i32(1)}
    rt.kv_pages_assign(rt.upload_i32(cached), rt.upload_i32(added), rt.upload_i32(free), rt.upload_i32([free_start]),
                       page, table_t, np.shape(table)[1], out["starts"], out["lens"], out["slots"], out["free_next"])
    return (*(rt.download_i32(out[k]) for k in ("starts", "lens", "slots")),
            rt.download_i32(table_t).reshape(np.shape(table)), int(rt.download_i32(out["free_next"])[0]))


def _same(got, exp):
    for name, a, b in zip(("starts", "lens", "slots", "table", "free_next"), got, exp):
        assert np.array_equal(a, b), (name, a, b)


@pytest.mark.parametrize("requests, page, most_new, most_cached, spare", [
    (1, 1, 1, 0, 0), (1, 16, 100, 50, 3), (7, 64, 1, 500, 0), (300, 16, 40, 100, 11), (1000, 32, 5, 900, 0),
    (4096, 4, 3, 20, 1), (3, 4096, 9000, 5000, 1000)])
def test_pages_against_a_walk(rt, requests, page, most_new, most_cached, spare):
    u = seeded.uniform01(requests, 2 * requests)
    cached, added = (u[:requests] * (most_cached + 1)).astype(int), (u[requests:] * (most_new + 1)).astype(int)
    held = -(-cached // page)
    need = -(-(cached + added) // page)
    order = _slots(9, need.sum() + 5, need.sum() + 5)
    table = np.full((requests, need.max() + 1), -1, np.int32)
    at = 0
    for r in range(requests):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    free = np.concatenate([[-7, -7], order[at:]])
    args = (cached, added, free, 2, page, table, int(added.sum()) + spare)
    _same(_assign(rt, *args), ref.pages(*args))


@pytest.mark.parametrize("case", ["no requests", "all empty", "list ends", "row ends", "batch too small", "negative",
                                  "free start past the list", "negative free start", "page too far", "no free list"])
def test_pages_at_the_edges(rt, case):
    cached, added, free, start, page = [5, 0, 17], [4, 20, 1], np.arange(100, 120), 0, 8
    table = np.full((3, 5), -1)
    table[0, 0], table[2, :3] = 1, [2, 3, 4]
    tokens = 30
    if case == "no requests":
        cached, added, table = [], [], np.zeros((0, 5), int)
    elif case == "all empty":
        added = [0, 0, 0]
    elif case == "list ends":
        free = free[:2]
    elif case == "row ends":
        table = table[:, :3]
        added = [4, 30, 1]
        tokens = 40
    elif case == "batch too small":
        tokens = 11
    elif case == "negative":
        cached, added = [5, -3, 17], [-4, 20, 1]
    elif case == "free start past the list":
        start = 2**31 - 2
    elif case == "negative free start":
        start = -2
    elif case == "page too far":
        free = np.array([2**31 - 1, 2**28 + 1, 2**28 - 2, 7, 8, 9])
    elif case == "no free list":
        free = np.zeros(0, int)
    got = _assign(rt, cached, added, free, start, page, table, tokens)
    starts, lens, slots, tab, nxt = ref.pages(cached, added, free, start, page, table, tokens)
    # A slot past 2^31 does not exist.
    slots = np.where(slots >= 2**31 - page, -1, slots)
    _same(got, (starts, lens, slots, tab, min(nxt, 2**31 - 1)))


def test_pages_step_by_step(rt):
    """Three steps whose outputs are the next one's inputs, against the same tokens in one."""
    requests, page, width = 5, 8, 12
    free = _slots(3, 60, 60)
    new = [[9, 0, 16, 1, 30], [1, 1, 1, 1, 1], [7, 20, 8, 0, 3]]
    cached, start = rt.upload_i32([0] * requests), rt.upload_i32([0])
    table = rt.upload_i32(np.full(requests * width, -1))
    seen = [[] for _ in range(requests)]
    for n in new:
        starts, lens, slots, nxt = rt.alloc_i32(requests + 1), rt.alloc_i32(requests), rt.alloc_i32(70), rt.alloc_i32(1)
        rt.kv_pages_assign(cached, rt.upload_i32(n), rt.upload_i32(free), start, page, table, width, starts, lens, slots,
                           nxt)
        s, at = rt.download_i32(slots), rt.download_i32(starts)
        for r in range(requests):
            seen[r] += list(s[at[r]:at[r + 1]])
        assert (s[at[-1]:] == -1).all()
        cached, start = lens, nxt
    total = np.sum(new, 0)
    assert np.array_equal(rt.download_i32(cached), total)
    tab = rt.download_i32(table).reshape(requests, width)
    every = sum(seen, [])
    assert len(set(every)) == len(every) == total.sum()
    for r in range(requests):
        assert seen[r] == [tab[r, p // page] * page + p % page for p in range(total[r])]


# ---- refusals ------------------------------------------------------------------------


def test_index_round_trip_and_refusals(rt):
    i = rt.upload_i32([1, -2, 2**31 - 1])
    assert len(i) == 3 and i.device_ptr and list(rt.download_i32(i)) == [1, -2, 2**31 - 1]
    assert len(rt.upload_i32([])) == 0
    with pytest.raises(vh.LengthMismatch):
        vh._check(vh.lib().vh_download_i32(rt.handle, i.handle, (ctypes.c_int * 2)(), 2))
    other = vh.Runtime(0)
    with pytest.raises(vh.InvalidArgument):
        other.download_i32(i)


@pytest.mark.parametrize("hd, pairs, freq", [(0, [1], 1.0), (6, [1], 1.0), (260, [1], 1.0), (64, [], 1.0),
                                             (64, [1] * 5, 1.0), (64, [0, 4], 1.0), (64, [16, 17], 1.0),
                                             (64, [2**63, 2**63], 1.0), (64, [4], 0.0), (64, [4], -1.0),
                                             (64, [4], np.inf), (64, [4], np.nan)])
def test_rope_axes_refuses(rt, hd, pairs, freq):
    with pytest.raises(vh.KernelError):
        rt.prepare_rope_axes(hd, pairs, freq)


def test_rope_axes_run_refuses(rt):
    rope = rt.prepare_rope_axes(64, [16, 16], 100.0)
    x, p = rt.alloc_f32(3 * 64), rt.upload_i32(np.zeros(6))
    for bad in (lambda: rope.run(x, 2, 3, p, x), lambda: rope.run(x, 1, 3, p, rt.alloc_f32(64)),
                lambda: rope.run(x, 1, 3, rt.upload_i32(np.zeros(5)), x),
                lambda: rope.run(x, 2**62, 2**62, p, x)):
        with pytest.raises(vh.LengthMismatch):
            bad()
    other = vh.Runtime(0)
    for bad in (lambda: rope.run(other.alloc_f32(192), 1, 3, p, x), lambda: rope.run(x, 1, 3, p, other.alloc_f32(192)),
                lambda: rope.run(x, 1, 3, other.upload_i32(np.zeros(6)), x)):
        with pytest.raises(vh.InvalidArgument):
            bad()


@pytest.mark.parametrize("kind, pages, page, kvh, hd", [
    ("f16", 1, 16, 1, 64), ("f32", 1, 0, 1, 64), ("f32", 1, 24, 1, 64), ("f32", 1, 8192, 1, 64), ("f32", 1, 16, 0, 64),
    ("f32", 1, 16, 70000, 64), ("f32", 1, 16, 1, 0), ("f32", 1, 16, 1, 6), ("f32", 1, 16, 1, 132),
    ("q8_0", 1, 16, 1, 36), ("f32", 2**27, 16, 1, 64), ("f32", 2**60, 16, 1, 64), ("f32", 2**64 - 1, 4096, 65535, 64)])
def test_cache_refuses(rt, kind, pages, page, kvh, hd):
    with pytest.raises(vh.KernelError):
        rt.kv_cache(kind, pages, page, kvh, hd)


def test_append_and_gather_refuse(rt):
    cache = rt.kv_cache("f32", 2, 16, 2, 64)
    x, y, z, s = rt.alloc_f32(3 * 128), rt.alloc_f32(3 * 128), rt.alloc_f32(4 * 128), rt.upload_i32([0, 1, 2])
    rope, p = rt.prepare_rope_axes(64, [16], 100.0), rt.upload_i32([0, 1, 2])
    qkv, q = rt.alloc_f32(3 * 8 * 64), rt.alloc_f32(3 * 4 * 64)
    for bad in (lambda: cache.append(z, x, 3, s), lambda: cache.append(x, z, 3, s), lambda: cache.append(z, z, 4, s),
                lambda: cache.append(x, x, 2**60, s), lambda: cache.gather(s, 3, z, y), lambda: cache.gather(s, 3, x, z),
                lambda: cache.gather(s, 4, z, rt.alloc_f32(4 * 128)), lambda: cache.append_qkv(qkv, 4, 4, s, q),
                lambda: cache.append_qkv(qkv, 4, 3, s, x), lambda: cache.append_qkv(qkv, 4, 3, rt.upload_i32([0]), q),
                lambda: cache.append_qkv(qkv, 4, 3, s, q, rope=rope, positions=rt.upload_i32([0, 1]))):
        with pytest.raises(vh.LengthMismatch):
            bad()
    for bad in (lambda: cache.append_qkv(qkv, 3, 3, s, q), lambda: cache.append_qkv(qkv, 0, 3, s, q),
                lambda: cache.append_qkv(qkv, 4, 3, s, q, rope=rt.prepare_rope_axes(32, [8], 1.0), positions=p)):
        with pytest.raises(vh.KernelError):
            bad()
    other = vh.Runtime(0)
    ox, os = other.alloc_f32(3 * 128), other.upload_i32([0, 1, 2])
    for bad in (lambda: cache.append(ox, x, 3, s), lambda: cache.append(x, ox, 3, s), lambda: cache.append(x, x, 3, os),
                lambda: cache.gather(s, 3, ox, x), lambda: cache.gather(os, 3, x, y), lambda: cache.gather(s, 3, x, x),
                lambda: cache.append_qkv(qkv, 4, 3, os, q),
                lambda: cache.append_qkv(qkv, 4, 3, s, q, rope=rope),
                lambda: cache.append_qkv(qkv, 4, 3, s, q, rope=rope, positions=os)):
        with pytest.raises(vh.InvalidArgument):
            bad()
    square = rt.kv_cache("f32", 1, 16, 1, 64)
    with pytest.raises(vh.LengthMismatch):
        square.append_qkv(qkv, 6, 3, s, qkv)
    with pytest.raises(vh.InvalidArgument):
        vh._check(vh.lib().vh_kv_cache_append_f32(None, x.handle, x.handle, 3, 0, s.handle))


def test_pages_refuse(rt):
    def call(over=None, **kw):
        rt_ = rt
        a = {"cached": rt.upload_i32([0, 0]), "added": rt.upload_i32([1, 1]), "free": rt.upload_i32([0, 1]),
             "free_start": rt.upload_i32([0]), "page": 16, "table": rt.alloc_i32(6), "max_pages": 3,
             "starts": rt.alloc_i32(3), "lens": rt.alloc_i32(2), "slots": rt.alloc_i32(2), "free_next": rt.alloc_i32(1)}
        a |= kw
        a |= over(a) if over else {}
        rt_.kv_pages_assign(*a.values())

    call()
    for name, n in (("added", 3), ("free_start", 2), ("table", 7), ("starts", 2), ("lens", 3), ("free_next", 2)):
        with pytest.raises(vh.LengthMismatch):
            call(**{name: rt.alloc_i32(n)})
    for page in (0, 3, 8192):
        with pytest.raises(vh.KernelError):
            call(page=page)
    with pytest.raises(vh.KernelError):
        n = 4097
        call(cached=rt.alloc_i32(n), added=rt.alloc_i32(n), table=rt.alloc_i32(3 * n), starts=rt.alloc_i32(n + 1),
             lens=rt.alloc_i32(n))
    for over in (lambda a: {"lens": a["cached"]}, lambda a: {"free_next": a["free_start"]},
                 lambda a: {"slots": a["lens"]}, lambda a: {"slots": a["added"]}):
        with pytest.raises(vh.InvalidArgument):
            call(over)
    other = vh.Runtime(0)
    for name in ("cached", "lens"):
        with pytest.raises(vh.InvalidArgument):
            call(**{name: other.alloc_i32(2)})
