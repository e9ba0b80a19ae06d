"""The operators of a stream at their edges, where a call is legal and its values unusual: against float64 numpy
(tests/stream64.py)."""
import numpy as np
import pytest

import stream64 as ref
import vestra_hip as vh
from conftest import assert_bits_equal
from test_gpu_stream_attention import KINDS, Stream, close
from vestra_hip import seeded

pytestmark = pytest.mark.gpu


# ---- requests that outgrow their row of the table ------------------------------------


def _cut(s, columns):
    """The table's first columns; which keys lie behind them."""
    s.width, s.table = columns, np.ascontiguousarray(s.table[:, :columns])
    return [np.arange(n) >= columns * s.page for n in s.lens]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, lens, columns, heads, kvh, hd", [
    ([4, 1, 2], [50, 49, 20], 3, 4, 2, 64), ([10, 1], [70, 300], 4, 2, 2, 128),
    ([200, 90], [260, 100], 12, 4, 2, 64), ([150, 140], [700, 300], 20, 4, 1, 128)])
@pytest.mark.parametrize("block, window", [(1, 0), (50, 0), (1, 20), (0, 30), (16, 100)])
def test_a_request_past_its_row_keeps_its_positions(rt, kind, new, lens, columns, heads, kvh, hd, block, window):
    """Positions, blocks and windows follow from lens; only the keys that the row cannot hold are missing."""
    s = Stream(rt, kind, new, lens, heads, kvh, hd, 16, spare_rows=1)
    s.check(block, window, absent=_cut(s, columns))


@pytest.mark.parametrize("new", [3, 300])
def test_the_longest_length_of_a_short_row(rt, new):
    """A length of 2^31 - 1 over a row of 64 tokens: every key for a late position, none in a window at its end."""
    s = Stream(rt, "f32", [new], [64], 2, 1, 64, 16)
    _cut(s, 4)
    exp = s.run(0)
    s.lens = np.array([2**31 - 1])
    for block in (0, 1, 865, 2**31, 2**40):
        assert_bits_equal(s.run(block).ravel(), exp.ravel(), f"block {block}")
    for block in (0, 1, 865):
        assert (s.run(block, window=1000) == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [1, 10])
def test_a_step_past_the_row_of_a_table(rt, kind, block):
    """Tables, appends and attention of a step whose first request outgrows its row of 64 tokens and whose second does
    not: the tokens that found a place see themselves."""
    heads, kvh, hd, page, width, had, new = 4, 2, 64, 16, 4, [60, 5], [10, 3]
    cache = rt.kv_cache(kind, 12, page, kvh, hd)
    table = rt.upload_i32(np.full(2 * width, -1))
    free, cached, start = rt.upload_i32([7, 3, 9, 0, 11, 5, 2]), rt.upload_i32([0, 0]), rt.upload_i32([0])
    ks, vs = ([seeded.normal(s + r, (a + b) * kvh * hd).reshape(-1, kvh, hd) for r, (a, b) in enumerate(zip(had, new))]
              for s in (1, 11))
    q = seeded.normal(5, sum(new) * heads * hd).reshape(-1, heads, hd)
    for step, n in enumerate((had, new)):
        starts, lens, slots, nxt = rt.alloc_i32(3), rt.alloc_i32(2), rt.alloc_i32(sum(n)), rt.alloc_i32(1)
        rt.kv_pages_assign(cached, rt.upload_i32(n), free, start, page, table, width, starts, lens, slots, nxt)
        rows = [np.concatenate([x[a * step:a * step + b] for x, a, b in zip(xs, had, n)]) for xs in (ks, vs)]
        cache.append(rt.upload_f32(rows[0]), rt.upload_f32(rows[1]), sum(n), slots, token_major=True)
        cached, start = lens, nxt
    assert list(rt.download_i32(slots)[:10] >= 0) == [True] * 4 + [False] * 6
    out = rt.alloc_f32(q.size)
    cache.attention(rt.upload_f32(q), heads, sum(new), table, width, starts, lens, out, block=block)
    lens = rt.download_i32(lens)
    args = (q, [ref.stored(k, kind) for k in ks], [ref.stored(v, kind) for v in vs], rt.download_i32(starts), lens,
            heads, block, 0, [np.arange(n) >= width * page for n in lens])
    close(rt.download_f32(out).reshape(q.shape), ref.attention(*args), ref.attention(*args, dtype=np.float32))


# ---- starts that fall ---------------------------------------------------------------


def _walk_of_starts(case, requests, tokens):
    u = seeded.uniform01(requests + tokens, requests + 1)
    if case == "up and down":
        return (u * (tokens + 1)).astype(int)
    if case == "all of it again":
        return np.tile([0, tokens], requests)[:requests + 1]
    # Rising, with a fall in one place of every hundred.
    rise = np.linspace(0, tokens, requests + 1).astype(int)
    return np.where(u < 0.01, (rise * u * 100).astype(int), rise)


@pytest.mark.parametrize("kind, heads, kvh", [("f32", 2, 2), ("bf16", 8, 1), ("q8_0", 4, 2)])
@pytest.mark.parametrize("case, requests, tokens", [
    ([50, 100, 50, 100, 50, 100, 0, 50], 7, 100), ([0, 90, 0, 90, 0, 100], 5, 100), ([0, 400, 100, 390, 200, 900], 5, 900),
    ([-7, 3, 2**31 - 1, -2**31, 50], 4, 60), ([60, 40, 20, 0], 3, 60), ("up and down", 40, 700),
    ("all of it again", 301, 64), ("rising", 600, 700), ("rising", 1200, 9000)])
def test_a_start_that_falls_counts_as_the_highest_before_it(rt, kind, heads, kvh, case, requests, tokens):
    """Each row is one request's, or none's: of the rows that two requests name the first one's, at the position that
    its distance from the request's end gives; rows before the first start and behind the last stay as they were."""
    starts = np.array(case) if isinstance(case, list) else _walk_of_starts(case, requests, tokens)
    lens = [20 + int(60 * u) for u in seeded.uniform01(requests, requests)]
    s = Stream(rt, kind, [0] * requests, lens, heads, kvh, 64, 16, spare_rows=tokens)
    s.starts = starts
    high = np.maximum.accumulate(np.clip(starts, 0, tokens))
    for block, window in ((1, 0), (0, 17)):
        got = s.run(block, window, fill=7.0)
        args = (s.q, s.k, s.v, high, s.lens, heads, block, window)
        lo, hi = high[0], high[-1]
        close(got[lo:hi], ref.attention(*args)[lo:hi], ref.attention(*args, dtype=np.float32)[lo:hi])
        assert (got[:lo] == 7.0).all() and (got[hi:] == 7.0).all()
        assert_bits_equal(s.run(block, window, fill=7.0).ravel(), got.ravel(), "again")


# ---- values near the largest ------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("requests, new, heads, hd", [(128, 1, 8, 64), (128, 1, 8, 128), (32, 40, 16, 64),
                                                      (32, 40, 16, 128)])
@pytest.mark.parametrize("rise", [7.9, 8.1])
def test_large_values_of_a_score_that_rises_late(rt, kind, requests, new, heads, hd, rise):
    """Flat scores and, steps later, one key whose score passes them by about 8 (base 2), all values at the size up to
    which rows are finite.  Enough tiles that a workgroup has several steps of each."""
    n = 300
    size = 2.0 ** 120 / n

    def change(r, k, v):
        k[:] = 0
        k[280, :, 0] = rise * np.log(2.0) * np.sqrt(hd)
        v[:] = np.clip(v, -1, 1) * np.float32(size) * np.float32(0.99)  # (of what bf16 makes of it)
        v[280] = np.float32(size * 0.99)

    s = Stream(rt, kind, [new] * requests, [n] * requests, heads, heads, hd, 16, change=change)
    s.q[:] = 0
    s.q[..., 0] = 1
    got = s.run(0)
    args = (s.q, s.k, s.v, s.starts, s.lens, heads)
    exp, plain = ref.attention(*args), ref.attention(*args, dtype=np.float32)
    assert np.isfinite(plain).all()
    close(got, exp, plain)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("exponent", [-100, -110, -118, -126])
def test_small_values_keep_what_they_have(rt, kind, new, exponent):
    """Values near the smallest: off by no more than the parts below 2^-126 that count as zero."""

    def change(r, k, v):
        v *= np.float32(2.0) ** np.float32(exponent)

    Stream(rt, kind, [new], [333], 4, 2, 64, 16, change=change).check(1)


# ---- limits -------------------------------------------------------------------------------


def test_calls_of_more_than_2_27_tokens_are_refused(rt):
    n = (1 << 27) + 1
    cache, slots = rt.kv_cache("bf16", 1, 16, 1, 4), rt.alloc_i32(n)
    k, v = rt.alloc_f32(4 * n), rt.alloc_f32(4 * n)
    rope = rt.prepare_rope_axes(4, [1], 100.0)
    for call in (lambda: cache.gather(slots, n, k, v), lambda: cache.append(k, v, n, slots),
                 lambda: rope.run(k, 1, n, slots, v)):
        with pytest.raises(vh.KernelError, match="2\\^27 tokens"):
            call()


def test_page_tables_say_how_many_tokens_they_take(rt):
    """2^31 - 1025 tokens; one more is refused, with that number."""
    one, two, slots = rt.upload_i32([0]), rt.alloc_i32(2), rt.alloc_i32(2**31 - 1024)
    with pytest.raises(vh.KernelError, match="2\\^31 - 1025 tokens"):
        rt.kv_pages_assign(one, rt.upload_i32([1]), rt.upload_i32([0]), rt.upload_i32([0]), 16, rt.alloc_i32(4), 4, two,
                           rt.alloc_i32(1), slots, rt.alloc_i32(1))


# ---- appends that pass by the caches ----------------------------------------------------------


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("token_major", [False, True])
def test_appends_past_the_caches_are_exact(rt, kind, token_major):
    tokens, kvh, hd, page = 16501, 24, 64, 32  # 203 MB
    k, v = (seeded.normal(s, tokens * kvh * hd).reshape(tokens, kvh, hd) for s in (1, 2))
    pages = -(-tokens // page)
    slots = np.argsort(seeded.uniform01(3, pages * page), kind="stable")[:tokens]
    cache = rt.kv_cache(kind, pages, page, kvh, hd)
    given = [rt.upload_f32(x if token_major else np.ascontiguousarray(x.transpose(1, 0, 2))) for x in (k, v)]
    at = rt.upload_i32(slots)
    cache.append(*given, tokens, at, token_major=token_major)
    out = [rt.alloc_f32(tokens * kvh * hd) for _ in range(2)]
    cache.gather(at, tokens, *out)
    for x, t in zip((k, v), out):
        assert_bits_equal(rt.download_f32(t) + 0.0, ref.stored(x, kind).ravel() + 0.0, kind)


# ---- pages past a row -----------------------------------------------------------------------


def test_pages_past_a_row_are_those_that_no_row_has(rt):
    """A request past its row takes pages that the table cannot hold.  They are what the step took less what the rows
    have; given back they serve the next request."""
    page, width, free = 8, 3, np.array([40, 41, 42, 43, 44, 45, 46, 47])
    table = np.full((3, width), -1)
    table[0, :3], table[1, :1] = [1, 2, 3], [4]
    cached, added = [20, 8, 0], [25, 6, 9]
    t, starts, lens = rt.upload_i32(table), rt.alloc_i32(4), rt.alloc_i32(3)
    slots, nxt = rt.alloc_i32(sum(added)), rt.alloc_i32(1)
    rt.kv_pages_assign(rt.upload_i32(cached), rt.upload_i32(added), rt.upload_i32(free), rt.upload_i32([1]), page, t,
                       width, starts, lens, slots, nxt)
    got, taken = rt.download_i32(t).reshape(3, width), free[1:int(rt.download_i32(nxt)[0])]
    assert list(taken) == [41, 42, 43, 44, 45, 46] and got.tolist() == [[1, 2, 3], [4, 44, -1], [45, 46, -1]]
    assert list(np.setdiff1d(taken, got)) == [41, 42, 43]
    s = rt.download_i32(slots)
    assert (s[4:25] == -1).all() and list(s[:4]) == [28, 29, 30, 31] and (s[25:] >= 0).all()


# ---- a batch in two calls -------------------------------------------------------------------


@pytest.mark.parametrize("kind", KINDS)
def test_a_batch_in_two_calls(rt, kind):
    """A chunk and single tokens over the same queries and output, each call with its own requests: they are those of
    the batch, and neither call writes the other's rows."""
    s = Stream(rt, kind, [300] + [1] * 20, [500] + list(range(40, 60)), 8, 2, 64, 16, spare_rows=3)
    q, both = rt.upload_f32(s.q), rt.upload_f32(np.full(s.q.size, 7.0))
    got = []
    for requests in (slice(0, 1), slice(1, 21)):
        starts = s.starts[requests.start:requests.stop + 1]
        args = (q, 8, s.tokens, rt.upload_i32(s.table[requests]), s.width, rt.upload_i32(starts),
                rt.upload_i32(s.lens[requests]))
        out = rt.upload_f32(np.full(s.q.size, 7.0))
        for t in (out, both):
            s.cache.attention(*args, t, block=1)
        got.append(rt.download_f32(out).reshape(s.q.shape))
        rows = np.r_[0:starts[0], starts[-1]:s.tokens]
        assert (got[-1][rows] == 7.0).all()
    assert_bits_equal(rt.download_f32(both)[:-3 * 512], np.concatenate([got[0][:300], got[1][300:320]]).ravel(), "both")
    args = (s.q, s.k, s.v, s.starts, s.lens, 8, 1)
    close(rt.download_f32(both).reshape(s.q.shape)[:320], ref.attention(*args)[:320],
          ref.attention(*args, dtype=np.float32)[:320])
