"""Attention over the paged cache on the GPU, against float64 numpy (tests/stream64.py)."""
import numpy as np
import pytest

import stream64 as ref
import vestra_hip as vh
from conftest import assert_bits_equal
from vestra_hip import seeded

pytestmark = pytest.mark.gpu

KINDS = ["f32", "bf16", "q8_0"]


class Stream:
    """A cache that holds the requests' keys and values in scattered pages, and the tables of a step."""

    def __init__(self, rt, kind, new, lens, heads, kvh, hd, page, seed=1, spare_rows=0, std=1.0, change=None):
        self.rt, self.heads, self.kvh, self.hd, self.page = rt, heads, kvh, hd, page
        self.new, self.lens = np.array(new), np.array(lens)
        self.starts = np.concatenate([[0], np.cumsum(new)])
        self.tokens = int(self.starts[-1]) + spare_rows
        held = [-(-n // page) for n in lens]
        pages = sum(held) + 3
        order = np.argsort(seeded.uniform01(seed + 50, pages), kind="stable")
        self.width = max(held + [1]) + 1
        self.table = np.full((len(lens), self.width), -1, np.int64)
        self.cache = rt.kv_cache(kind, pages, page, kvh, hd)
        self.q = seeded.normal(seed, max(1, self.tokens) * heads * hd, std).reshape(-1, heads, hd)[:self.tokens]
        self.k, self.v, at = [], [], 0
        # What earlier requests left in the pages.
        if pages * page * kvh * hd <= 1 << 22:
            junk = rt.upload_f32(np.full(pages * page * kvh * hd, np.nan if kind != "q8_0" else 1e30))
            self.cache.append(junk, junk, pages * page, rt.upload_i32(np.arange(pages * page)))
        for r, n in enumerate(lens):
            self.table[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
            k, v = (seeded.normal(seed + 7 * r + s, max(1, n) * kvh * hd).reshape(-1, kvh, hd)[:n] for s in (2, 3))
            if change is not None:
                change(r, k, v)
            if n:
                j = np.arange(n)
                slots = self.table[r, j // page] * page + j % page
                self.cache.append(rt.upload_f32(k), rt.upload_f32(v), n, rt.upload_i32(slots), token_major=True)
            self.k.append(ref.stored(k, kind) if n else k)
            self.v.append(ref.stored(v, kind) if n else v)

    def run(self, block=0, window=0, fill=np.nan, table=None, **kw):
        out = self.rt.upload_f32(np.full(self.q.size, fill, np.float32))
        self.cache.attention(self.rt.upload_f32(self.q), self.heads, self.tokens,
                             self.rt.upload_i32(self.table if table is None else table), self.width,
                             self.rt.upload_i32(self.starts), self.rt.upload_i32(self.lens), out, block=block,
                             window=window, **kw)
        return self.rt.download_f32(out).reshape(self.q.shape)

    def check(self, block=0, window=0, absent=None, table=None, **kw):
        got = self.run(block, window, table=table, **kw)
        args = (self.q, self.k, self.v, self.starts, self.lens, self.heads, block, window, absent)
        exp = ref.attention(*args)
        n = int(self.starts[-1])
        assert np.isnan(got[n:]).all(), "rows behind the last request"
        close(got[:n], exp[:n], ref.attention(*args, dtype=np.float32)[:n])
        return got


def close(got, exp, plain):
    """Within twice the 2-norm error of the same formula in float32 numpy and four roundings; not finite where that is
    NaN, anything where it is infinite."""
    wrong = np.isfinite(got) != ~np.isnan(exp)
    assert not (wrong & ~np.isinf(exp)).any(), np.argwhere(wrong & ~np.isinf(exp))[:5]
    f = np.isfinite(exp)
    got, exp, plain = (x[f].astype(np.float64) for x in (got, exp, plain))
    if not exp.size:
        return
    norm = np.linalg.norm(exp)
    err, own = np.linalg.norm(got - exp), np.linalg.norm(plain - exp)
    print(f"error {err / max(norm, 1e-300):.2e}, float32 {own / max(norm, 1e-300):.2e}")
    # The matrix instructions take a bf16 part below 2^-126 for zero.  A float has two parts behind its first, so each
    # value is off by less than 2 * 2^-126 there, and an average of values (weights that sum to one) by no more.
    tiny = 2.0 ** -125
    assert err <= 2 * own + 4 * 2.0 ** -24 * norm + tiny * np.sqrt(exp.size), (err, own, norm)
    # No single value is far off either: 40 such errors of the root mean square.
    rms = norm / np.sqrt(exp.size)
    tol = 40 * (2 * own / np.sqrt(exp.size) + 2.0 ** -22 * rms) + tiny
    worst = np.abs(got - exp) / np.maximum(1.0, np.abs(exp) / rms)
    assert worst.max() <= tol, (worst.max(), tol)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, lens, heads, kvh, hd, page, block, window", [
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([1], [2], 12, 12, 64, 1, 1, 0),
    ([1], [865], 12, 12, 64, 64, 0, 0),
    ([1], [5000], 2, 1, 128, 32, 1, 0),
    ([1, 1, 1], [1, 63, 64], 8, 2, 64, 16, 1, 0),
    ([1, 1, 1, 1, 1], [65, 127, 1024, 33, 700], 32, 8, 128, 64, 1, 0),
    ([1] * 40, list(range(30, 70)), 4, 4, 64, 8, 1, 0),
    ([4, 1, 3], [100, 40, 333], 9, 3, 96, 16, 1, 0),
    ([2, 2], [300, 301], 6, 6, 32, 256, 1, 37),
    ([7], [7], 3, 3, 64, 16, 1, 0),
    ([130], [130], 4, 2, 64, 32, 1, 0),
    ([129], [640], 2, 2, 128, 16, 1, 100),
    ([300], [901], 3, 3, 64, 128, 100, 0),
    ([300], [901], 3, 3, 64, 128, 100, 250),
    ([257], [777], 2, 1, 64, 64, 0, 0),
    ([257], [777], 2, 1, 64, 64, 0, 64),
    ([33, 1, 200, 64], [500, 77, 200, 65], 8, 2, 128, 16, 1, 0),
    ([90, 17], [1500, 30], 16, 2, 32, 16, 1, 0),
    ([40], [41], 8, 1, 12, 4, 1, 0) , ([70], [200], 5, 5, 100, 32, 1, 0)])
def test_attention_against_float64(rt, kind, new, lens, heads, kvh, hd, page, block, window):
    if kind == "q8_0" and hd % 32:
        hd = 32 * (1 + hd // 32)
    Stream(rt, kind, new, lens, heads, kvh, hd, page, spare_rows=len(new) % 3).check(block, window)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_a_frame_against_earlier_ones(rt, kind):
    Stream(rt, kind, [865], [2595], 12, 12, 64, 32).check(865)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_many_streams_of_unlike_lengths(rt, kind):
    lens = [1 + int(9000 * u ** 4) for u in seeded.uniform01(3, 70)]
    Stream(rt, kind, [1] * 70, lens, 4, 2, 64, 16).check(1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, lens", [([1, 0, 1, 0], [9, 50, 70, 0]), ([0, 0], [5, 0]), ([0, 150, 0], [3, 150, 9]),
                                       ([3, 2, 1], [1, 0, 1])])
def test_requests_without_tokens_and_tokens_without_keys(rt, kind, new, lens):
    """Requests that get nothing this step; lengths below the number of new tokens, whose first ones see no key."""
    s = Stream(rt, kind, new, lens, 4, 2, 64, 16, spare_rows=2)
    s.check(1)
    s.check(0)


@pytest.mark.parametrize("kind", KINDS)
def test_absent_pages_are_not_seen(rt, kind):
    s = Stream(rt, kind, [1, 80, 3], [100, 400, 40], 4, 2, 64, 16)
    table = s.table.copy()
    table[0, 2], table[0, 6], table[1, [0, 5, 24]] = -1, 2**31 - 1, [-5, s.cache.slots // 16, -1]
    table[2, :3] = -1
    absent = [np.isin(np.arange(n) // 16, np.flatnonzero((table[r] < 0) | (table[r] >= s.cache.slots // 16)))
              for r, n in enumerate(s.lens)]
    got = s.check(1, absent=absent, table=table)
    assert (got[s.starts[2]:s.starts[3]] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, lens, block, window", [([1, 1], [100, 70], 1, 20), ([70], [200], 1, 0),
                                                      ([150], [400], 1, 90), ([140], [300], 50, 0)])
def test_unseen_infinities_and_nan_do_not_show(rt, kind, new, lens, block, window):
    def change(r, k, v):
        n = len(k)
        if kind == "q8_0":  # blocks whose scale passes binary16
            v[n - 1, 0, 5], k[n - 2, 1, 7], v[n // 2, 1, 63], k[n // 3, 0, 0], v[3, 0, :], k[5, 1, :] = [1e30] * 6
            return
        v[n - 1, 0, 5], k[n - 2, 1, 7], v[n // 2, 1, 63] = np.inf, np.nan, np.nan
        k[n // 3, 0, 0], v[3, 0, :], k[5, 1, :] = -np.inf, -np.inf, np.inf

    Stream(rt, kind, new, lens, 4, 2, 64, 16, change=change).check(block, window)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("big", [1e4, 1e-20, 1e-38, 1e30])
def test_values_of_any_size(rt, kind, big):
    """Keys against queries whose product stays ordinary, values of any size: nothing is lost to a narrower range."""
    if kind == "q8_0" and big > 1e5 or kind == "q8_0" and big < 1e-6:
        big = 1e4 if big > 1 else 1e-3

    def change(r, k, v):
        v *= np.float32(big)
        v[:, :, ::7] *= np.float32(1e-4)

    Stream(rt, kind, [1, 70], [300, 200], 4, 2, 64, 16, change=change).check(1)


@pytest.mark.parametrize("std", [0.0, 30.0, 1000.0])
def test_scores_of_any_size(rt, std):
    """Flat scores, and scores so far apart that one key takes all."""
    s = Stream(rt, "f32", [1, 70], [300, 200], 4, 2, 64, 16, std=max(std, 1e-30))
    if std == 0.0:
        s.q[:] = 0
    got = s.run(1)
    exp = ref.attention(s.q, s.k, s.v, s.starts, s.lens, 4, 1)
    # A score is off by at most 66 * 2^-24 of the sum of its products' sizes (64 sums, the scale, the exponent), its
    # weight by that much of itself, an output by twice that times its largest value.
    size = max(float((np.abs(s.q).max() * np.abs(k).sum(-1).max())) / 8 for k in s.k)
    tol = min(2.0, 2 * 66 * 2.0 ** -24 * size + 300 * 2.0 ** -24) * 5
    assert np.abs(got - exp).max() <= tol


def test_equal_scores_of_one_key_repeat_the_value(rt):
    """One key: the output is the value itself, bit for bit in f32 (p = 1)."""
    s = Stream(rt, "f32", [1], [1], 2, 2, 64, 16)
    assert_bits_equal(s.run(1).ravel(), s.v[0].ravel(), "single key")


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_call_gives_the_same_bits(rt, kind):
    s = Stream(rt, kind, [1, 1, 200], [3000, 10, 900], 4, 2, 64, 16)
    a = s.run(1)
    for _ in range(3):
        assert_bits_equal(s.run(1).ravel(), a.ravel(), "again")


def test_a_cache_past_4_gib(rt):
    """Pages whose bytes lie past 2^32 from the start of K and of V."""
    page, hd = 4096, 128
    pages = (1 << 32) // (page * hd * 4) + 20
    cache = rt.kv_cache("f32", pages, page, 1, hd)
    n = 5000
    k, v = (seeded.normal(s, n * hd).reshape(n, 1, hd) for s in (1, 2))
    table = np.array([[pages - 1, pages - 3]])
    j = np.arange(n)
    slots = table[0, j // page] * page + j % page
    cache.append(rt.upload_f32(k), rt.upload_f32(v), n, rt.upload_i32(slots), token_major=True)
    back = [rt.alloc_f32(n * hd) for _ in range(2)]
    cache.gather(rt.upload_i32(slots), n, *back)
    assert_bits_equal(rt.download_f32(back[0]), k.ravel(), "k")
    assert_bits_equal(rt.download_f32(back[1]), v.ravel(), "v")
    for new in (1, 100):
        q = seeded.normal(4, new * 2 * hd).reshape(new, 2, hd)
        out = rt.alloc_f32(q.size)
        cache.attention(rt.upload_f32(q), 2, new, rt.upload_i32(table), 2, rt.upload_i32([0, new]),
                        rt.upload_i32([n]), out, block=1)
        args = (q, [k], [v], [0, new], [n], 2, 1)
        close(rt.download_f32(out).reshape(q.shape), ref.attention(*args), ref.attention(*args, dtype=np.float32))


def test_lengths_and_starts_out_of_range_stay_inside(rt):
    """Device values that no step writes: lengths past the table's row count to its end, starts past the batch to
    the batch's, falling starts and negative lengths are empty.  The other rows are as ever."""
    s = Stream(rt, "f32", [2, 3, 1, 4], [40, 48, 20, 30], 4, 2, 64, 16)
    s.width = 3
    s.table = s.table[:, :3]
    args = dict(block=0)
    good = s.run(**args)
    lens, starts = s.lens.copy(), s.starts.copy()
    s.lens = np.array([40, 2**31 - 1, -2**31, 30])
    got = s.run(**args)
    assert_bits_equal(got[:5].ravel(), good[:5].ravel(), "length past the row: all of it")
    assert (got[5] == 0).all()
    assert_bits_equal(got[6:].ravel(), good[6:].ravel(), "others")
    s.lens, s.starts = lens, np.array([0, 2, 5, 3, 2**31 - 1])
    got = s.run(**args)
    assert_bits_equal(got[:2].ravel(), good[:2].ravel(), "before")
    assert s.run(fill=3.0, **args).shape == got.shape
    s.starts = np.array([-2**31, 2, 5, 6, 10])
    s.run(**args)


def test_nothing_to_do(rt):
    cache = rt.kv_cache("f32", 0, 16, 2, 64)
    e, z = rt.upload_f32([]), rt.upload_i32([])
    cache.attention(e, 4, 0, z, 0, rt.upload_i32([0]), z, rt.upload_f32([]))
    out = rt.upload_f32(np.full(256, 5.0))
    cache.attention(rt.alloc_f32(256), 4, 1, z, 0, rt.upload_i32([0]), z, out)
    assert (rt.download_f32(out) == 5.0).all()
    cache.attention(rt.alloc_f32(256), 4, 1, z, 0, rt.upload_i32([0, 1]), rt.upload_i32([7]), out)
    assert (rt.download_f32(out) == 0.0).all()


def test_attention_refuses(rt):
    cache = rt.kv_cache("f32", 4, 16, 2, 64)
    a = {"q": rt.alloc_f32(3 * 256), "heads": 4, "tokens": 3, "table": rt.upload_i32([0, 1, 2, 3]), "max_pages": 2,
         "starts": rt.upload_i32([0, 1, 3]), "lens": rt.upload_i32([5, 5]), "out": rt.alloc_f32(3 * 256)}
    cache.attention(**a)
    for over in ({"q": rt.alloc_f32(255)}, {"out": rt.alloc_f32(2 * 256)}, {"tokens": 4}, {"tokens": 2**62},
                 {"max_pages": 3}, {"max_pages": 2**63}, {"starts": rt.upload_i32([0, 3])},
                 {"lens": rt.upload_i32([1])}, {"table": rt.upload_i32([0, 1])}):
        with pytest.raises(vh.LengthMismatch):
            cache.attention(**(a | over))
    for over in ({"heads": 3}, {"heads": 0}, {"heads": 65536}):
        with pytest.raises(vh.KernelError):
            cache.attention(**(a | over))
    n = 4097
    with pytest.raises(vh.KernelError):
        cache.attention(**(a | {"lens": rt.alloc_i32(n), "starts": rt.alloc_i32(n + 1), "table": rt.alloc_i32(2 * n)}))
    other = vh.Runtime(0)
    for over in ({"q": other.alloc_f32(768)}, {"out": other.alloc_f32(768)}, {"lens": other.upload_i32([5, 5])},
                 {"out": a["q"]}):
        with pytest.raises(vh.InvalidArgument):
            cache.attention(**(a | over))
