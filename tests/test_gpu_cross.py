"""An encoder's states and the attention over them on the GPU, against float64 numpy (tests/fp8_64.py).

What is stored is compared value for value.  The attention's tolerance, in the norm of a head's output against the
norm that its weights could give it, sqrt(sum p^2) |v|: a score of s (base e) is off by 2^-22 of it for what the
split of q leaves (2^-23), the sums of 64 or 128 products and the scaling, so a weight by 2^-22 max |s| + 2^-21
(exp2, its split, the running sums); against the exact attention over the stored values that is 2^-21 (2 + max
|s|) of the sum of the |weighted values|, the bound used."""
import numpy as np
import pytest

import fp8_64 as ref
import vestra_hip as vh
from conftest import assert_bits_equal
from vestra_hip import seeded

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16"]


def same_values(got, exp):
    """Equal values; a negative value that two halves leave nothing of is a zero of either sign (-0 + 0)."""
    assert np.array_equal(got, exp.astype(np.float32))


class States:
    """Images' K and V in a handle, some tokens unseen, and what the handle should hold."""

    def __init__(self, rt, kind, images, tokens, kvh, hd, seen=None, capacity=None, token_major=True, rows=False,
                 seed=1, change=None):
        self.rt, self.images, self.kvh, self.hd = rt, images, kvh, hd
        shape = (images, tokens, kvh, hd)
        k, v = (seeded.normal(seed + i, max(1, int(np.prod(shape))))[:int(np.prod(shape))].reshape(shape)
                for i in (0, 1))
        k[..., -1] += 2.0
        if change is not None:
            change(k, v)
        self.capacity = tokens if capacity is None else capacity
        self.kv = rt.cross_kv(kind, images, self.capacity, kvh, hd)
        self.mask = None
        if seen is not None:
            u = seeded.uniform01(seed + 9, images * max(1, tokens)).reshape(images, -1)[:, :tokens]
            self.mask = (u < np.broadcast_to(np.reshape(seen, (-1, 1)), (images, 1))) * (1 + np.arange(tokens) % 3)
        self.write(k, v, rows, token_major)
        held = [ref.stored(k[i], v[i], kind, None if self.mask is None else self.mask[i]) for i in range(images)]
        self.k, self.v = [h[0] for h in held], [h[1] for h in held]

    def write(self, k, v, rows=False, token_major=True):
        n, t = self.images, k.shape[1]
        seen = None if self.mask is None else self.rt.upload_i32(self.mask)
        if rows:
            both = np.concatenate([k.reshape(n * t, -1), v.reshape(n * t, -1)], 1)
            self.kv.write_rows(self.rt.upload_f32(both), t, seen=seen)
        else:
            a, b = (x if token_major else np.ascontiguousarray(x.transpose(0, 2, 1, 3)) for x in (k, v))
            self.kv.write(self.rt.upload_f32(a), self.rt.upload_f32(b), t, token_major=token_major, seen=seen)

    def read(self):
        n = self.images * self.capacity * self.kvh * self.hd
        k, v = (self.rt.upload_f32(np.full(n, 7.0)) for _ in range(2))
        lens = self.rt.alloc_i32(self.images)
        self.kv.read(k, v, lens)
        shape = (self.images, self.capacity, self.kvh, self.hd)
        return (*(self.rt.download_f32(x).reshape(shape) for x in (k, v)), self.rt.download_i32(lens))

    def run(self, q, token_major=True, kv=None):
        """q [images, n, heads, hd]."""
        images, n, heads, _ = q.shape
        x = q if token_major else np.ascontiguousarray(q.transpose(0, 2, 1, 3))
        out = self.rt.upload_f32(np.full(q.size, np.nan))
        self.kv.attention(self.rt.upload_f32(x), heads, n, out, token_major=token_major)
        got = self.rt.download_f32(out).reshape(x.shape)
        return got if token_major else got.transpose(0, 2, 1, 3)

    def check(self, heads, n, std=1.0, token_major=True, seed=40):
        q = seeded.normal(seed, self.images * n * heads * self.hd, std).reshape(self.images, n, heads, self.hd)
        got = self.run(q, token_major)
        for i in range(self.images):
            close(got[i], q[i], self.k[i], self.v[i])
        return got


def close(got, q, k, v):
    want = ref.attention(q, k, v)
    assert np.isfinite(got).all()
    if not len(k):
        assert not got.any()
        return
    heads = q.shape[1]
    for h in range(heads):
        one = h // (heads // k.shape[1])
        s = q[:, h].astype(np.float64) @ k[:, one].T / np.sqrt(q.shape[2])
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        # Of a score: the size of the terms it is summed of.
        size = np.abs(q[:, h].astype(np.float64)) @ np.abs(k[:, one]).T / np.sqrt(q.shape[2])
        bound = 2.0 ** -21 * ((2 + size) * p) @ np.abs(v[:, one]) + \
            2.0 ** -21 * ((2 + size) * p).sum(1, keepdims=True) * np.abs(want[:, h]) + 1e-37
        worst = np.max(np.abs(got[:, h] - want[:, h]) / bound)
        assert worst <= 1.0, (h, worst)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("images, tokens, kvh, hd, seen, capacity, token_major, rows", [
    (1, 1, 1, 4, None, None, True, False), (1, 1, 2, 64, None, 200, False, False),
    (2, 31, 3, 52, 0.7, 40, True, False), (3, 33, 1, 128, [1.0, 0.0, 0.4], 129, False, False),
    (1, 865, 12, 64, 0.9, None, False, False), (2, 1000, 9, 96, None, 1001, True, True),
    (70, 65, 1, 32, 0.5, 128, True, True), (1, 5000, 17, 64, 0.3, None, True, False),
    (2, 300, 300, 4, 0.8, None, True, True)])
def test_what_is_stored(rt, kind, images, tokens, kvh, hd, seen, capacity, token_major, rows):
    s = States(rt, kind, images, tokens, kvh, hd, seen, capacity, token_major, rows)
    k, v, lens = s.read()
    assert list(lens) == [len(x) for x in s.k]
    for i in range(images):
        n = lens[i]
        same_values(k[i, :n], s.k[i])
        same_values(v[i, :n], s.v[i])
        assert not k[i, n:].any() and not v[i, n:].any()


@pytest.mark.parametrize("kind", KINDS)
def test_new_states_hold_nothing_and_a_write_replaces_all(rt, kind):
    s = States(rt, kind, 2, 0, 2, 64, capacity=300)
    assert list(s.read()[2]) == [0, 0] and not s.read()[0].any()
    s.check(4, 3)
    q = seeded.normal(5, 2 * 3 * 4 * 64).reshape(2, 3, 4, 64)
    fresh = rt.cross_kv(kind, 2, 300, 2, 64)
    out = rt.upload_f32(np.full(q.size, 7.0))
    fresh.attention(rt.upload_f32(q), 4, 3, out)
    assert not rt.download_f32(out).any()
    for tokens, scale in ((300, 1e20), (7, 1e-20), (150, 1.0)):
        k, v = (seeded.normal(tokens + i, 2 * tokens * 128, scale).reshape(2, tokens, 2, 64) for i in (0, 1))
        s.write(k, v)
        got_k, got_v, lens = s.read()
        assert list(lens) == [tokens] * 2 and not got_k[:, tokens:].any() and not got_v[:, tokens:].any()
        for i in range(2):
            ek, ev = ref.stored(k[i], v[i], kind)
            same_values(got_k[i, :tokens], ek)
            same_values(got_v[i, :tokens], ev)


@pytest.mark.parametrize("kind", KINDS)
def test_stored_range(rt, kind):
    """Heads and dims of very different size side by side, each on an exponent of its own, subnormal floats and
    the largest ones."""
    def change(k, v):
        k *= np.float32(2.0) ** np.array([-140, -20, 0, 120])[None, None, :, None]
        v *= np.exp2(np.linspace(-140, 120, 32)).astype(np.float32)
        k[0, 3], v[0, 3] = np.finfo(np.float32).max, np.finfo(np.float32).max
    s = States(rt, kind, 1, 40, 4, 32, change=change)
    k, v, _ = s.read()
    with np.errstate(over="ignore"):
        same_values(k[0], s.k[0])
        same_values(v[0], s.v[0])


SHAPES = [  # images, queries, tokens, heads, kv_heads, head_dim, seen
    (1, 1, 1, 1, 1, 4, None), (1, 1, 3460, 12, 12, 64, None), (2, 1, 127, 12, 12, 64, None),
    (3, 1, 129, 8, 1, 32, [0.0, 1.0, 0.5]), (5, 3, 700, 20, 4, 100, 0.6), (48, 1, 300, 32, 8, 128, 0.7),
    (1, 16, 33, 3, 3, 64, None), (1, 17, 64, 3, 3, 64, None), (2, 5, 2000, 32, 8, 128, 0.5),
    (1, 128, 128, 2, 2, 64, None), (1, 129, 1, 2, 2, 64, None), (2, 200, 1000, 6, 6, 52, [0.0, 0.8]),
    (1, 865, 1730, 6, 6, 64, 0.9), (3, 257, 511, 9, 3, 96, [0.1, 1.0, 0.0]), (1, 900, 3000, 4, 2, 128, None),
    (300, 2, 40, 2, 1, 64, 0.5), (4, 1500, 65, 2, 2, 64, None),
    (300, 100, 600, 1, 1, 64, 0.6), (290, 200, 300, 2, 1, 128, 0.9), (30, 300, 400, 4, 2, 64, 0.5),
    (54, 9, 44, 40, 10, 100, 0.9), (64, 8, 129, 12, 12, 64, [0.0, 0.02, 1.0, 0.5] * 16)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("images, n, tokens, heads, kvh, hd, seen", SHAPES)
def test_attention_against_float64(rt, kind, images, n, tokens, heads, kvh, hd, seen):
    s = States(rt, kind, images, tokens, kvh, hd, seen)
    a = s.check(heads, n)
    assert_bits_equal(s.check(heads, n, token_major=False), a)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 40, 300])
@pytest.mark.parametrize("std", [0.0, 30.0, 1e-30])
def test_scores_of_any_size(rt, kind, n, std):
    """Equal scores, scores that leave one key, and queries of the smallest size."""
    States(rt, kind, 1, 500, 2, 64).check(2, n, std=std)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 200])
def test_a_score_that_rises_late(rt, kind, n):
    """The last keys' scores pass all before by far: what was summed until then is corrected."""
    def change(k, v):
        k[:, :, :, 0] = np.linspace(-30, 30, k.shape[1])[None, :, None]
    s = States(rt, kind, 1, 1500, 2, 64, change=change)
    q = seeded.normal(3, n * 2 * 64).reshape(1, n, 2, 64)
    q[..., 0] = 20.0
    close(s.run(q)[0], q[0], s.k[0], s.v[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 200])
def test_values_of_any_size(rt, kind, n):
    """Dims of V at both ends of the floats, K and queries of unlike size."""
    def change(k, v):
        v *= np.exp2(np.linspace(-120, 110, 64)).astype(np.float32)
        k *= np.float32(1e18)
    s = States(rt, kind, 1, 700, 2, 64, change=change)
    q = (seeded.normal(3, n * 2 * 64) * np.float32(1e-18)).reshape(1, n, 2, 64)
    close(s.run(q)[0], q[0], s.k[0], s.v[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 200])
def test_infinities_and_nan(rt, kind, n):
    """Unseen ones do not show; one in a value reaches its dim alone, one in a query its row alone, one in a key
    its image and head alone."""
    bad = np.array([np.nan, np.inf, -np.inf])

    def spoil(k, v):
        k[1, 5:8, 0, 3] = k[1, 5:8, 1, 9] = v[1, 5:8, 0, 3] = bad
    s = States(rt, kind, 3, 90, 2, 64, change=spoil)
    q = seeded.normal(4, 3 * n * 2 * 64).reshape(3, n, 2, 64)
    s.mask = np.ones((3, 90), int)
    s.mask[1, 5:8] = 0
    k, v = (seeded.normal(1 + i, 3 * 90 * 128).reshape(3, 90, 2, 64) for i in (0, 1))
    k[..., -1] += 2.0
    spoil(k, v)
    s.write(k, v)
    got = s.run(q)
    for i in range(3):
        close(got[i], q[i], *ref.stored(k[i], v[i], kind, s.mask[i]))
    # One value.
    s.mask, k[1, 5:8], v[1, 5:8] = None, 0.5, 0.25
    v[1, 6, 1, 7] = np.inf
    s.write(k, v)
    got = s.run(q)
    assert not np.isfinite(got[1, :, 1, 7]).any()
    spoilt = np.zeros(got.shape, bool)
    spoilt[1, :, 1, 7] = True
    assert np.isfinite(got[~spoilt]).all()
    # One key.
    v[1, 6, 1, 7], k[1, 6, 1, 7] = 0.25, np.nan
    s.write(k, v)
    got = s.run(q)
    spoilt[1, :, 1] = True
    assert np.isnan(got[1, :, 1]).all() and np.isfinite(got[~spoilt]).all()
    # One query.
    k[1, 6, 1, 7] = 0.5
    s.write(k, v)
    q[2, n // 2, 0, 5] = np.nan
    got = s.run(q)
    spoilt[:] = False
    spoilt[2, n // 2, 0] = True
    assert np.isnan(got[spoilt]).all() and np.isfinite(got[~spoilt]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 100, 700])
def test_the_same_call_gives_the_same_bits(rt, kind, n):
    s = States(rt, kind, 2, 900, 4, 64, 0.8)
    q = seeded.normal(3, 2 * n * 4 * 64).reshape(2, n, 4, 64)
    a = s.run(q)
    for _ in range(3):
        assert_bits_equal(s.run(q), a)


def test_nothing_to_do(rt):
    s = States(rt, "f16", 2, 10, 2, 64)
    s.kv.attention(rt.alloc_f32(0), 2, 0, rt.alloc_f32(0))
    s.kv.write(rt.alloc_f32(0), rt.alloc_f32(0), 0)
    assert list(s.read()[2]) == [0, 0]


@pytest.mark.parametrize("kind, images, tokens, kvh, hd", [
    ("f64", 1, 1, 1, 64), ("f16", 0, 1, 1, 64), ("f16", 65536, 1, 1, 64), ("f16", 1, 0, 1, 64),
    ("f16", 1, 2 ** 30 + 1, 1, 64), ("f16", 1, 1, 0, 64), ("f16", 1, 1, 65536, 64), ("f16", 1, 1, 1, 0),
    ("f16", 1, 1, 1, 62), ("f16", 1, 1, 1, 132)])
def test_states_refuse(rt, kind, images, tokens, kvh, hd):
    with pytest.raises(vh.KernelError):
        rt.cross_kv(kind, images, tokens, kvh, hd)


def test_calls_refuse(rt):
    kv, other = rt.cross_kv("f16", 2, 10, 2, 64), vh.Runtime(0)
    x, y, z = rt.alloc_f32(2 * 10 * 128), rt.alloc_f32(2 * 10 * 128), other.alloc_f32(2 * 10 * 128)
    rows, lens = rt.alloc_f32(2 * 10 * 256), rt.alloc_i32(2)
    bad = [
        (vh.KernelError, lambda: kv.write(x, y, 11)), (vh.LengthMismatch, lambda: kv.write(x, y, 9)),
        (vh.LengthMismatch, lambda: kv.write(x, rows, 10)), (vh.InvalidArgument, lambda: kv.write(x, z, 10)),
        (vh.LengthMismatch, lambda: kv.write(x, y, 10, seen=rt.alloc_i32(10))),
        (vh.InvalidArgument, lambda: kv.write(x, y, 10, seen=other.alloc_i32(20))),
        (vh.LengthMismatch, lambda: kv.write_rows(x, 10)), (vh.KernelError, lambda: kv.write_rows(rows, 11)),
        (vh.LengthMismatch, lambda: kv.read(x, rows)), (vh.LengthMismatch, lambda: kv.read(x, y, rt.alloc_i32(3))),
        (vh.InvalidArgument, lambda: kv.read(x, z)), (vh.InvalidArgument, lambda: kv.read(x, x)),
        (vh.InvalidArgument, lambda: kv.read(x, y, other.alloc_i32(2))),
        (vh.KernelError, lambda: kv.attention(x, 3, 10, y)), (vh.KernelError, lambda: kv.attention(x, 0, 10, y)),
        (vh.KernelError, lambda: kv.attention(x, 2, 2 ** 29 + 1, y)),
        (vh.LengthMismatch, lambda: kv.attention(x, 2, 9, y)), (vh.LengthMismatch, lambda: kv.attention(x, 4, 10, y)),
        (vh.InvalidArgument, lambda: kv.attention(x, 2, 10, x)), (vh.InvalidArgument, lambda: kv.attention(x, 2, 10, z))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    kv.read(x, y, lens)
    assert not rt.download_f32(x).any() and not rt.download_i32(lens).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 40, 300])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e12])
def test_scores_far_past_the_floats_between_them(rt, kind, n, size):
    """Scores of 1e8 and up, where neighbouring floats are 8 apart: a token along whose key each query lies has
    all of the weight.  Its score is above the others by a quarter of itself, and off by less than 2^-18 of that."""
    tokens, hd = 700, 64

    def change(k, v):
        k[...] = np.sign(k) * np.float32(size)
        k[0, 501, 0] = size

    states = States(rt, kind, 1, tokens, 1, hd, change=change)
    gap = states.k[0][501, 0] @ states.k[0][:, 0].T
    assert np.sort(gap)[-2] <= 0.75 * gap[501]
    q = np.full((1, n, 2, hd), np.float32(size))
    q[:, :, 1] *= -1.0  # the least score there is, and the others around zero
    q[:, :, 1, ::2] *= 0.0
    got = states.run(q)
    v = states.v[0][501, 0]
    assert np.abs(got[0, :, 0] - v).max() <= 2.0 ** -18 * np.abs(v).max()
    assert np.isfinite(got).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 300])
@pytest.mark.parametrize("gap", [17.0, 20.4, 21.5, 23.0])
def test_many_small_weights_behind_a_large_one(rt, kind, n, gap):
    """One token that has nearly all of the weight, and 60000 whose weights are alike and e^-gap of its: what
    these come to.  A weight is held to within 2^-34 of the largest, so 60000 to 2^-18.1 together, of values of
    1; a score of 23 in 32 bits and its exp2 to 2^-18."""
    tokens, hd = 60000, 64

    def change(k, v):
        k[...] = 0.0
        k[0, 123, 0, 0] = 8.0
        v[...] = 1.0
        v[0, 123] = 0.0

    states = States(rt, kind, 1, tokens, 1, hd, change=change)
    q = np.zeros((1, n, 1, hd), np.float32)
    q[..., 0] = gap
    got = states.run(q)
    w = (tokens - 1) * np.exp(-float(q[0, 0, 0, 0]))
    want = w / (1 + w)
    assert np.abs(got - want).max() <= 2.0 ** -18 * (1 + want)
