"""The operators of a stream of frames run together, as a program uses them: page tables, the QKV projection, cache
writes with rotation, attention over the cache and the output projection, step after step; captured into graphs; from
several runtimes at once.  Against float64 numpy (tests/stream64.py) and against the encoder's own path."""
import ctypes
import threading

import numpy as np
import pytest

import stream64 as ref
import vestra_hip as vh
from conftest import assert_bits_equal
from test_gpu_graph import _capture, _hip
from test_gpu_stream import ROPE_TOL, _tiled
from test_gpu_stream_attention import KINDS, Stream, close
from vestra_hip import da3, seeded

pytestmark = pytest.mark.gpu


def _norm_error(got, exp):
    return np.linalg.norm(got - exp) / np.linalg.norm(exp)


@pytest.mark.parametrize("kind", KINDS)
def test_frames_and_tokens_through_a_layer(rt, kind):
    """Two streams whose frames come at different times, then single tokens, in a padded batch."""
    heads, kvh, hd, dim, page, width = 4, 2, 64, 128, 16, 14
    frame, batch, pairs, freq = 43, 2 * 43 + 3, [8, 12, 12], 100.0
    rows = (heads + 2 * kvh) * hd
    wq, bq = seeded.normal(1, dim * rows, 0.1), seeded.normal(2, rows, 0.1)
    wp, bp = seeded.normal(3, heads * hd * dim, 0.1), seeded.normal(4, dim, 0.1)
    qkv_lin, proj = rt.prepare_linear_f32(dim, rows, wq, bq), rt.prepare_linear_f32(heads * hd, dim, wp, bp)
    rope = rt.prepare_rope_axes(hd, pairs, freq)
    cache = rt.kv_cache(kind, 2 * width, page, kvh, hd)
    free = rt.upload_i32(np.argsort(seeded.uniform01(5, 2 * width), kind="stable"))
    table = rt.upload_i32(np.full(2 * width, -1))
    cached, start = rt.upload_i32([0, 0]), rt.upload_i32([0])
    grid = da3.positions_yx(6, 7).reshape(-1, 2)
    had = [0, 0]
    for step, (new, block) in enumerate([([frame, frame], frame), ([frame, 0], frame), ([frame, frame], frame),
                                         ([0, frame], frame), ([1, 1], 1), ([1, 0], 1)]):
        starts, lens, slots, nxt = rt.alloc_i32(3), rt.alloc_i32(2), rt.alloc_i32(batch), rt.alloc_i32(1)
        rt.kv_pages_assign(cached, rt.upload_i32(new), free, start, page, table, width, starts, lens, slots, nxt)
        pos = np.zeros((batch, 3), np.int32)
        at = 0
        for r, n in enumerate(new):
            pos[at:at + n] = [[had[r], 0, 0]] if n == 1 else np.c_[np.full(frame, had[r] // frame), grid][:n]
            at += n
            had[r] += n
        x = seeded.normal(10 + step, batch * dim)
        xt, q, out = rt.upload_f32(x), rt.alloc_f32(batch * heads * hd), rt.upload_f32(np.zeros(batch * heads * hd))
        qkv = qkv_lin.run(xt, batch)
        cache.append_qkv(qkv, heads, batch, slots, q, rope=rope, positions=rt.upload_i32(pos))
        cache.attention(q, heads, batch, table, width, starts, lens, out, block=block)
        proj.run_residual(out, batch, xt)
        cached, start = lens, nxt

        assert list(rt.download_i32(lens)) == had and rt.download_i32(starts)[-1] == sum(new)
        got_qkv = rt.download_f32(qkv).reshape(batch, heads + 2 * kvh, hd)
        exp = x.reshape(batch, dim).astype(np.float64) @ wq.reshape(dim, rows) + bq
        assert _norm_error(got_qkv.reshape(batch, rows), exp) <= 1e-6
        # What this step stored: V exactly, K and Q to the rotation's rounding and K to its type's half step.
        turned = ref.rotate(got_qkv[:, :heads + kvh], pos, pairs, freq, False)
        size = ROPE_TOL * 2 * np.abs(got_qkv[:, :heads + kvh]).max(-1, keepdims=True)
        got_q = rt.download_f32(q).reshape(batch, heads, hd)
        assert (np.abs(got_q - turned[:, :heads]) <= size[:, :heads]).all()
        k, v = rt.alloc_f32(batch * kvh * hd), rt.alloc_f32(batch * kvh * hd)
        cache.gather(slots, batch, k, v)
        n = sum(new)
        key = turned[:n, heads:]
        half = {"f32": 2.0 ** -24 * np.abs(key), "bf16": 2.0 ** -8 * np.abs(key),
                # Half a step of the scale amax / 127, which binary16 holds to 2^-11 of itself, 127 steps at most.
                "q8_0": np.repeat(np.abs(key).reshape(n, kvh, 2, 32).max(-1), 32, -1) / 127 * (0.5 + 128 * 2.0 ** -11)}
        assert (np.abs(rt.download_f32(k).reshape(batch, kvh, hd)[:n] - key) <= 1.01 * half[kind] + size[:n, heads:]).all()
        assert_bits_equal(rt.download_f32(v).reshape(batch, kvh, hd)[:n].ravel() + 0.0,
                          ref.stored(got_qkv[:n, heads + kvh:], kind).ravel() + 0.0, "v")
        # Attention over all that the streams hold by now, and the layer's output.
        ks, vs, tab = [], [], rt.download_i32(table).reshape(2, width)
        for r, length in enumerate(had):
            j = np.arange(length)
            k, v = rt.alloc_f32(length * kvh * hd), rt.alloc_f32(length * kvh * hd)
            cache.gather(rt.upload_i32(tab[r, j // page] * page + j % page), length, k, v)
            ks.append(rt.download_f32(k).reshape(length, kvh, hd))
            vs.append(rt.download_f32(v).reshape(length, kvh, hd))
        args = (got_q, ks, vs, np.concatenate([[0], np.cumsum(new)]), had, heads, block)
        got = rt.download_f32(out).reshape(got_q.shape)
        close(got[:n], ref.attention(*args)[:n], ref.attention(*args, dtype=np.float32)[:n])
        assert (got[n:] == 0).all()
        exp = x.reshape(batch, dim) + got.reshape(batch, -1).astype(np.float64) @ wp.reshape(-1, dim) + bp
        assert _norm_error(rt.download_f32(xt).reshape(batch, dim), exp) <= 1e-6


def test_one_frame_equals_the_encoders_attention(rt):
    heads, tokens, dim = 12, 865, 768
    lin = rt.prepare_linear_f32(dim, 3 * dim, seeded.normal(1, 3 * dim * dim, 0.02), seeded.normal(2, 3 * dim, 0.02))
    x, pos = rt.upload_f32(seeded.normal(3, tokens * dim)), da3.positions_yx(24, 36)
    q, k, v = lin.run_qkv_hnd(x, 1, tokens, heads, pos, 100.0)
    exp = rt.download_f32(rt.flash_attention_f32_da3_base(q, k, v, heads, tokens, token_major=True))
    cache = rt.kv_cache("f32", 28, 32, heads, 64)
    q, out = rt.alloc_f32(tokens * dim), rt.alloc_f32(tokens * dim)
    cache.append_qkv(lin.run(x, tokens), heads, tokens, rt.upload_i32(np.arange(tokens)), q,
                     rope=rt.prepare_rope_axes(64, [16, 16], 100.0),
                     positions=rt.upload_i32(pos.reshape(-1).astype(np.int32)))
    cache.attention(q, heads, tokens, rt.upload_i32(np.arange(28)), 28, rt.upload_i32([0, tokens]),
                    rt.upload_i32([tokens]), out)
    # The encoder's angles are 32-bit: off by 36 * 3 * 2^-24 rad at most, Q and K by that much of themselves, a score
    # by twice that of |q| |k| / 8 (about 4 here, 10 at most), a weight by that much of itself.
    assert _norm_error(rt.download_f32(out), exp) <= 2 * 36 * 3 * 2.0 ** -24 * 10


class Tokens:
    """Requests that get a token each in every step, on buffers of their own.  What a step writes is the next one's
    input, so steps of even and odd number take turns with two sets of lengths."""

    def __init__(self, rt, kind, lens, heads=4, kvh=2, hd=64, page=8):
        self.rt, self.heads, self.page, n = rt, heads, page, len(lens)
        self.width = max(lens) // page + 4
        pages = sum(-(-x // page) for x in lens) + 4 * n
        self.cache = rt.kv_cache(kind, pages, page, kvh, hd)
        self.rope = rt.prepare_rope_axes(hd, [hd // 2], 10000.0, shared=True)
        self.free = rt.upload_i32(np.arange(pages)[::-1])
        self.table = rt.upload_i32(np.full(n * self.width, -1))
        self.lens = [rt.alloc_i32(n), rt.alloc_i32(n)]
        self.at = [rt.alloc_i32(1), rt.alloc_i32(1)]
        self.ones, self.starts, self.slots = rt.upload_i32([1] * n), rt.alloc_i32(n + 1), rt.alloc_i32(n)
        self.n, self.rows = n, (heads + 2 * kvh) * hd
        self.qkv, self.q, self.out = (rt.alloc_f32(n * w) for w in (self.rows, heads * hd, heads * hd))
        total = sum(lens)
        slots = rt.alloc_i32(total)
        rt.kv_pages_assign(rt.upload_i32([0] * n), rt.upload_i32(lens), self.free, rt.upload_i32([0]), page, self.table,
                           self.width, self.starts, self.lens[0], slots, self.at[0])
        k, v = (rt.upload_f32(seeded.normal(s, total * kvh * hd)) for s in (1, 2))
        self.cache.append(k, v, total, slots, token_major=True)

    def feed(self, step):
        """This step's rows (eagerly, before the step)."""
        x = self.rt.upload_f32(seeded.normal(100 + step, self.n * self.rows))
        self.rt.copy_segment_into_f32(self.qkv, 0, x, 0, self.n * self.rows)

    def step(self, odd):
        had, has = self.lens[odd], self.lens[1 - odd]
        self.rt.kv_pages_assign(had, self.ones, self.free, self.at[odd], self.page, self.table, self.width, self.starts,
                                has, self.slots, self.at[1 - odd])
        self.cache.append_qkv(self.qkv, self.heads, self.n, self.slots, self.q, rope=self.rope, positions=had)
        self.cache.attention(self.q, self.heads, self.n, self.table, self.width, self.starts, has, self.out, block=1)


@pytest.mark.parametrize("kind", KINDS)
def test_two_graphs_step_a_stream(rt, kind):
    """A graph for the even steps and one for the odd ones, with the same steps of another state eagerly between."""
    hip, stream = _hip(), ctypes.c_void_p(rt.stream())
    lens = [1, 7, 100, 3000, 33]
    eager, graph = Tokens(rt, kind, lens), Tokens(rt, kind, lens)
    exp = []

    def eager_step():
        eager.feed(len(exp))
        eager.step(len(exp) % 2)
        exp.append(rt.download_f32(eager.out))

    made = []
    try:
        for odd in (0, 1):
            eager_step()  # room for the capture that follows
            made.append(_capture(hip, stream, lambda: graph.step(odd)))
        for step in range(12):
            graph.feed(step)
            assert hip.hipGraphLaunch(made[step % 2][1], stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            assert_bits_equal(rt.download_f32(graph.out), exp[step], f"step {step}")
            eager_step()
        assert list(rt.download_i32(graph.lens[0])) == [n + 12 for n in lens]
    finally:
        for g, e in made:
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)


class Call:
    """One attention call on buffers of its own."""

    def __init__(self, s, block=1):
        self.s, self.block, rt = s, block, s.rt
        self.q, self.out = rt.upload_f32(s.q), rt.upload_f32(np.zeros(s.q.size))
        self.table, self.starts, self.lens = rt.upload_i32(s.table), rt.upload_i32(s.starts), rt.upload_i32(s.lens)
        rt.synchronize()

    def run(self):
        self.s.cache.attention(self.q, self.s.heads, self.s.tokens, self.table, self.s.width, self.starts, self.lens,
                               self.out, block=self.block)

    def clear(self):
        rt = self.s.rt
        rt.copy_segment_into_f32(self.out, 0, rt.upload_f32(np.zeros(len(self.out))), 0, len(self.out))

    def take(self):
        got = self.s.rt.download_f32(self.out)
        self.clear()
        return got

    def check(self, got):
        s = self.s
        args = (s.q, s.k, s.v, s.starts, s.lens, s.heads, self.block)
        close(got.reshape(s.q.shape), ref.attention(*args), ref.attention(*args, dtype=np.float32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1], [200, 40]])
def test_a_graph_of_a_size_that_has_not_run(kind, new):
    """Without room for parts each tile stays with one workgroup: right, and the same on every replay."""
    rt = vh.Runtime(0)  # its own, without workspaces
    hip, stream = _hip(), ctypes.c_void_p(rt.stream())
    call = Call(Stream(rt, kind, new, [2000, 300], 4, 2, 64, 16))
    graph, exe = _capture(hip, stream, call.run)
    try:
        got = []
        for _ in range(3):
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            got.append(call.take())
            call.run()
            eager = call.take()
        call.check(got[0])
        call.check(eager)
        for g in got[1:]:
            assert_bits_equal(g, got[0])
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("new", [[1, 1], [200, 40]])
def test_graphs_on_several_streams_at_once(rt, new):
    """Three graphs of one runtime, the third captured right after the second, replayed on streams of their own while
    the runtime runs a larger call: no two of them share a workspace."""
    hip = _hip()
    hip.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    hip.hipStreamDestroy.argtypes = [ctypes.c_void_p]
    stream = ctypes.c_void_p(rt.stream())
    calls = [Call(Stream(rt, "f32", new, [5000, 700], 4, 2, 64, 16, seed=20 * i + 1)) for i in range(3)]
    larger = Call(Stream(rt, "f32", [300, 1], [6000, 9000], 4, 2, 64, 16, seed=90))
    made, streams = [], []
    try:
        for i, c in enumerate(calls):
            if i < 2:
                c.run()
            made.append(_capture(hip, stream, c.run))
            streams.append(ctypes.c_void_p())
            assert hip.hipStreamCreateWithFlags(ctypes.byref(streams[-1]), 1) == 0
        larger.run()
        first = larger.take()
        for c in calls:
            c.clear()
        rt.synchronize()
        exp = []
        for _, e in made:  # one by one
            assert hip.hipGraphLaunch(e, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
        for c in calls:
            exp.append(c.take())
            c.check(exp[-1])
        for _ in range(3):
            rt.synchronize()
            for _ in range(10):
                for (_, e), s in zip(made, streams):
                    assert hip.hipGraphLaunch(e, s) == 0
                larger.run()
            for s in streams:
                assert hip.hipStreamSynchronize(s) == 0
            for c, e in zip(calls, exp):
                assert_bits_equal(c.take(), e, "at once")
            assert_bits_equal(larger.take(), first, "the runtime's own")
    finally:
        for g, e in made:
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)
        for s in streams:
            hip.hipStreamDestroy(s)


def test_a_cache_is_not_made_inside_a_capture(rt):
    hip, stream = _hip(), ctypes.c_void_p(rt.stream())
    call = Call(Stream(rt, "f32", [3], [40], 2, 2, 64, 16))

    def run():
        with pytest.raises(vh.KernelError):
            rt.kv_cache("f32", 4, 16, 2, 64)
        call.run()

    graph, exe = _capture(hip, stream, run)
    try:
        assert hip.hipGraphLaunch(exe, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
        call.check(call.take())
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


def test_runtimes_in_threads_of_their_own():
    calls = []
    for i, new in enumerate(([1, 1, 1], [150, 1])):
        calls.append(Call(Stream(vh.Runtime(0), "bf16", new, [3000, 80, 500][:len(new)], 8, 2, 128, 16, seed=i + 1)))
    exp = []
    for c in calls:
        c.run()
        exp.append(c.take())
        c.check(exp[-1])
    wrong = []

    def work(c, e):
        for _ in range(30):
            c.run()
            if not np.array_equal(c.take(), e):
                wrong.append(c.s.new)

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, exp)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("kind", KINDS)
def test_as_many_requests_as_a_call_takes(rt, kind):
    n = 4096
    lens = [int(40 * u) for u in seeded.uniform01(5, n)]
    Stream(rt, kind, [1] * n, lens, 2, 1, 64, 8).check(1)
    new = [int(3 * u) for u in seeded.uniform01(6, n)]
    Stream(rt, kind, new, [a + b for a, b in zip(lens, new)], 2, 1, 64, 8).check(1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 70, 70]])
def test_requests_that_share_pages(rt, kind, new):
    """The same pages in the rows of several requests, which are only read: a prefix kept once."""
    s = Stream(rt, kind, new, [200, 200, 200], 4, 2, 64, 16)
    s.table[1, :8] = s.table[0, :8]
    s.table[2] = s.table[0]
    for kv in (s.k, s.v):
        kv[1][:128], kv[2] = kv[0][:128], kv[0]
    s.q[s.starts[2]:] = s.q[:new[0]]
    got = s.check(1)
    assert_bits_equal(got[s.starts[2]:].ravel(), got[:new[0]].ravel(), "the same request again")


def test_queries_past_4_gib(rt):
    """Queries and outputs whose bytes pass 2^32, against few keys: the last tokens."""
    heads, kvh, hd, tokens, tail, n = 2, 1, 64, (1 << 23) + 50, 500, 10
    piece = seeded.normal(31, (1 << 16) * heads * hd)
    q, out = _tiled(rt, tokens * heads * hd, piece), rt.alloc_f32(tokens * heads * hd)
    cache = rt.kv_cache("f32", 1, 16, kvh, hd)
    k, v = (seeded.normal(s, n * hd).reshape(n, 1, hd) for s in (32, 33))
    cache.append(rt.upload_f32(k), rt.upload_f32(v), n, rt.upload_i32(np.arange(n)), token_major=True)
    cache.attention(q, heads, tokens, rt.upload_i32([0]), 1, rt.upload_i32([0, tokens]), rt.upload_i32([n]), out)
    got = rt.download_f32(rt.copy_segment_f32(out, (tokens - tail) * heads * hd, tail * heads * hd))
    last = piece.reshape(-1, heads, hd)[np.arange(tokens - tail, tokens) % (1 << 16)]
    args = (last, [k], [v], [0, tail], [n], heads)
    close(got.reshape(last.shape), ref.attention(*args), ref.attention(*args, dtype=np.float32))


@pytest.mark.parametrize("new", [[1, 1], [100, 90]])
def test_starts_that_fall_cost_no_more_than_a_batch(rt, new):
    """Starts that name every token for every second request: the call takes no longer than its batch allows, writes
    nothing behind the batch, and the runtime's next call is as ever."""
    s = Stream(rt, "bf16", new, [300, 500], 4, 2, 64, 16)
    good = s.run(1)
    n, t = 3000, s.tokens
    starts = np.tile([0, t], n // 2 + 1)[:n + 1]
    table, lens = np.tile(s.table[:1], (n, 1)), np.full(n, 300)
    out = rt.upload_f32(np.full(s.q.size, 5.0))
    s.cache.attention(rt.upload_f32(s.q), 4, t, rt.upload_i32(table), s.width, rt.upload_i32(starts),
                      rt.upload_i32(lens), out, block=1)
    assert rt.download_f32(out).shape == (s.q.size,)
    assert_bits_equal(s.run(1).ravel(), good.ravel(), "the next call")
