"""Projections in 8-bit floating point and the attention over an encoder's states run together, as a decoder behind
the encoder uses them; captured into graphs; from several runtimes at once; past 4 GiB.  Against float64 numpy
(tests/fp8_64.py), stage by stage on what the stage before left on the device."""
import ctypes
import threading

import numpy as np
import pytest

import fp8_64 as ref
import vestra_hip as vh
from conftest import assert_bits_equal
from test_gpu_cross import KINDS, States, close
from test_gpu_fp8 import _close
from test_gpu_graph import _capture, _hip
from vestra_hip import da3, seeded

pytestmark = pytest.mark.gpu


class Layer:
    """A decoder layer's cross attention and MLP: weights of floats or a checkpoint's blocks."""

    def __init__(self, rt, kind, images, states, most, dim=256, state_dim=768, heads=4, kvh=2, hd=64, seed=7):
        self.rt, self.images, self.states, self.heads, self.kvh, self.hd, self.dim = rt, images, states, heads, kvh, hd, dim
        self.kv = rt.cross_kv(kind, images, states, kvh, hd)
        self.values = {}

        def linear(name, k, n, gamma=None):
            bias = seeded.normal(seed + len(name), n, 0.1)
            g = None if gamma is None else np.full(n, gamma, np.float32)
            if name == "fc1":
                codes = ref.e4m3((seeded.normal(seed + 2, n * k, 40.0).reshape(n, k)).clip(-448, 448))
                scales = np.full(ref.blocks(n) * ref.blocks(k), 0.001 / 3)
                self.values[name] = (ref.block_values(codes, scales.astype(np.float32)), bias, g)
                return rt.prepare_linear_fp8_blocks(k, n, codes, scales, bias, g)
            w = seeded.normal(seed + 2 * len(name), k * n, 0.05).reshape(k, n)
            self.values[name] = (ref.values(*ref.quantise(np.ascontiguousarray(w.T))), bias, g)
            return rt.prepare_linear_fp8(k, n, w, bias, g)

        self.to_kv = linear("to_kv", state_dim, 2 * kvh * hd)
        self.to_q = linear("q", dim, heads * hd)
        self.proj = linear("proj", heads * hd, dim, 0.5)
        self.fc1, self.fc2 = linear("fc1", dim, 4 * dim), linear("fc2", 4 * dim, dim, 0.5)
        self.ones, self.zeros = rt.upload_f32(np.ones(dim)), rt.upload_f32(np.zeros(dim))
        rows = images * most
        self.kv_rows = rt.alloc_f32(images * states * 2 * kvh * hd)
        self.q, self.o = rt.alloc_f32(rows * heads * hd), rt.alloc_f32(rows * heads * hd)
        self.hidden = rt.alloc_f32(rows * 4 * dim)

    def read_states(self, quantised, seen):
        self.to_kv.run_rows(quantised, self.kv_rows)
        self.kv.write_rows(self.kv_rows, self.states, seen=seen)

    def attend(self, h, x, n):
        """x += proj(attention(q(h))) for n tokens an image."""
        rows = self.images * n
        self.to_q.run(h, rows, self.q)
        self.kv.attention(self.q, self.heads, n, self.o, token_major=True)
        self.proj.run_residual(self.o, rows, x)

    def mlp(self, h, x, n):
        rows = self.images * n
        self.fc1.run_gelu(h, rows, self.hidden)
        self.fc2.run_residual(self.hidden, rows, x)

    def check(self, name, x, got, before=None, gelu=False):
        w, bias, g = self.values[name]
        k = w.shape[1]
        v = ref.values(*ref.quantise(x))
        y, size = v @ w.T + bias, np.abs(v) @ np.abs(w).T + np.abs(bias)
        extra = 0.0
        if gelu:
            y, size, extra = ref.gelu(y), 1.13 * size, 1e-6 * np.maximum(1, np.abs(y))
        if g is not None:
            y, size = y * g, size * np.abs(g)
        if before is not None:
            y, size = y + before, size + np.abs(before)
        _close(got.reshape(y.shape), y, size, k, extra)


@pytest.mark.parametrize("kind", KINDS)
def test_a_decoder_behind_an_encoder_block(rt, kind):
    """Two images' states from an encoder block, quantised once for two layers; some masked; 40 tokens, then
    single ones."""
    images, tokens, dim = 2, 1 + 6 * 7, 256
    block = rt.prepare_block(da3.block_weights(seed=3))
    x0 = rt.upload_f32(seeded.normal(1, images * tokens * 768))
    rt.vit_block_run(block, x0, images, tokens, da3.positions_yx(6, 7))
    states = rt.download_f32(x0).reshape(images * tokens, 768)
    quantised = rt.quantize_fp8(x0, images * tokens, 768)
    mask = (np.arange(images * tokens) % 5 != 3).astype(int)
    mask[tokens:tokens + 30] = 0
    seen = rt.upload_i32(mask)
    layers = [Layer(rt, kind, images, tokens, 40, seed=s) for s in (7, 70)]
    stored = []
    for layer in layers:
        layer.read_states(quantised, seen)
        rows = rt.download_f32(layer.kv_rows)
        layer.check("to_kv", states, rows)
        both = rows.reshape(images, tokens, 2, layer.kvh, layer.hd)
        stored.append([ref.stored(both[i, :, 0], both[i, :, 1], kind, mask[i * tokens:(i + 1) * tokens])
                       for i in range(images)])
    for step, n in enumerate([40, 1, 1]):
        rows = images * n
        x = rt.upload_f32(seeded.normal(30 + step, rows * dim))
        for layer, held in zip(layers, stored):
            # The buffers of a call have its size.
            layer.q, layer.o = rt.alloc_f32(rows * 256), rt.alloc_f32(rows * 256)
            layer.hidden = rt.alloc_f32(rows * 1024)
            before = rt.download_f32(x).reshape(rows, dim)
            h = rt.layernorm_f32(x, layer.ones, layer.zeros, rows, dim, 1e-6)
            layer.attend(h, x, n)
            q, o = (rt.download_f32(t).reshape(images, n, layer.heads, layer.hd) for t in (layer.q, layer.o))
            layer.check("q", rt.download_f32(h).reshape(rows, dim), q)
            for i in range(images):
                close(o[i], q[i], *held[i])
            after = rt.download_f32(x).reshape(rows, dim)
            layer.check("proj", o.reshape(rows, -1), after, before)
            h = rt.layernorm_f32(x, layer.ones, layer.zeros, rows, dim, 1e-6)
            layer.mlp(h, x, n)
            hidden = rt.download_f32(layer.hidden).reshape(rows, -1)
            layer.check("fc1", rt.download_f32(h).reshape(rows, dim), hidden, gelu=True)
            layer.check("fc2", hidden, rt.download_f32(x), after)


class Step:
    """A layer's states and one step of n tokens an image on buffers of its own, the states written anew each time."""

    def __init__(self, rt, kind, n, images=2, states=300, seed=7):
        self.rt, self.n, self.images = rt, n, images
        self.layer = Layer(rt, kind, images, states, n, seed=seed)
        self.x0 = rt.alloc_f32(images * states * 768)
        self.quantised = rt.alloc_fp8(images * states, 768)
        self.h, self.x = rt.alloc_f32(images * n * 256), rt.alloc_f32(images * n * 256)
        self.seen = rt.alloc_i32(images * states)

    def feed(self, seed):
        rt = self.rt
        for t, s in ((self.x0, 1), (self.h, 2), (self.x, 3)):
            v = rt.upload_f32(seeded.normal(100 * seed + s, len(t)))
            rt.copy_segment_into_f32(t, 0, v, 0, len(t))
        rt.synchronize()

    def run(self, seen=None):
        rt, layer = self.rt, self.layer
        rt.quantize_fp8_into(self.x0, self.images * layer.states, 768, self.quantised)
        layer.read_states(self.quantised, seen)
        layer.attend(self.h, self.x, self.n)
        layer.mlp(self.h, self.x, self.n)

    def take(self):
        return self.rt.download_f32(self.x)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 30, 150])
def test_a_graph_of_a_step_replays_what_runs_eagerly(rt, kind, n):
    hip, stream = _hip(), ctypes.c_void_p(rt.stream())
    eager, step = Step(rt, kind, n), Step(rt, kind, n)
    eager.feed(1)
    eager.run()
    graph, exe = _capture(hip, stream, step.run)
    try:
        for i in range(5):
            eager.feed(i)
            eager.run()
            exp = eager.take()
            step.feed(i)
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            assert_bits_equal(step.take(), exp, f"replay {i}")
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("n", [1, 60])
def test_graphs_on_several_streams_at_once(rt, n):
    """Three graphs of one runtime replayed on streams of their own while the runtime runs a step itself: no two of
    them share a workspace."""
    hip = _hip()
    hip.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    hip.hipStreamDestroy.argtypes = [ctypes.c_void_p]
    stream = ctypes.c_void_p(rt.stream())
    steps = [Step(rt, "f16", n, states=500, seed=7 + i) for i in range(3)]
    own = Step(rt, "f16", 2 * n, states=600, seed=70)
    made, streams = [], []
    try:
        for i, s in enumerate(steps):
            s.feed(i)
            own.feed(9)
            own.run()  # room for the capture that follows
            rt.synchronize()
            made.append(_capture(hip, stream, s.run))
            streams.append(ctypes.c_void_p())
            assert hip.hipStreamCreateWithFlags(ctypes.byref(streams[-1]), 1) == 0
        exp = []
        for i, ((_, e), s) in enumerate(zip(made, steps)):
            s.feed(i)
            assert hip.hipGraphLaunch(e, stream) == 0
            exp.append(s.take())
        own.feed(9)
        own.run()
        first = own.take()
        for _ in range(4):
            for i, s in enumerate(steps):
                s.feed(i)
            own.feed(9)
            for (_, e), t in zip(made, streams):
                assert hip.hipGraphLaunch(e, t) == 0
            own.run()
            for t in streams:
                assert hip.hipStreamSynchronize(t) == 0
            for s, e in zip(steps, exp):
                assert_bits_equal(s.take(), e, "at once")
            assert_bits_equal(own.take(), first, "the runtime's own")
    finally:
        for g, e in made:
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)
        for t in streams:
            hip.hipStreamDestroy(t)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 200])
def test_a_graph_of_a_size_that_has_not_run(kind, n):
    """The attention goes without room for parts: right, and the same on every replay.  A projection that needs a
    workspace is refused, nothing of it recorded."""
    rt = vh.Runtime(0)  # its own, without workspaces
    hip, stream = _hip(), ctypes.c_void_p(rt.stream())
    s = States(rt, kind, 2, 700, 2, 64, 0.9)
    q = seeded.normal(3, 2 * n * 4 * 64).reshape(2, n, 4, 64)
    qt, out = rt.upload_f32(q), rt.upload_f32(np.zeros(q.size))
    lin = rt.prepare_linear_fp8(256, 256, seeded.normal(1, 256 * 256, 0.05))
    x, y = rt.upload_f32(seeded.normal(2, 200 * 256)), rt.upload_f32(np.full(200 * 256, 7.0))
    rt.synchronize()

    def run():
        with pytest.raises(vh.UploadError, match="once before"):
            lin.run(x, 200, y)
        with pytest.raises(vh.KernelError):
            rt.cross_kv(kind, 1, 10, 1, 64)
        s.kv.attention(qt, 4, n, out, token_major=True)

    graph, exe = _capture(hip, stream, run)
    try:
        got = []
        for _ in range(3):
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            got.append(rt.download_f32(out).reshape(q.shape))
            rt.copy_segment_into_f32(out, 0, rt.upload_f32(np.zeros(q.size)), 0, q.size)
            s.run(q)
        for i in range(2):
            close(got[0][i], q[i], s.k[i], s.v[i])
        for g in got[1:]:
            assert_bits_equal(g, got[0])
        assert (rt.download_f32(y) == 7.0).all()
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


def test_runtimes_in_threads_of_their_own():
    exp, got = {}, {}

    def work(seed, to):
        rt = vh.Runtime(0)
        step = Step(rt, KINDS[seed % 2], 20 + seed, seed=seed)
        for i in range(4):
            step.feed(i)
            step.run()
            to[seed, i] = step.take()

    for seed in range(4):
        work(seed, exp)
    threads = [threading.Thread(target=work, args=(seed, got)) for seed in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got.keys() == exp.keys()
    for key, e in exp.items():
        assert_bits_equal(got[key], e, str(key))


def test_a_call_on_another_runtimes_memory_is_refused_and_changes_nothing(rt):
    other = vh.Runtime(0)
    step, x = Step(rt, "f16", 3), other.upload_f32(np.full(2 * 3 * 256, 5.0))
    step.feed(1)
    with pytest.raises(vh.InvalidArgument):
        step.layer.fc2.run_residual(step.layer.hidden, 6, x)
    with pytest.raises(vh.InvalidArgument):
        step.layer.kv.attention(step.layer.q, 4, 3, x)
    assert (other.download_f32(x) == 5.0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_states_past_4_gib(rt, kind):
    """Images whose keys and values lie past 4 GiB give the first one's bits; the first is checked."""
    images, tokens, kvh, hd = (42, 65536, 4, 128) if kind == "f16" else (22, 65536, 4, 128)
    n = tokens * kvh * hd
    k, v = (seeded.normal(i + 1, n) for i in (0, 1))
    big = []
    for x in (k, v):
        one, t = rt.upload_f32(x), rt.alloc_f32(images * n)
        for i in range(images):
            rt.copy_segment_into_f32(t, i * n, one, 0, n)
        big.append(t)
    kv = rt.cross_kv(kind, images, tokens, kvh, hd)
    kv.write(*big, tokens, token_major=True)
    del big
    k, v = (x.reshape(tokens, kvh, hd) for x in (k, v))
    held = ref.stored(k, v, kind)
    for queries in (1, 70):
        q = np.tile(seeded.normal(9, queries * 8 * hd), images)
        out = rt.alloc_f32(q.size)
        kv.attention(rt.upload_f32(q), 8, queries, out, token_major=True)
        got = rt.download_f32(out).reshape(images, queries, 8, hd)
        close(got[0], q[:queries * 8 * hd].reshape(queries, 8, hd), *held)
        # An image's keys are shared out in another place for each: the sums' order differs.  Both are within 2^-21
        # (2 + |s|) sum p |v| of what is exact (test_gpu_cross), so within twice that of each other, and sum p |v|
        # over 65536 keys of N(0, 1) is their mean |v| to within some percent: 2^-20 of it is less.
        assert np.abs(got[1:] - got[:1]).max() <= 2.0 ** -20 * np.abs(v).mean()


def test_rows_past_4_gib(rt):
    """2^21 + 5 rows of 2100 values: codes past 4 GiB, floats past 16; the last rows as the first."""
    rows, k, n, part = 2 ** 21 + 5, 2100, 16, 4096
    x = seeded.normal(1, part * k)
    one, t = rt.upload_f32(x), rt.alloc_f32(rows * k)
    for at in range(0, rows, part):
        rt.copy_segment_into_f32(t, at * k, one, 0, min(part, rows - at) * k)
    w = seeded.normal(2, k * n, 0.05).reshape(k, n)
    lin, out = rt.prepare_linear_fp8(k, n, w), rt.alloc_f32(rows * n)
    lin.run(t, rows, out)
    got = rt.download_f32(out).reshape(rows, n)
    x = x.reshape(part, k)
    vx, vw = ref.values(*ref.quantise(x)), ref.values(*ref.quantise(np.ascontiguousarray(w.T)))
    _close(got[:part], vx @ vw.T, np.abs(vx) @ np.abs(vw).T, k)
    for at in range(0, rows, part):
        assert_bits_equal(got[at:at + part], got[:min(part, rows - at)])
    q = rt.quantize_fp8(t, rows, k)
    rt.dequantize_fp8_into(q, t)
    last = rt.copy_segment_f32(t, (rows - 5) * k, 5 * k)
    assert_bits_equal(rt.download_f32(last).reshape(5, k), vx[:5].astype(np.float32))
