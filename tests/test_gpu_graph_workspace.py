"""Workspaces of captured calls on the GPU: what a runtime has queued and what a graph of the same calls does on another
stream at the same time leave each other alone, with no wait between the eager calls, the capture and the replays."""
import ctypes

import numpy as np
import pytest

import vestra_hip as vh
from conftest import assert_bits_equal
from test_gpu_cross import States
from test_gpu_graph import _capture, _hip
from test_gpu_stream_attention import Stream
from test_gpu_stream_frames import Call
from vestra_hip import seeded

pytestmark = pytest.mark.gpu


class Projection:
    """Floats through an 8-bit projection: the quantised rows are in the workspace."""

    def __init__(self, rt, seed, rows):
        self.rt, self.rows = rt, rows
        self.lin = rt.prepare_linear_fp8(512, 384, seeded.normal(seed, 512 * 384, 0.05))
        self.x, self.out = rt.upload_f32(seeded.normal(seed + 1, rows * 512)), rt.alloc_f32(rows * 384)

    def run(self):
        self.lin.run(self.x, self.rows, self.out)

    def take(self):
        return self.rt.download_f32(self.out)


class Cross:
    """Queries over an encoder's states: parts and counters of the tiles."""

    def __init__(self, rt, seed, n):
        self.rt, self.n = rt, n
        self.states = States(rt, "f16", 1, 3000, 2, 64, seed=seed)
        self.q, self.out = rt.upload_f32(seeded.normal(seed + 5, n * 4 * 64)), rt.alloc_f32(n * 4 * 64)

    def run(self):
        self.states.kv.attention(self.q, 4, self.n, self.out, token_major=True)

    def take(self):
        return self.rt.download_f32(self.out)


def _paged(rt, seed, n):
    return Call(Stream(rt, "f32", [n, 1], [5000, 700], 4, 2, 64, 16, seed=seed))


@pytest.mark.parametrize("kind, size", [(Projection, 40), (Projection, 3000), (Cross, 1), (Cross, 300), (_paged, 1),
                                        (_paged, 200)])
def test_queued_calls_and_a_graph_at_once(kind, size):
    rt, hip = vh.Runtime(0), _hip()
    hip.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    hip.hipStreamDestroy.argtypes = [ctypes.c_void_p]
    stream, other = ctypes.c_void_p(rt.stream()), ctypes.c_void_p()
    own, recorded = [kind(rt, 10 * i + 1, size) for i in range(4)], kind(rt, 91, size)
    rt.synchronize()
    for c in own + [recorded]:
        c.run()
    exp = [c.take() for c in own + [recorded]]
    k = 4096
    slow = rt.prepare_linear_f32(k, k, seeded.normal(5, k * k, 0.01), np.zeros(k))
    x, y = rt.upload_f32(seeded.normal(6, k * k)), rt.upload_f32(np.zeros(k * k))
    slow.run_residual(x, k, y)
    rt.synchronize()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(other), 1) == 0
    made = []
    try:
        for _ in range(3):
            for _ in range(3):  # a few ms, behind which the calls wait
                slow.run_residual(x, k, y)
            for _ in range(10):
                for c in own:
                    c.run()
            made.append(_capture(hip, stream, recorded.run))
            for _ in range(400):  # past the moment in which the queued calls run
                assert hip.hipGraphLaunch(made[-1][1], other) == 0
            rt.synchronize()
            assert hip.hipStreamSynchronize(other) == 0
            for c, e in zip(own + [recorded], exp):
                assert_bits_equal(c.take(), e, "at once")
    finally:
        rt.synchronize()
        for g, e in made:
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)
        hip.hipStreamDestroy(other)


@pytest.mark.parametrize("kind", [Cross, _paged])
def test_each_capture_behind_a_call_of_its_size_has_room(kind):
    """Graphs captured one after the other, each behind one call: the same bits as that call, which shares its keys
    among several workgroups; also behind a larger and a smaller one."""
    rt, hip = vh.Runtime(0), _hip()
    stream = ctypes.c_void_p(rt.stream())
    calls = [kind(rt, 7 * i + 1, n) for i, n in enumerate((1, 200, 1))]
    made = []
    try:
        for c in calls:
            c.run()
            exp = c.take()
            made.append(_capture(hip, stream, c.run))
            for _ in range(3):
                assert hip.hipGraphLaunch(made[-1][1], stream) == 0
                assert hip.hipStreamSynchronize(stream) == 0
                assert_bits_equal(c.take(), exp)
    finally:
        for g, e in made:
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)
