"""CPU checks of the stream operators' entry points: null handles and pointers are refused before any device call,
and what the float64 reference of their tests stands on is itself checked against closed forms."""
import ctypes

import numpy as np
import pytest

import stream64 as ref
import vestra_hip as vh


def test_null_handles_are_refused():
    L, out, n = vh.lib(), ctypes.c_void_p(), None
    calls = [
        ("vh_upload_i32", (n, n, 4, ctypes.byref(out))), ("vh_download_i32", (n, n, n, 0)),
        ("vh_index_alloc", (n, 4, ctypes.byref(out))),
        ("vh_prepare_rope_axes", (n, 64, 1, (ctypes.c_size_t * 1)(4), 100.0, 0, ctypes.byref(out))),
        ("vh_rope_axes_run", (n, n, 1, 1, 0, n, n)), ("vh_kv_cache_new", (n, 0, 1, 16, 1, 64, ctypes.byref(out))),
        ("vh_kv_cache_append_f32", (n, n, n, 1, 0, n)), ("vh_kv_cache_append_qkv_f32", (n, n, n, 1, 1, n, n, n)),
        ("vh_kv_cache_gather_f32", (n, n, 1, n, n)),
        ("vh_kv_pages_assign", (n, n, n, 1, n, n, 16, n, 1, n, n, n, 1, n)),
        ("vh_kv_cache_attention_f32", (n, n, 1, 1, 1, n, 1, n, n, 0, 0, n))]
    for name, args in calls:
        assert getattr(L, name)(*args) == vh.InvalidArgument.status, name
        assert b"null" in L.vh_last_error() and out.value is None
    assert L.vh_index_len(None) == 0 and not L.vh_index_device_ptr(None) and L.vh_kv_cache_slots(None) == 0
    for name in ("vh_index_free", "vh_rope_free", "vh_kv_cache_free"):
        getattr(L, name)(None)


def test_values_outside_int32_are_refused():
    assert list(vh._i32([0.0, -2**31, 2**31 - 1])) == [0, -2**31, 2**31 - 1] and vh._i32([]).size == 0
    for bad in (np.array([2**31]), [-2**31 - 1], [0.5], [np.nan], np.array([2**32 + 5])):
        with pytest.raises(vh.InvalidArgument):
            vh._i32(bad)


def test_reference_rotation_keeps_lengths_and_relative_angles():
    x = np.random.default_rng(1).normal(size=(2, 1, 64))
    a, b = (ref.rotate(x, np.array([[p], [p + 7]]), [32], 10000.0, True) for p in (0, 1000))
    assert np.allclose((a ** 2).sum(-1), (x ** 2).sum(-1))
    assert np.isclose((a[0] * a[1]).sum(), (b[0] * b[1]).sum())
    assert np.allclose(ref.rotate(x, np.zeros((2, 2), int), [3, 5], 100.0, False), x)


@pytest.mark.parametrize("block, window", [(0, 0), (1, 0), (3, 0), (1, 4), (3, 4), (0, 5)])
def test_reference_attention_by_hand(block, window):
    """Two heads over one of the cache, four new tokens of nine, key by key."""
    rng = np.random.default_rng(2)
    q, k, v = rng.normal(size=(4, 2, 8)), rng.normal(size=(9, 1, 8)), rng.normal(size=(9, 1, 8))
    got = ref.attention(q, [k], [v], [0, 4], [9], 2, block, window)
    for i in range(4):
        pos = 5 + i
        hi = 9 if block == 0 else min(9, (pos // block + 1) * block)
        keys = range(max(0, hi - window) if window else 0, hi)
        for h in range(2):
            w = np.array([np.exp(q[i, h] @ k[j, 0] / np.sqrt(8)) for j in keys])
            assert np.allclose(got[i, h], sum(x * v[j, 0] for x, j in zip(w, keys)) / w.sum())


def test_reference_roundings():
    x = np.float32([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -3.3895314e38, 0.0])
    assert list(ref.bf16(x)) == [1.0, 1.0, np.float32(1 + 2.0 ** -6), np.float32(-3.3895314e38), 0.0]
    y = ref.q8_0(np.linspace(-127, 127, 32, dtype=np.float32)[None] / 2)
    assert np.array_equal(y[0], np.copysign(np.floor(np.abs(np.linspace(-127, 127, 32)) + 0.5), y[0]) / 2)


def test_reference_pages_by_hand():
    starts, lens, slots, table, taken = ref.pages([3, 0], [2, 5], [9, 8, 7], 0, 4, [[5, -1], [-1, -1]], 8)
    assert list(starts) == [0, 2, 7] and list(lens) == [5, 5] and taken == 3
    assert list(slots) == [23, 36, 32, 33, 34, 35, 28, -1] and table.tolist() == [[5, 9], [8, 7]]
