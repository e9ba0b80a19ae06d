"""CPU checks of the entry points of 8-bit floating point and of an encoder's states: null handles and pointers are refused before any device
call, and what the float64 reference of their tests stands on is checked against torch and by hand."""
import ctypes

import numpy as np
import pytest
import torch

import fp8_64 as ref
import vestra_hip as vh


def test_null_handles_are_refused():
    L, out, n = vh.lib(), ctypes.c_void_p(), None
    calls = [
        ("vh_fp8_alloc", (n, 1, 1, ctypes.byref(out))), ("vh_fp8_upload", (n, n, n, 1, 1, ctypes.byref(out))),
        ("vh_fp8_download", (n, n, n, n)), ("vh_quantize_fp8", (n, n, 1, 1, ctypes.byref(out))),
        ("vh_quantize_fp8_into", (n, n, 1, 1, n)), ("vh_dequantize_fp8_into", (n, n, n)),
        ("vh_gemm_fp8_into", (n, n, n, n)), ("vh_prepare_linear_fp8", (n, 1, 1, n, n, n, ctypes.byref(out))),
        ("vh_prepare_linear_fp8_blocks", (n, 1, 1, n, n, n, n, ctypes.byref(out))),
        ("vh_linear_fp8_run", (n, n, 1, n)), ("vh_linear_fp8_run_gelu", (n, n, 1, n)),
        ("vh_linear_fp8_run_residual", (n, n, 1, n)), ("vh_linear_fp8_run_rows", (n, n, n)),
        ("vh_linear_fp8_run_rows_gelu", (n, n, n)), ("vh_linear_fp8_run_rows_residual", (n, n, n)),
        ("vh_cross_kv_new", (n, 0, 1, 1, 1, 64, ctypes.byref(out))), ("vh_cross_kv_write_f32", (n, n, n, 1, 0, n)),
        ("vh_cross_kv_write_rows_f32", (n, n, 1, n)), ("vh_cross_kv_read_f32", (n, n, n, n)),
        ("vh_cross_attention_f32", (n, n, 1, 1, 0, n))]
    for name, args in calls:
        assert getattr(L, name)(*args) == vh.InvalidArgument.status, name
        assert b"null" in L.vh_last_error() and out.value is None
    assert L.vh_fp8_rows(None) == 0 and L.vh_fp8_k(None) == 0
    assert L.vh_linear_fp8_input_features(None) == 0 and L.vh_linear_fp8_output_features(None) == 0
    L.vh_fp8_free(None)
    L.vh_linear_fp8_free(None)
    L.vh_cross_kv_free(None)


def test_buffers_of_another_size_are_refused():
    with pytest.raises(vh.InvalidArgument):
        vh._vector(np.zeros(5), 6)
    with pytest.raises(vh.InvalidArgument):
        vh._bytes(np.zeros(6, np.uint8), 5)
    with pytest.raises(vh.InvalidArgument):
        vh._bytes(np.zeros(5, np.int32), 5)
    assert vh._bytes(np.array([-1], np.int8), 1)[0] == 255


def test_reference_codes_are_torchs():
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.VALUES, v, equal_nan=True)
    rng = np.random.default_rng(1)
    # Every code, every midpoint between two, and random values.
    grid = ref.VALUES[:127]
    x = np.concatenate([grid, (grid[1:] + grid[:-1]) / 2, rng.normal(size=4000) * 60, rng.normal(size=4000) * 2.0 ** -8])
    x = np.concatenate([x, -x]).clip(-448, 448)
    assert np.array_equal(ref.e4m3(x), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_reference_blocks_by_hand():
    x = np.zeros((1, 130), np.float32)
    x[0, :3] = [448.0, 449.0, -1.0]
    x[0, 128:] = [np.inf, 3.0]
    codes, exps = ref.quantise(x)
    assert list(exps[0] - 127.0) == [1, -7]  # 449 needs 2; 3 = 384 * 2^-7
    assert list(ref.values(codes, exps)[0, :3]) == [448, 448, -1] and ref.values(codes, exps)[0, 129] == 3
    assert codes[0, 128] == 127
    assert np.allclose(ref.gelu(np.array([0.0, 1.0, -2.0])), [0, 0.8413447460685429, -0.04550026389635842])


def test_reference_states_by_hand():
    k = np.array([[[3.0, 1.0]], [[np.nan, 5.0]], [[-0.75, 0.1]]], np.float32)
    a, b = ref.stored(k, k, "f16", np.array([1, 0, 2]))
    assert a.shape == (2, 1, 2) and list(a[:, 0, 0]) == [3.0, -0.75]
    assert abs(a[1, 0, 1] - np.float32(0.1)) <= 2.0 ** -11 * 0.1 and a[1, 0, 1] == b[1, 0, 1]
    c, _ = ref.stored(k, k, "f32", np.array([1, 0, 2]))
    assert abs(c[1, 0, 1] - np.float32(0.1)) <= 2.0 ** -22 * 0.1
    q = np.array([[[1.0, 0.0], [0.0, 2.0]]])
    got = ref.attention(q, a, b)
    for h in range(2):
        w = [np.exp(q[0, h] @ a[j, 0] / np.sqrt(2)) for j in range(2)]
        assert np.allclose(got[0, h], (w[0] * b[0, 0] + w[1] * b[1, 0]) / sum(w))
    assert not ref.attention(q, a[:0], b[:0]).any()
