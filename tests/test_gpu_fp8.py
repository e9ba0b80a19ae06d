"""Rows in 8-bit floating point and the projections on them on the GPU, against float64 numpy (tests/fp8_64.py).

Codes and exponents are compared bit for bit.  A product's tolerance: every product of two codes is exact in
f32; each of the K / 32 instructions rounds what it adds to at most 2^-23 of the sum of the magnitudes so far, and
scales, bias, gamma and residual round a handful of times more: (K / 32 + 8) 2^-23 of sum |a b| + |bias|
covers it, a factor of two or more above what is expected."""
import numpy as np
import pytest

import fp8_64 as ref
import vestra_hip as vh
from conftest import assert_bits_equal
from vestra_hip import seeded

pytestmark = pytest.mark.gpu


def _rows(seed, rows, k, spread=0.0):
    x = seeded.normal(seed, rows * k).reshape(rows, k)
    if spread:
        x = x * np.exp2(spread * seeded.normal(seed + 1, rows * ref.blocks(k))).reshape(rows, -1).repeat(128, 1)[:, :k]
    return x.astype(np.float32)


def _uploaded(rt, x):
    return rt.quantize_fp8(rt.upload_f32(x), *x.shape)


@pytest.mark.parametrize("rows, k", [(1, 1), (1, 127), (3, 128), (15, 129), (17, 130), (33, 1000), (865, 768),
                                     (16, 5003), (4099, 96), (70000, 4)])
@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_quantise_is_exact(rt, rows, k, spread):
    x = _rows(rows + k, rows, k, spread)
    t = _uploaded(rt, x)
    assert (t.rows, t.k) == (rows, k)
    codes, exps = rt.fp8_download(t)
    want, want_exps = ref.quantise(x)
    assert np.array_equal(exps, want_exps) and np.array_equal(codes, want)
    out = rt.upload_f32(np.full(rows * k, 7.0))
    rt.dequantize_fp8_into(t, out)
    assert_bits_equal(rt.download_f32(out), ref.values(want, want_exps).astype(np.float32).reshape(-1))


def test_quantise_at_the_borders(rt):
    """Midpoints between codes, both ends of the range of floats, the border between two exponents, NaN,
    infinities and zeros of either sign."""
    grid = ref.VALUES[:127]
    x = np.zeros((8, 256), np.float32)
    x[0, :126] = (grid[1:] + grid[:-1]) / 2
    x[0, 126] = 448
    x[1] = -x[0]
    x[2, ::5] = [np.float32(448 * 2.0 ** e) for e in range(-26, 26)]
    x[3, 0], x[3, 130] = np.finfo(np.float32).max, np.float32(1e-45)
    x[4, 1::2], x[4, 0], x[4, 130] = 2.0 ** -130, np.float32(448 * 2.0 ** -127), -2.0 ** -136
    x[5, 3:6], x[5, 9] = [np.nan, np.inf, -np.inf], 5.0
    x[6] = -0.0
    x[7, :128], x[7, 128:] = np.nan, np.nextafter(np.float32(448), np.float32(500))
    t = _uploaded(rt, x)
    codes, exps = rt.fp8_download(t)
    want, want_exps = ref.quantise(x)
    nan = want == 127
    assert np.array_equal(exps, want_exps)
    assert np.array_equal(codes[~nan], want[~nan]) and (codes[nan] & 127 == 127).all()
    again = rt.fp8_upload(codes, exps, 8, 256)
    assert all(np.array_equal(a, b) for a, b in zip(rt.fp8_download(again), (codes, exps)))


def test_quantise_into_what_held_more(rt):
    """Codes and exponents of an earlier call leave nothing behind; two calls in a row give the same bits."""
    t = rt.alloc_fp8(40, 300)
    for seed, scale in ((1, 1e30), (2, 1e-30), (2, 1e-30)):
        x = _rows(seed, 40, 300) * np.float32(scale)
        rt.quantize_fp8_into(rt.upload_f32(x), 40, 300, t)
        assert all(np.array_equal(a, b) for a, b in zip(rt.fp8_download(t), ref.quantise(x)))


def _close(got, exact, size, k, extra=0.0):
    """size: the sum of the magnitudes of an output's terms."""
    bound = (k / 32 + 8) * 2.0 ** -23 * size + extra
    worst = np.max(np.abs(got.astype(np.float64) - exact) / np.maximum(bound, 1e-300)) if got.size else 0.0
    assert np.isfinite(got).all() and worst <= 1.0, worst


SHAPES = [(1, 1, 1), (1, 768, 2304), (3, 129, 5), (16, 130, 17), (17, 96, 130), (40, 1000, 260), (64, 3000, 33),
          (65, 256, 1000), (129, 127, 129), (200, 2200, 301), (865, 768, 768), (1000, 520, 1100), (2500, 64, 2100),
          (5000, 16, 3)]


@pytest.mark.parametrize("m, k, n", SHAPES)
def test_gemm_against_float64(rt, m, k, n):
    a, b = _rows(m, m, k, 3.0), _rows(n + 7, n, k, 1.0)
    va, vb = (ref.values(*ref.quantise(x)) for x in (a, b))
    c = rt.upload_f32(np.full(m * n, np.nan))
    rt.gemm_fp8_into(_uploaded(rt, a), _uploaded(rt, b), c)
    _close(rt.download_f32(c).reshape(m, n), va @ vb.T, np.abs(va) @ np.abs(vb).T, k)


def _linear(rt, kind, k, n, bias, gamma, seed=3):
    """The prepared linear and its weights' values [N, K]."""
    if kind == "rows":
        w = seeded.normal(seed, k * n, 0.05).reshape(k, n)
        w[:, n // 2] *= 50.0
        return rt.prepare_linear_fp8(k, n, w, bias, gamma), ref.values(*ref.quantise(np.ascontiguousarray(w.T)))
    codes = ref.e4m3((seeded.normal(seed, n * k, 40.0).reshape(n, k)).clip(-448, 448))
    scales = seeded.normal(seed + 1, ref.blocks(n) * ref.blocks(k), 0.01)  # of either sign
    scales[-1] = 0.0
    return rt.prepare_linear_fp8_blocks(k, n, codes, scales, bias, gamma), ref.block_values(codes, scales)


@pytest.mark.parametrize("kind", ["rows", "blocks"])
@pytest.mark.parametrize("m, k, n", SHAPES)
def test_linear_against_float64(rt, kind, m, k, n):
    """run with bias and gamma, run_gelu, run_residual; from floats and from rows quantised before, with
    the same bits."""
    x, bias, gamma, res = _rows(m + 1, m, k), seeded.normal(5, n), seeded.normal(6, n), seeded.normal(7, m * n)
    vx = ref.values(*ref.quantise(x))
    xt, rows = rt.upload_f32(x), _uploaded(rt, x)

    def both(run, run_rows):
        out, again = (rt.upload_f32(res) for _ in range(2))
        run(xt, m, out)
        run_rows(rows, again)
        got = rt.download_f32(out)
        assert_bits_equal(rt.download_f32(again), got)
        return got.reshape(m, n)

    lin, vw = _linear(rt, kind, k, n, bias, gamma)
    assert (lin.input_features(), lin.output_features()) == (k, n)
    y, size = vx @ vw.T + bias, np.abs(vx) @ np.abs(vw).T + np.abs(bias)
    _close(both(lin.run, lin.run_rows), y * gamma, size * np.abs(gamma), k)
    r = res.reshape(m, n)
    _close(both(lin.run_residual, lin.run_rows_residual), y * gamma + r, size * np.abs(gamma) + np.abs(r), k)
    lin, vw = _linear(rt, kind, k, n, bias, None)
    # The slope of GELU is at most 1.13, its fast form within 1e-6 max(1, |v|).
    _close(both(lin.run_gelu, lin.run_rows_gelu), ref.gelu(y), 1.13 * size, k, 1e-6 * np.maximum(1, np.abs(y)))
    lin, vw = _linear(rt, kind, k, n, None, None)
    _close(both(lin.run, lin.run_rows), vx @ vw.T, np.abs(vx) @ np.abs(vw).T, k)


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_rows_of_wide_range(rt, m):
    """Blocks of a row whose exponents differ by up to 60: those far below the largest count to within
    2^-25 of 2^E, E the row's largest exponent."""
    k, n = 1024, 48
    a, b = _rows(m, m, k, 12.0), _rows(9, n, k, 12.0)
    (ca, ea), (cb, eb) = ref.quantise(a), ref.quantise(b)
    va, vb = ref.values(ca, ea), ref.values(cb, eb)
    c = rt.alloc_f32(m * n)
    rt.gemm_fp8_into(_uploaded(rt, a), _uploaded(rt, b), c)
    big = [np.ldexp(1.0, e.max(1).astype(int) - 127 - 25)[:, None] for e in (ea, eb)]
    lost = big[0] @ np.abs(vb).sum(1)[None] + np.abs(va).sum(1)[:, None] @ big[1].T + k * big[0] @ big[1].T
    _close(rt.download_f32(c).reshape(m, n), va @ vb.T, np.abs(va) @ np.abs(vb).T, k, lost)


@pytest.mark.parametrize("m", [1, 40, 200, 1000, 20000])
@pytest.mark.parametrize("power", [-120, 0, 116])
def test_block_scales_of_any_size(rt, m, power):
    """Scales of a checkpoint whose product with a block's sum is no float, where that with the row's exponent
    is: rows of the size that the scales are not."""
    k, n = 300, 200
    x = _rows(5, m, k) * np.float32(2.0 ** -power)
    codes = ref.e4m3(seeded.normal(6, n * k, 40.0).reshape(n, k).clip(-448, 448))
    scales = seeded.normal(7, ref.blocks(n) * ref.blocks(k)) * np.float32(2.0 ** power)
    scales[:3] *= np.float32(2.0 ** 9)  # 128 rows of their own size
    lin = rt.prepare_linear_fp8_blocks(k, n, codes, scales)
    out = rt.upload_f32(np.full(m * n, np.nan))
    lin.run(rt.upload_f32(x), m, out)
    va, vb = ref.values(*ref.quantise(x)), ref.block_values(codes, scales)
    _close(rt.download_f32(out).reshape(m, n), va @ vb.T, np.abs(va) @ np.abs(vb).T, k)


def test_more_rows_than_a_launch_has_in_a_direction(rt):
    """Of a few columns: 65536 workgroups of 16 rows, and 17 rows."""
    m, k, n = 65536 * 16 + 17, 20, 7
    x, w = _rows(1, m, k), seeded.normal(2, k * n, 0.1).reshape(k, n)
    lin = rt.prepare_linear_fp8(k, n, w)
    out = rt.upload_f32(np.full(m * n, np.nan))
    lin.run(rt.upload_f32(x), m, out)
    va, vb = ref.values(*ref.quantise(x)), ref.values(*ref.quantise(np.ascontiguousarray(w.T)))
    _close(rt.download_f32(out).reshape(m, n), va @ vb.T, np.abs(va) @ np.abs(vb).T, k)


@pytest.mark.parametrize("k, n", [(65535 * 32 + 65, 3), (3, 65535 * 32 + 65)])
def test_weights_longer_than_a_launch_has_in_a_direction(rt, k, n):
    x, w = _rows(1, 2, k), seeded.normal(2, k * n, 0.1).reshape(k, n)
    lin = rt.prepare_linear_fp8(k, n, w)
    out = rt.upload_f32(np.full(2 * n, np.nan))
    lin.run(rt.upload_f32(x), 2, out)
    va, vb = ref.values(*ref.quantise(x)), ref.values(*ref.quantise(np.ascontiguousarray(w.T)))
    _close(rt.download_f32(out).reshape(2, n), va @ vb.T, np.abs(va) @ np.abs(vb).T, k)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_nan_stays_in_its_row(rt, m):
    k, n = 300, 50
    a, b = _rows(1, m, k), _rows(2, n, k)
    want = ref.values(*ref.quantise(a)) @ ref.values(*ref.quantise(b)).T
    a[m // 2, 7], b[n // 3, 299] = np.inf, np.nan
    c = rt.alloc_f32(m * n)
    rt.gemm_fp8_into(_uploaded(rt, a), _uploaded(rt, b), c)
    got = rt.download_f32(c).reshape(m, n)
    bad = np.zeros((m, n), bool)
    bad[m // 2], bad[:, n // 3] = True, True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    assert np.allclose(got[~bad], want[~bad], rtol=1e-4, atol=1e-3)


@pytest.mark.parametrize("m, n", [(1, 700), (40, 700), (1000, 700)])
def test_the_same_call_gives_the_same_bits(rt, m, n):
    x, lin = rt.upload_f32(_rows(1, m, 900)), _linear(rt, "rows", 900, n, seeded.normal(5, n), None)[0]
    outs = [rt.alloc_f32(m * n) for _ in range(3)]
    for out in outs:
        lin.run(x, m, out)
    a, b, c = (rt.download_f32(o) for o in outs)
    assert_bits_equal(a, b)
    assert_bits_equal(a, c)


def test_no_rows(rt):
    lin, out = _linear(rt, "rows", 128, 8, None, None)[0], rt.alloc_f32(0)
    lin.run(rt.alloc_f32(0), 0, out)
    t = rt.quantize_fp8(rt.alloc_f32(0), 0, 128)
    assert (t.rows, t.k) == (0, 128)
    lin.run_rows(t, out)
    rt.dequantize_fp8_into(t, out)
    rt.gemm_fp8_into(t, t, out)
    assert rt.fp8_download(t)[0].shape == (0, 128)
    rt.synchronize()


def test_refusals(rt):
    x, out = rt.upload_f32(_rows(1, 4, 128)), rt.alloc_f32(4 * 8)
    t, lin = _uploaded(rt, _rows(1, 4, 128)), _linear(rt, "rows", 128, 8, None, seeded.normal(1, 8))[0]
    other = vh.Runtime(0)
    foreign = other.alloc_f32(4 * 8)
    bad = [
        (vh.KernelError, lambda: rt.alloc_fp8(4, 0)), (vh.KernelError, lambda: rt.alloc_fp8(2 ** 27 + 1, 1)),
        (vh.KernelError, lambda: rt.quantize_fp8(x, 512, 0)),
        (vh.KernelError, lambda: rt.fp8_upload(np.zeros(4, np.uint8), np.full(1, 255, np.uint8), 1, 4)),
        (vh.LengthMismatch, lambda: rt.quantize_fp8(x, 4, 127)),
        (vh.LengthMismatch, lambda: rt.quantize_fp8_into(x, 4, 128, rt.alloc_fp8(4, 129))),
        (vh.LengthMismatch, lambda: rt.dequantize_fp8_into(t, out)),
        (vh.LengthMismatch, lambda: rt.gemm_fp8_into(t, rt.alloc_fp8(8, 256), out)),
        (vh.LengthMismatch, lambda: rt.gemm_fp8_into(t, t, out)),
        (vh.BlasError, lambda: rt.prepare_linear_fp8(0, 8, np.zeros(0))),
        (vh.BlasError, lambda: rt.prepare_linear_fp8_blocks(8, 1, np.zeros(8, np.uint8), [np.inf])),
        (vh.BlasError, lambda: lin.run(x, 5, out)), (vh.BlasError, lambda: lin.run_gelu(x, 4, out)),
        (vh.BlasError, lambda: lin.run_rows(rt.alloc_fp8(4, 129), out)),
        (vh.LengthMismatch, lambda: lin.run(x, 4, rt.alloc_f32(33))),
        (vh.LengthMismatch, lambda: lin.run_rows(t, rt.alloc_f32(31))),
        (vh.InvalidArgument, lambda: lin.run(x, 4, foreign)), (vh.InvalidArgument, lambda: lin.run_rows(t, foreign)),
        (vh.InvalidArgument, lambda: other.quantize_fp8(x, 4, 128)),
        (vh.InvalidArgument, lambda: other.fp8_download(t)),
        (vh.InvalidArgument, lambda: other.dequantize_fp8_into(t, x)),
        (vh.InvalidArgument, lambda: rt.gemm_fp8_into(t, other.alloc_fp8(8, 128), out))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    square = _linear(rt, "rows", 128, 128, None, None)[0]
    with pytest.raises(vh.InvalidArgument, match="also an input"):
        square.run(x, 4, x)
