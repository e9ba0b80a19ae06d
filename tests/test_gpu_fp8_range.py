"""Products of rows in 8-bit floating point whose blocks differ in size by tens of powers of two, against float64
numpy (tests/fp8_64.py), in every form of the kernels.

The tolerance is that of test_gpu_fp8: (K / 32 + 8) 2^-23 of the sum of the magnitudes of an output's terms.  A block's
sum is exact to within its own roundings and joins the others at its own size, so nothing is allowed on top for
blocks that are far below the largest of their row."""
import numpy as np
import pytest

import fp8_64 as ref
from test_gpu_fp8 import _close
from vestra_hip import seeded

pytestmark = pytest.mark.gpu


def _sized(seed, rows, powers, k):
    """Rows of k values, those of block b of the size 2^powers[b]."""
    x = seeded.normal(seed, rows * k).reshape(rows, k).astype(np.float64)
    return (x * np.exp2(np.asarray(powers, float)).repeat(128)[:k]).astype(np.float32)


def _checkpoint(rt, seed, k, n, scales, bias=None):
    codes = ref.e4m3((seeded.normal(seed, n * k, 40.0).reshape(n, k)).clip(-448, 448))
    return rt.prepare_linear_fp8_blocks(k, n, codes, scales, bias), ref.block_values(codes, scales)


@pytest.mark.parametrize("m", [1, 16, 40, 200])
@pytest.mark.parametrize("powers, scales", [
    # Of the rows' blocks and of their scales.  The sums of the second and later ones pass the floats until their
    # scales meet them; one is zero.
    ([0, 110, 0, 0], [1.0, 2.0 ** -30, 1.0, 0.5]),
    ([0, 114, 118, 118], [1.0, 2.0 ** -60, -0.7 * 2.0 ** -60, 0.0]),
    ([-100, 20, 118, 0], [2.0 ** 100, 2.0 ** -3, -2.0 ** -40, 2.0 ** 50]),
    ([-100, 118, 118, 118], [2.0 ** -20, 2.0 ** -140, 0.0, -2.0 ** -130])])  # no normal floats
def test_scales_far_below_the_largest_of_their_rows(rt, m, powers, scales):
    k, n = 500, 200
    x = _sized(m, m, powers, k)
    s = np.tile(np.array(scales, np.float32), (2, 1))
    s[1, 0] = 0.0  # the second 128 rows, without the largest
    lin, vw = _checkpoint(rt, 6, k, n, s.reshape(-1))
    out = rt.upload_f32(np.full(m * n, np.nan))
    lin.run(rt.upload_f32(x), m, out)
    vx = ref.values(*ref.quantise(x))
    _close(rt.download_f32(out).reshape(m, n), vx @ vw.T, np.abs(vx) @ np.abs(vw).T, k)


@pytest.mark.parametrize("extra", [1, 12])
@pytest.mark.parametrize("m, k, n", [(2000, 520, 1088), (3000, 520, 2080), (3500, 384, 4288), (1999, 130, 1280)])
def test_columns_past_the_end_leave_the_others_rows_alone(rt, m, k, n, extra):
    """The last columns' tiles, in tiles of 64, 128 and 256: most lanes of a wave have nothing to write, and
    its strips of 16 rows go through the same LDS."""
    a, b = _sized(3, m, [0] * ref.blocks(k), k), _sized(4, n + extra, [0] * ref.blocks(k), k)
    va, vb = (ref.values(*ref.quantise(x)) for x in (a, b))
    c = rt.upload_f32(np.full(m * (n + extra), np.nan))
    rt.gemm_fp8_into(*(rt.quantize_fp8(rt.upload_f32(x), *x.shape) for x in (a, b)), c)
    _close(rt.download_f32(c).reshape(m, n + extra), va @ vb.T, np.abs(va) @ np.abs(vb).T, k)


# Rows of few, of tiles of 64, of 128 and of 256, as the model of a launch has them.
FORMS = [(1, 512, 700), (12, 1100, 70), (40, 512, 300), (2000, 520, 1100), (700, 2300, 2000), (3000, 520, 2100),
         (3500, 384, 4300)]


def _powers(blocks, low, high):
    """Sizes of a row's blocks, the largest first, the others far below: what the other side has there is far above."""
    p = np.full(blocks, low)
    p[0] = high
    return p


@pytest.mark.parametrize("m, k, n", FORMS)
@pytest.mark.parametrize("gap", [16, 24, 70])
def test_a_small_block_against_a_large_one(rt, m, k, n, gap):
    """The outputs come from the blocks that are small in one side's rows and large in the other's."""
    nb = ref.blocks(k)
    a, b = _sized(1, m, _powers(nb, -gap, 0), k), _sized(2, n, -_powers(nb, -gap, 0), k)
    a[:, :128] *= (np.arange(m) % 3 == 0)[:, None]  # zeros: rows whose exponents are alike
    va, vb = (ref.values(*ref.quantise(x)) for x in (a, b))
    c = rt.upload_f32(np.full(m * n, np.nan))
    qa, qb = (rt.quantize_fp8(rt.upload_f32(x), *x.shape) for x in (a, b))
    rt.gemm_fp8_into(qa, qb, c)
    want, size = va @ vb.T, np.abs(va) @ np.abs(vb).T
    got = rt.download_f32(c).reshape(m, n)
    _close(got, want, size, k)
    # Rows that came as codes.
    up = [rt.fp8_upload(*rt.fp8_download(q), *x.shape) for q, x in ((qa, a), (qb, b))]
    again = rt.upload_f32(np.full(m * n, np.nan))
    rt.gemm_fp8_into(*up, again)
    assert np.array_equal(rt.download_f32(again).reshape(m, n), got)


@pytest.mark.parametrize("m, k, n", FORMS)
def test_projections_of_rows_of_wide_range(rt, m, k, n):
    """From floats and from rows, with every epilogue: one row in seven has a block 2^40 above the others, where the
    weights are 2^40 below theirs."""
    nb = ref.blocks(k)
    x = _sized(1, m, np.zeros(nb), k)
    wide = np.arange(m) % 7 == 0
    x[wide, :128] *= np.float32(2.0 ** 40)
    w = np.ascontiguousarray(_sized(2, n, _powers(nb, -4, -44), k).T)
    bias, gamma, res = seeded.normal(5, n), seeded.normal(6, n), seeded.normal(7, m * n)
    vx, vw = ref.values(*ref.quantise(x)), ref.values(*ref.quantise(np.ascontiguousarray(w.T)))
    xt, rows = rt.upload_f32(x), rt.quantize_fp8(rt.upload_f32(x), m, k)
    y, size = vx @ vw.T + bias, np.abs(vx) @ np.abs(vw).T + np.abs(bias)
    lin, r = rt.prepare_linear_fp8(k, n, w, bias, gamma), res.reshape(m, n)
    for run, arg in ((lin.run_residual, (xt, m)), (lin.run_rows_residual, (rows,))):
        out = rt.upload_f32(res)
        run(*arg, out)
        _close(rt.download_f32(out).reshape(m, n), y * gamma + r, size * np.abs(gamma) + np.abs(r), k)
    lin, out = rt.prepare_linear_fp8(k, n, w, bias), rt.upload_f32(res)
    lin.run_gelu(xt, m, out)
    _close(rt.download_f32(out).reshape(m, n), ref.gelu(y), 1.13 * size, k, 1e-6 * np.maximum(1, np.abs(y)))


@pytest.mark.parametrize("m, k, n", FORMS)
@pytest.mark.parametrize("gap", [24, 100])
def test_block_scales_of_wide_range(rt, m, k, n, gap):
    """A checkpoint's scales that run the other way than the rows' blocks, and are zero for the largest of them."""
    nb = ref.blocks(k)
    x = _sized(1, m, _powers(nb, 10 - gap, 10), k)
    scales = np.exp2(-_powers(nb, 10 - gap, 10)) * np.exp(seeded.normal(3, ref.blocks(n) * nb, 0.3).reshape(-1, nb))
    scales[::2, 0] = 0.0
    lin, vw = _checkpoint(rt, 6, k, n, scales.astype(np.float32).reshape(-1))
    out = rt.upload_f32(np.full(m * n, np.nan))
    lin.run(rt.upload_f32(x), m, out)
    vx = ref.values(*ref.quantise(x))
    _close(rt.download_f32(out).reshape(m, n), vx @ vw.T, np.abs(vx) @ np.abs(vw).T, k)


@pytest.mark.parametrize("m, k, n", FORMS[3:])
def test_nan_stays_in_its_row_of_wide_range(rt, m, k, n):
    nb = ref.blocks(k)
    a, b = _sized(1, m, _powers(nb, -30, 0), k), _sized(2, n, np.zeros(nb), k)
    want = ref.values(*ref.quantise(a)) @ ref.values(*ref.quantise(b)).T
    size = np.abs(a).astype(np.float64) @ np.abs(b).T.astype(np.float64)
    a[m // 2, k - 1], b[n // 3, 7] = np.inf, np.nan
    c = rt.upload_f32(np.zeros(m * n))
    rt.gemm_fp8_into(*(rt.quantize_fp8(rt.upload_f32(x), *x.shape) for x in (a, b)), c)
    got = rt.download_f32(c).reshape(m, n)
    bad = np.zeros((m, n), bool)
    bad[m // 2], bad[:, n // 3] = True, True
    assert np.isnan(got[bad]).all()
    _close(got[~bad], want[~bad], 1.13 * size[~bad], k)  # the codes' values: each within 2^-4 of its own


@pytest.mark.parametrize("m, k, n", [(40, 512, 300), (2000, 520, 1100), (3000, 520, 2100), (3500, 384, 4300)])
@pytest.mark.parametrize("gap", [14, 15, 16, 17])
def test_the_least_codes_at_the_border_of_wide_rows(rt, m, k, n, gap):
    """Blocks `gap` powers of two below the first one of their row, of the least codes there are, whose sums are
    what comes out, to the bit: every product is a multiple of 2^-9 by one of 1, 2 or 4, below 2^24 of them in all."""
    a = np.zeros((m, k), np.float32)
    a[:, 0], a[:, 128::128] = 448.0 * 2.0 ** gap, 448.0  # the exponents gap and 0
    a[:, 129:160] = (1 + (np.arange(m)[:, None] + np.arange(31)) % 7) * 2.0 ** -9
    b = np.zeros((n, k), np.float32)
    b[:, 129:160] = 2.0 ** ((np.arange(n)[:, None] + np.arange(31)) % 3)
    want = a[:, 129:160].astype(np.float64) @ b[:, 129:160].T.astype(np.float64)
    c = rt.upload_f32(np.full(m * n, np.nan))
    rt.gemm_fp8_into(*(rt.quantize_fp8(rt.upload_f32(x), *x.shape) for x in (a, b)), c)
    assert np.array_equal(rt.download_f32(c).reshape(m, n), want)
