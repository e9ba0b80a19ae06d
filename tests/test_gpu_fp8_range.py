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
