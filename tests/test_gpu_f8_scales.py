"""gemmF8 with scales of any size: a block's factor, x's scale times w's, is rounded to f32. Held here: what that costs where the product leaves
f32's normal range below, and that nothing is lost just inside of the range, at either end."""
import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import f8_ref as R
from .test_gpu_f8 import Mat, Rows, out_mat

pytestmark = pytest.mark.gpu
N, K = 200, 400
# the forms: without tensor memory, few tokens (each width), many tokens (partly in a second row of tiles)
TOKENS = [1, 3, 20, 50, 130, 700]


def codes(rng, rows, lo=0x30, hi=0x7f):
    """codes of normal values and of either sign"""
    return (rng.integers(lo, hi, (rows, K)) | (rng.integers(0, 2, (rows, K)) << 7)).astype(np.uint8)


def operands(g, M, x_scales, w_scales, seed, spread=2.0, **kw):
    rng = np.random.default_rng(seed)
    mats = []
    for rows, sizes, tile in ((M, x_scales, False), (N, w_scales, True)):
        q = codes(rng, rows, **kw)
        shape = (R.blocks(rows), R.blocks(K)) if tile else (R.blocks(K), rows)
        s = (np.asarray(sizes, np.float64).reshape((1, -1) if tile else (-1, 1)) * rng.uniform(1, spread, shape)).astype(np.float32)
        mats.append((Mat(g, q, s), R.values(q, s, tile)))
    return mats


def run(g, M, mats, off):
    """f32 results; off: what a result may be off besides the sums' bound"""
    (x, xv), (w, wv) = mats
    y = Rows(g, np.zeros((M, N), np.float32))
    p0.gemmF8(g, {"x": x.arg(), "w": w.arg(), "M": M, "N": N, "K": K, "epi": "f32", "y": y.arg()})
    want, size = R.product(xv, wv)
    got = y.read().astype(np.float64)
    tol = size * R.sum_bound(K) + off
    assert np.isfinite(want).all() and (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())
    return want


# of a product below 2^-126: rounded to a multiple of 2^-149, 2^-150 off, times a block's sum, 128 * 448 * 448 at most: 2^-125.3 a block
OFF = 4 * 128 * 448.0 * 448.0 * 2.0 ** -150


@pytest.mark.parametrize("M", TOKENS)
def test_two_small_scales(g, M):
    # products of scales near 2^-135 and 2^-146, of which f32 holds 15 bits and four
    mats = operands(g, M, [2.0 ** -70, 2.0 ** -60, 2.0 ** -78, 2.0 ** -65], [2.0 ** -65, 2.0 ** -86, 2.0 ** -68, 2.0 ** -70], M, lo=0x70)
    want = run(g, M, mats, OFF)
    assert np.abs(want).max() > 2.0 ** -117     # far more than what may be lost


@pytest.mark.parametrize("M", TOKENS)
def test_products_of_scales_within_the_range(g, M):
    # 2^-126 and just above: nothing is lost (sums of codes up to 2^25, so no result is a subnormal that matters: 2^-150 for each of its additions)
    mats = operands(g, M, [2.0 ** -70, 2.0 ** -106, 2.0 ** -20, 2.0 ** -63], [2.0 ** -56, 2.0 ** -20, 2.0 ** -106, 2.0 ** -63], M, lo=0x70)
    run(g, M, mats, 8 * 2.0 ** -150)
    # up to 2^127.9, the smallest codes: results near 2^113
    mats = operands(g, M, [2.0 ** 107, 2.0 ** 20, 1.0, 2.0 ** 60], [2.0 ** 20, 2.0 ** 107, 2.0 ** 127, 2.0 ** 67], M, spread=1.3, lo=0x01, hi=0x02)
    assert np.abs(run(g, M, mats, 0.0)).max() > 2.0 ** 109


@pytest.mark.parametrize("M", TOKENS)
def test_a_block_with_an_infinity(g, M):
    # as packF8 writes it: the largest scale, 448 for the infinity, zeros for the others; with weights up to 2^8 and sums that are 0 or within f32
    q, s = np.zeros((M, K), np.uint8), np.ones((R.blocks(K), M), np.float32)
    q[0, 5], s[0, 0] = 0x7e, R.MOST / np.float32(448)
    q[:, 200] = 0x38
    wq, ws = np.full((N, K), 0x38, np.uint8), np.full((R.blocks(N), R.blocks(K)), 2.0 ** 8 / 448, np.float32)
    wq[:, 5] = np.where(np.arange(N) % 3 == 0, 0x01, 0)
    want = run(g, M, [(Mat(g, q, s), R.values(q, s)), (Mat(g, wq, ws), R.values(wq, ws, True))], 0.0)
    assert np.abs(want[0]).max() > 2.0 ** 117


@pytest.mark.parametrize("M", TOKENS)
def test_scales_of_zero(g, M):
    # a scale of zero is a value: its block adds nothing, whatever it meets
    mats = operands(g, M, [0.0, 1.0, 2.0 ** -100, 0.0], [2.0 ** 120, 2.0 ** -120, 0.0, 0.0], M)
    run(g, M, mats, 8 * 2.0 ** -150)


@pytest.mark.parametrize("M", [3, 50, 700])
@pytest.mark.parametrize("epi", ["swiglu", "geglu"])
def test_gated_with_scales_far_apart(g, M, epi):
    # x's scales are tiny and w's and u's large: z = 3000 exactly, gate(3000) = 3000 (the rest of it is beyond f32's least), times 1500
    q, s = np.zeros((M, K), np.uint8), np.full((R.blocks(K), M), 2.0 ** -108, np.float32)
    q[:, 200] = 0x38
    wq, ws = np.full((N, K), 0x38, np.uint8), np.full((R.blocks(N), R.blocks(K)), 3000 * 2.0 ** 108, np.float32)
    x, w, u, y = Mat(g, q, s), Mat(g, wq, ws), Mat(g, wq, np.float32(0.5) * ws), out_mat(g, M, N)
    p0.gemmF8(g, {"x": x.arg(), "w": w.arg(), "u": u.arg(), "M": M, "N": N, "K": K, "epi": epi, "y": y.arg()})
    got, scales = y.read()
    assert (got == 0x7e).all() and (np.abs(scales * 448 - 3000.0 * 1500.0) <= 4.5e6 * 2.0 ** -20).all()
