"""The gate of gemmF8's gated results by itself: products that are exact, so that nothing hides what the gate is off."""
import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import f8_ref as R
from .test_gpu_f8 import Mat, out_mat

pytestmark = pytest.mark.gpu
N, K, U = 200, 256, 2.0 ** 40


def run(g, x, epi):
    """act(x) * U by the operator, [M], from the blocks' scales: every column of a row has the same value, so its code is that of +-448"""
    M = x.size
    # the argument is a block's scale, and u's factor another block's
    q, s = np.zeros((M, K), np.uint8), np.stack([np.abs(x), np.ones(M)]).astype(np.float32)
    q[:, 3], q[:, 130] = np.where(x < 0, 0xb8, 0x38), 0x38
    wq, uq, ws = np.zeros((N, K), np.uint8), np.zeros((N, K), np.uint8), np.ones((2, 2), np.float32)
    wq[:, 3], uq[:, 130] = 0x38, 0x38
    xb, w, u, y = Mat(g, q, s), Mat(g, wq, ws), Mat(g, uq, ws * np.float32([1.0, U])), out_mat(g, M, N)
    p0.gemmF8(g, {"x": xb.arg(), "w": w.arg(), "u": u.arg(), "M": M, "N": N, "K": K, "epi": epi, "y": y.arg()})
    codes, scales = y.read()
    assert (scales[0] == scales[1]).all() and (codes == codes[:, :1]).all()
    return R.VALUE[codes[:, 0]] * scales[0].astype(np.float64), codes[:, 0]


def arguments(M, epi, seed):
    """f32 arguments, of either sign and of all sizes, down to an exponent of -87"""
    rng = np.random.default_rng(seed)
    least = -87.0 if epi == "swiglu" else -9.9
    x = np.concatenate([rng.uniform(least, 0, M), rng.uniform(0, 40, M), -np.exp(rng.uniform(-20, np.log(-least), M)), np.exp(rng.uniform(-20, 6, M))])
    return rng.permutation(x)[:M].astype(np.float32)


@pytest.mark.parametrize("epi", ["swiglu", "geglu"])
@pytest.mark.parametrize("M", [7, 30, 60, 700])       # each form
def test_gate(g, M, epi):
    for seed in range(4 if M < 100 else 2):
        x = arguments(M, epi, seed)
        got, codes = run(g, x, epi)
        v = x.astype(np.float64)
        z = v if epi == "swiglu" else 2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)
        e = np.exp(-z)
        want = v / (1 + e) * U
        # e^-z: ex2.approx 2^-22 and the product behind it 2^-24; 1 + e 2^-24; the quotient 2 units: 2^-22. The product with u, the scale and the
        # code's value 448 times it: 2^-24 each. z of geglu: five roundings of 2^-24, each of which moves e^-z by z
        tol = 2.0 ** -22 * (1.25 * e / (1 + e) + 0.25 + 1) + 3 * 2.0 ** -24 + (5 * 2.0 ** -24 * np.abs(z) * e / (1 + e) if epi == "geglu" else 0)
        assert ((codes & 127) == 0x7e).all() and (np.abs(got - want) <= tol * np.abs(want)).all(), float((np.abs(got / want - 1) / tol).max())


@pytest.mark.parametrize("epi", ["swiglu", "geglu"])
@pytest.mark.parametrize("M", [7, 60, 700])
def test_gate_far_out(g, M, epi):
    # below an exponent of -87.3 the act is less than 2^-119, and may be 0; far above it is x
    far = np.array([-87.4, -88.0, -88.1, -88.8, -100.0, -1e4, -1e30, 89.0, 1e4, 1e20] if epi == "swiglu" else [-10.01, -10.1, -12.0, -100.0, -1e15, -1e30, 11.0, 100.0, 1e15, 1e20])
    x = np.resize(far, M).astype(np.float32)
    got, codes = run(g, x, epi)
    want = np.where(x < 0, 0.0, x.astype(np.float64) * U)
    assert not ((codes & 127) == 0x7f).any() and (np.abs(got - want) <= np.where(x < 0, U * 2.0 ** -119, want * 2.0 ** -22)).all()
