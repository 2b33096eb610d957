"""normF8 with h given as x's own rows."""
import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import f8_ref as R
from .test_gpu_f8 import SLACK, Rows, out_mat

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,ld,h_ld", [(1, 0, 320), (1, 304, 0), (1, 301, 302), (3, 304, 304), (3, 0, 300), (200, 301, 301)])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_h_is_x(g, M, ld, h_ld, scale):
    # a row alone has no stride to speak of: whatever two are given, the rows are the same
    D = 300
    x = np.random.default_rng(M + h_ld).standard_normal((M, D)).astype(np.float32)
    xs, w, y = Rows(g, x, ld), Rows(g, np.ones((1, D), np.float32)), out_mat(g, M, D)
    p0.normF8(g, {"x": {**xs.arg(), "ld": ld}, "h": {**xs.arg(), "ld": h_ld}, "w": w.arg(), "y": y.arg(), "M": M, "D": D, "scale": scale})
    h = xs.read()
    assert (h == x * np.float32(scale)).all()      # by a power of two: exact
    R.check_codes(*y.read(), R.norm(h, None, None, np.ones(D), 1e-6, 1.0)[2], SLACK)
