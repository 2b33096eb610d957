"""gemmF8 on tensor memory when the waits of its copies give up after few polls (and the others with them): the call reports it, what was in flight was waited for (those waits leave
a bit of their own, 0x1000, if they fail), and the next call on the same context is right."""
import re

import numpy as np
import pytest

import p0pc0rn_b200 as p0
from p0pc0rn_b200 import _lib as L

from . import f8_ref as R
from .test_gpu_f8 import Rows, out_mat, rand_mat, run_gemm

pytestmark = pytest.mark.gpu


def gives_up(g, monkeypatch, M, N, K, epi, polls, form):
    """one call whose copies' waits end after `polls` polls; whether one of them did"""
    rng = np.random.default_rng(M + polls)
    x, w = rand_mat(g, rng, M, K)[0], rand_mat(g, rng, N, K, True)[0]
    a = {"x": x.arg(), "w": w.arg(), "M": M, "N": N, "K": K, "epi": epi}
    y = out_mat(g, M, N) if epi == "swiglu" else Rows(g, np.zeros((M, N), np.float16))
    a["y"] = y.arg()
    if epi == "swiglu":
        a["u"] = w.arg()
    g.done()
    monkeypatch.setenv("P0MM_F8_POLLS", str(polls))
    try:
        p0.gemmF8(g, a)
    finally:
        monkeypatch.delenv("P0MM_F8_POLLS")
    try:
        g.done(20000)
    except p0.P0Error as e:
        code = int(re.search(r"code 0x([0-9a-f]+)", str(e)).group(1), 16)
        assert e.status == L.P0_ETIMEOUT and not code & 0x1000 and code & 0xff0 == form, str(e)
        return True
    return False


@pytest.mark.parametrize("M,epi", [(12, "f16"), (30, "f16"), (60, "f16"), (120, "f16"), (12, "swiglu"), (30, "swiglu"), (60, "swiglu")])
def test_few_tokens(g, monkeypatch, M, epi):
    N, K = 600, 4200      # clusters of four (12 tokens of shorter rows would go without tensor memory), eight blocks and more a CTA
    for polls in (0, 1, 4, 0):
        was = gives_up(g, monkeypatch, M, N, K, epi, polls, 0x8a0)
        assert was or polls
        run_gemm(g, M, N, K, epi)
        g.done()
