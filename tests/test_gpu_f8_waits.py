"""gemmF8 on tensor memory when the waits of its copies give up after few polls (and the others with them): the call reports it, what was in flight was waited for (those waits leave
a bit of their own, 0x1000, if they fail), and the next call on the same context is right."""
import re

import numpy as np
import pytest

import p0pc0rn_b200 as p0
from p0pc0rn_b200 import _lib as L

from .test_gpu_f8 import Rows, out_mat, rand_mat, run_gemm

pytestmark = pytest.mark.gpu


def gives_up(g, monkeypatch, M, N, K, epi, polls, form, mats):
    """one call whose copies' waits end after `polls` polls; whether one of them did"""
    a = {"x": mats[0][0].arg(), "w": mats[1][0].arg(), "M": M, "N": N, "K": K, "epi": epi}
    y = out_mat(g, M, N) if epi == "swiglu" else Rows(g, np.zeros((M, N), np.float16))
    a["y"] = y.arg()
    if epi == "swiglu":
        a["u"] = mats[2][0].arg()
    g.done()
    monkeypatch.setenv("P0MM_F8_POLLS", polls)
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


def check(g, monkeypatch, M, N, K, epi, form, limits):
    rng = np.random.default_rng(M)
    mats = [rand_mat(g, rng, M, K), rand_mat(g, rng, N, K, True), rand_mat(g, rng, N, K, True)]
    for polls, always in limits:
        was = gives_up(g, monkeypatch, M, N, K, epi, polls, form, mats)
        assert was or not always
        run_gemm(g, M, N, K, epi, mats=mats)
        g.done()


@pytest.mark.parametrize("M,epi", [(12, "f16"), (30, "f16"), (60, "f16"), (120, "f16"), (12, "swiglu"), (30, "swiglu"), (60, "swiglu")])
def test_few_tokens(g, monkeypatch, M, epi):
    # clusters of four (12 tokens of shorter rows would go without tensor memory), eight blocks and more a CTA
    check(g, monkeypatch, M, 600, 4200, epi, 0x8a0, [("0", True), ("1", False), ("4", False), ("0", True)])


# more blocks than twice a pair's stages, so that a CTA which goes on fills each stage once more; one tile a pair, and two
@pytest.mark.parametrize("M,N,K,epi", [(1100, 1300, 1700, "f16"), (1100, 1300, 1700, "swiglu"), (2100, 2300, 1700, "f16")])
def test_many_tokens(g, monkeypatch, M, N, K, epi):
    # both CTAs of a pair stop at once; the even one stops while the odd one goes on; the other way round
    check(g, monkeypatch, M, N, K, epi, 0x8f0, [("0", True), ("0,300", True), ("300,0", True), ("1", False), ("3,1", False), ("0", True)])
