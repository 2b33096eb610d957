"""beamSelect on the GPU against the plain statement in tests/kv_ref.py (lse from 64 bits). Inputs are such that no two
candidates are nearer than a last bit of lse could move them (or are equal on purpose, where the index decides)."""
import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import kv_ref as R

pytestmark = pytest.mark.gpu


def run(g, logits, score, groups, k, eos=None, fin=None, ld=0, off=0, V=None):
    n = groups * k
    b = {x: g.upload(np.full(n, 0x5a5a5a5a, np.uint32)) for x in ("parent", "token", "score", "fin")}
    a = {"logits": {"buf": g.upload(logits), "off": off, "ld": ld}, "score": {"buf": g.upload(score.astype(np.float32))}, "groups": groups, "beams": k,
         "V": V or logits.shape[1], "eos": eos, "parent": {"buf": b["parent"]}, "token": {"buf": b["token"]}, "scoreOut": {"buf": b["score"]},
         "finOut": {"buf": b["fin"]}}
    if fin is not None:
        a["fin"] = {"buf": g.upload(fin.astype(np.uint32))}
    p0.beamSelect(g, a)
    rd = lambda x, t: g.read(b[x], 0, n * 4, t)
    return rd("parent", np.uint32), rd("token", np.uint32), rd("score", np.float32), rd("fin", np.uint32)


def check(got, want, rel=2.0 ** -21):
    for i in (0, 1, 3):
        assert np.array_equal(got[i], want[i]), i
    live = want[2] > -np.inf
    assert np.array_equal(live, got[2] > -np.inf)
    # lse: a sum of V positive terms in f32 (pairwise by chunk), exp and log within 2^-22; then two f32 sums
    assert np.all(np.abs(got[2][live] - want[2][live]) <= rel * (np.abs(want[2][live]) + 30.0))


def spaced(rng, n, V):
    """distinct logits: multiples of 1/64 plus a 1/2048 per row class, largest ones thinned out"""
    x = np.round(rng.standard_normal((n, V)) * 4 * 64) / 64
    for r in range(n):
        top = np.argsort(-x[r], kind="stable")[:40]
        x[r, top] = x[r].max() + 0.25 * np.arange(40, 0, -1) * (1 + 0.01 * r)
    return x.astype(np.float32)


@pytest.mark.parametrize("groups,k,V", [(1, 1, 1), (1, 4, 7), (2, 3, 100), (1, 8, 4096), (3, 5, 4097), (2, 16, 12289), (1, 2, 262144), (40, 2, 999)])
def test_select(g, groups, k, V):
    rng = np.random.default_rng(V + k)
    n = groups * k
    x = rng.standard_normal((n, V)).astype(np.float32) * 4 if V < 64 else spaced(rng, n, V)
    score = -(rng.random(n) * 9 + 0.013 * np.arange(n)).astype(np.float32)
    fin = (rng.random(n) < 0.2).astype(np.uint32) if V > 3 else None
    eos = 2 if V > 3 else None
    check(run(g, x, score, groups, k, eos, fin), R.beam(x, score, groups, k, eos, fin))


def test_first_step_one_live_beam(g):
    rng = np.random.default_rng(1)
    x = spaced(rng, 16, 5000)
    score = np.full(16, -np.inf, np.float32)
    score[[0, 8]] = 0.0
    got = run(g, x, score, 2, 8)
    check(got, R.beam(x, score, 2, 8, None))
    assert np.all(got[0] == np.repeat([0, 8], 8))


def test_ties_go_to_the_lowest_index(g):
    # equal logits, equal beams: whole tokens of one value, repeated maxima across chunk borders, -0 against +0
    V = 20000
    same = np.zeros((6, V), np.float32)
    same[1::2] = -0.0
    got = run(g, same, np.zeros(6, np.float32), 1, 6)
    assert np.all(got[0] == 0) and np.array_equal(got[1], np.arange(6))
    x = np.full((4, V), -3.0, np.float32)
    x[:, [4095, 4096, 12000, 19999]] = 5.0
    got = run(g, x, np.zeros(4, np.float32), 1, 4)
    assert np.all(got[0] == 0) and np.array_equal(got[1], [4095, 4096, 12000, 19999])
    x[2, 3] = 6.0                                                    # one row ahead, its others behind the equal rows by its lse
    got = run(g, x, np.zeros(4, np.float32), 1, 4)
    check(got, R.beam(x, np.zeros(4, np.float32), 1, 4, None))


def test_ties_that_rounding_makes(g):
    # scores so large that many distinct logits round to one c: the lowest index wins, not the largest logit
    rng = np.random.default_rng(2)
    for V in (300, 9000):
        x = (rng.permutation(V)[None] * 1e-4 + np.zeros((3, 1))).astype(np.float32)
        score = np.full(3, -1e5, np.float32)
        got = run(g, x, score, 1, 3)
        want = R.beam(x, score, 1, 3, None)
        check(got, want)
    fin = np.array([0, 1, 0], np.uint32)                             # a finished beam among the equal ones
    x[:] = 0.0
    score = np.array([-1e6, -1e6, -1e6], np.float32)
    score[1] = np.float32(-1e6) - np.float32(np.log(9000.0))
    check(run(g, x, score, 1, 3, 5, fin), R.beam(x, score, 1, 3, 5, fin))


def test_never_chosen(g):
    # -inf masks, rows of nothing, NaN and +inf rows, fewer candidates than slots
    rng = np.random.default_rng(3)
    V = 5000
    x = spaced(rng, 8, V)
    x[0, :] = -np.inf
    x[1, 77] = np.nan
    x[2, 78] = np.inf
    x[3, :] = -np.inf
    x[3, [4500, 9]] = [1.0, 2.0]
    x[4:, :] = -np.inf
    x[5, 10] = 3.4e38
    x[6, 3] = -3.4e38
    score = np.zeros(8, np.float32)
    score[3] = 0.5
    got = run(g, x, score, 1, 8)
    check(got, R.beam(x, score, 1, 8, None))
    assert (got[0] == R.NONE).sum() == 4 and (got[1] == R.NONE).sum() == 4
    nothing = run(g, np.full((4, 10), -np.inf, np.float32), np.zeros(4, np.float32), 2, 2)
    assert np.all(nothing[0] == R.NONE) and np.all(nothing[2] == -np.inf) and not nothing[3].any()


def test_finished_beams(g):
    rng = np.random.default_rng(4)
    x = spaced(rng, 4, 600)
    score = np.array([-1.0, -2.0, -1.5, -30.0], np.float32)
    fin = np.array([1, 0, 1, 1], np.uint32)
    x[0] = np.nan                                                    # a finished beam's logits do not matter
    got = run(g, x, score, 1, 4, 599, fin)
    check(got, R.beam(x, score, 1, 4, 599, fin))
    assert got[3][list(got[0]).index(0)] == 1
    x[1, 599] = 100.0                                                # the unfinished beam ends now
    got = run(g, x, score, 1, 4, 599, fin)
    check(got, R.beam(x, score, 1, 4, 599, fin))


def test_strides_in_place(g):
    rng = np.random.default_rng(5)
    x = spaced(rng, 6, 1001)
    score = -np.arange(6, dtype=np.float32) * 0.37
    for ld, off in ((1001, 0), (1001, 3), (1024, 4), (1500, 1)):
        buf = np.full(off + 6 * ld, np.nan, np.float32)
        for r in range(6):
            buf[off + r * ld:off + r * ld + 1001] = x[r]
        check(run(g, buf, score, 2, 3, ld=ld, off=off, V=1001), R.beam(x, score, 2, 3, None))
    s, f, pt = g.upload(score), g.upload(np.array([0, 1, 0, 0, 0, 1], np.uint32)), [g.buffer(24) for _ in range(2)]
    p0.beamSelect(g, {"logits": {"buf": g.upload(x)}, "score": {"buf": s}, "fin": {"buf": f}, "groups": 2, "beams": 3, "V": 1001, "eos": 7,
                      "parent": {"buf": pt[0]}, "token": {"buf": pt[1]}, "scoreOut": {"buf": s}, "finOut": {"buf": f}})
    want = R.beam(x, score, 2, 3, 7, np.array([0, 1, 0, 0, 0, 1], np.uint32))
    check((g.read(pt[0], 0, 24, np.uint32), g.read(pt[1], 0, 24, np.uint32), g.read(s, 0, 24, np.float32), g.read(f, 0, 24, np.uint32)), want)


@pytest.mark.parametrize("order", ["rising", "falling", "steps"])
def test_ordered_rows(g, order):
    # rows in rising order: everything reaches the bound that the first logits gave
    V = 70001
    x = np.arange(V, dtype=np.float32)[None] * np.float32(1e-3) + np.zeros((4, 1), np.float32)
    if order == "falling":
        x = x[:, ::-1].copy()
    if order == "steps":
        x = np.floor(x * 10) / 10
    x = x.astype(np.float32)
    score = np.array([0.0, -0.25, -0.5, -7.0], np.float32)
    for groups, k in ((1, 4), (2, 2), (4, 1)):
        check(run(g, x, score, groups, k), R.beam(x, score, groups, k, None))


def test_refusals(g):
    b = g.buffer(4000)
    a = {"logits": {"buf": b}, "score": {"buf": b}, "groups": 1, "beams": 4, "V": 100, "eos": 1, "parent": {"buf": b}, "token": {"buf": b},
         "scoreOut": {"buf": b}}
    for msg, change in (("17 beams", {"beams": 17}), ("0 beams", {"beams": 0}), ("pass 32 bits", {"V": 0xffffffff // 4 + 1}), ("row stride 99", {"logits": {"buf": b, "ld": 99}}),
                        ("logits range", {"V": 251}), ("eos 100 outside", {"eos": 100, "fin": {"buf": b}}), ("missing binding score", {"score": {"buf": None}}),
                        ("65536 rows", {"groups": 16384}), ("a vocabulary of 16777217", {"V": 16777217})):
        with pytest.raises(p0.P0Error, match=msg):
            p0.beamSelect(g, {**a, **change})
    g.done()
