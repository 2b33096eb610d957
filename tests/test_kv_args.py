"""The cache and beam operators' arguments on CPU (no kernel runs): the argument objects as C structs, the structs'
layout against include/p0mm.h, bound calls, and the host statements of the tests against hand-made vectors."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import p0pc0rn_b200 as p0
from p0pc0rn_b200 import _lib as L

from . import kv_ref as R
from .test_ops_args import FakeBuf, FakeGpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = ["p0_kv", "p0_rows", "p0_kv4_rows_args", "p0_kv4_attn_args", "p0_kv_step_args", "p0_kv_compact_args", "p0_beam_args"]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layout_matches_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "p0mm.h"', "int main(void) {",
             '  printf("%u %u %d %d\\n", P0_KV_PAGE, P0_KV_NONE, P0_F32, P0_F16);']
    for s in STRUCTS:
        lines.append('  printf("%s %%zu\\n", sizeof(%s));' % (s, s))
        for f, _ in getattr(L, s)._fields_:
            lines.append('  printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (s, f, s, f))
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert out[0] == "%d %d %d %d" % (L.P0_KV_PAGE, L.P0_KV_NONE, L.TYPE["f32"], L.TYPE["f16"])
    got = dict(x.rsplit(" ", 1) for x in out[1:])
    for s in STRUCTS:
        cls = getattr(L, s)
        assert int(got[s]) == ctypes.sizeof(cls), s
        for f, _ in cls._fields_:
            assert int(got["%s.%s" % (s, f)]) == getattr(cls, f).offset, (s, f)


def kv():
    return {"pool": {"buf": FakeBuf(1), "off": 32, "stride": 4096}, "pages": 9, "table": {"buf": FakeBuf(2), "off": 3, "ld": 7}, "len": {"buf": FakeBuf(4)},
            "rows": 2, "D": 128, "nkv": 1}


def sent(op, a):
    g = FakeGpu()
    op(g, a)
    (name, rec), = g._lib.calls
    return name, rec[0]


def test_attention_arguments():
    a = {"kv": kv(), "q": {"buf": FakeBuf(5), "off": 6, "ld": 300, "ldh": 130}, "out": {"buf": FakeBuf(7)}, "type": "f16", "nh": 8, "n": 10,
         "cu": {"buf": FakeBuf(8), "off": 2}, "window": 512, "sinks": 4, "scale": 0.5}
    name, s = sent(p0.kv4Attn, a)
    assert name == "p0_kv4_attn"
    assert (s.kv.pool.id, s.kv.pool_off, s.kv.page_stride, s.kv.table.id, s.kv.table_off, s.kv.table_ld, s.kv.len.id, s.kv.len_off, s.kv.pages,
            s.kv.rows, s.kv.D, s.kv.nkv) == (1, 32, 4096, 2, 3, 7, 4, 0, 9, 2, 128, 1)
    assert (s.q.buf.id, s.q.off, s.q.ld, s.q.ldh, s.out.buf.id, s.out.ld) == (5, 6, 300, 130, 7, 0)
    assert (s.type, s.nh, s.n, s.T, s.cu.id, s.cu_off, s.window, s.sinks, s.scale) == (1, 8, 10, 0, 8, 2, 512, 4, 0.5)
    _, s = sent(p0.kv4Attn, {"kv": kv(), "q": {"buf": FakeBuf(5)}, "out": {"buf": FakeBuf(7)}, "nh": 8, "n": 2, "T": 1})
    assert (s.type, s.T, s.cu.id, s.window, s.sinks, s.scale) == (0, 1, 0, 0, 0, 0.0)
    with pytest.raises(p0.P0Error, match="kv4Attn: type f8"):
        sent(p0.kv4Attn, {**a, "type": "f8"})


def test_rows_step_compact_beam_arguments():
    for op, name in ((p0.kv4Put, "p0_kv4_put"), (p0.kv4Get, "p0_kv4_get")):
        got, s = sent(op, {"kv": kv(), "k": {"buf": FakeBuf(5)}, "v": {"buf": FakeBuf(6), "off": 9}, "n": 4, "T": 2})
        assert got == name and (s.k.buf.id, s.v.buf.id, s.v.off, s.type, s.n, s.T) == (5, 6, 9, 0, 4, 2)
    to = {"table": {"buf": FakeBuf(10)}, "len": {"buf": FakeBuf(11)}, "ref": {"buf": FakeBuf(12)}}
    a = {"kv": kv(), "ref": {"buf": FakeBuf(9)}, "to": to, "stat": {"buf": FakeBuf(13)}}
    _, s = sent(p0.kvStep, {**a, "add": 3})
    assert (s.ref.id, s.to_table.id, s.to_len.id, s.to_ref.id, s.parent.id, s.add.id, s.addn, s.stat.id) == (9, 10, 11, 12, 0, 0, 3, 13)
    _, s = sent(p0.kvStep, {**a, "add": {"buf": FakeBuf(14)}, "parent": {"buf": FakeBuf(15)}, "window": 8, "sinks": 2})
    assert (s.parent.id, s.add.id, s.addn, s.window, s.sinks) == (15, 14, 0, 8, 2)
    _, s = sent(p0.kvStep, a)
    assert (s.add.id, s.addn) == (0, 0)
    name, s = sent(p0.kvCompact, a)
    assert name == "p0_kv_compact" and (s.ref.id, s.to_table.id, s.to_ref.id, s.stat.id) == (9, 10, 12, 13)
    name, s = sent(p0.beamSelect, {"logits": {"buf": FakeBuf(1), "ld": 200}, "score": {"buf": FakeBuf(2)}, "groups": 2, "beams": 3, "V": 100,
                                   "parent": {"buf": FakeBuf(4)}, "token": {"buf": FakeBuf(5)}, "scoreOut": {"buf": FakeBuf(6)}})
    assert name == "p0_beam_select" and (s.logits.id, s.ld, s.score.id, s.fin.id, s.groups, s.beams, s.V, s.eos, s.parent.id, s.token.id, s.score_out.id,
                                         s.fin_out.id) == (1, 200, 2, 0, 2, 3, 100, L.P0_KV_NONE, 4, 5, 6, 0)


def test_bound_repeats_the_call():
    g = FakeGpu()
    call = p0.bound(p0.kv4Put, g, {"kv": kv(), "k": {"buf": FakeBuf(5)}, "v": {"buf": FakeBuf(6)}, "n": 2, "T": 1})
    assert not g._lib.calls
    call()
    call()
    assert [n for n, _ in g._lib.calls] == ["p0_kv4_put"] * 2


# ---------------------------------------------------------------- the tests' own statements
def test_ref_quantise_matches_the_packer():
    # away from borders of two codes, f32 and the packer's f64 agree
    from oracle import ref
    W = np.round(ref.randn(64 * 64, 5, 1.0) * 64) / 64
    want, deq = ref.pack_q4(W.astype(np.float32), 64, 64)
    c = R.Cache(np.random.default_rng(0), [64], 1, 64)
    for r in range(64):
        c.write(0, r, 0, 0, W.reshape(64, 64)[r])
    got = c.pool[c.table[0, 0], :2 * 1280]
    same = got == want[:2 * 1280]
    assert same.mean() > 0.999
    q, s, mn = R.quantise(np.array([[0.0] * 32, [np.nan, np.inf, -np.inf] + [1.0] * 29], np.float32))
    assert s[0] == 1 and not q[0].any() and np.isfinite(R.stands_for(q, s, mn)).all() and abs(R.stands_for(q, s, mn)[1, 1] - 6e4) < 4000


def test_ref_step_by_hand():
    # two rows sharing page 5; row 0 of 70 tokens (tail 2), row 1 of 64 + 1 (tail 3)
    table = np.array([[5, 2, R.NONE], [5, 3, R.NONE]], np.uint32)
    ref = np.array([0, 0, 1, 1, 0, 2], np.uint32)
    t, n, r, stat, copies = R.step(table, np.array([70, 65], np.uint32), ref, 6, [0, 0], 1)
    assert t.tolist() == [[5, 2, R.NONE], [5, 0, R.NONE]] and n.tolist() == [71, 71] and copies == [(2, 0)]
    assert r.tolist() == [1, 0, 1, 0, 0, 2] and stat == (0, 3)
    t, r, stat, moves = R.compact(t, r, 6)
    assert stat == (3, 1) and moves == [(5, 1)] and t.tolist() == [[1, 2, R.NONE], [1, 0, R.NONE]] and r.tolist() == [1, 2, 1, 0, 0, 0]


def test_ref_beam_by_hand():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.9, 0.05, 0.05]], np.float32))
    parent, token, score, fin = R.beam(x, np.array([0.0, -1.0], np.float32), 1, 2, 0)
    assert parent.tolist() == [0, 1] and token.tolist() == [0, 0] and fin.tolist() == [1, 1]
    assert np.allclose(score, [np.log(0.5), -1 + np.log(0.9)])


def test_beam_search_refuses_its_width():
    from p0pc0rn_b200 import beam
    cfg = {"beams": 9, "D": 512, "NH": 4, "NKV": 1, "hd": 128, "FF": 512, "vocab": 64, "kinds": ["full"], "eos": 0}
    for m in (0, 9):
        with pytest.raises(ValueError, match="1 to 8"):
            beam.BeamSearch(None, {**cfg, "beams": m}, None, 64)
