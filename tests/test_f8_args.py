"""The 8-bit operators on CPU (no kernel runs): the argument objects as C structs, the structs' layout against
include/p0mm.h, the calls that the library refuses before it launches anything, and the tests' own statements."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import p0pc0rn_b200 as p0
from p0pc0rn_b200 import _lib as L

from . import f8_ref as R
from .test_ops_args import FakeBuf, FakeGpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = ["p0_f8", "p0_pack_f8_args", "p0_norm_f8_args", "p0_gemm_f8_args"]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layout_matches_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "p0mm.h"', "int main(void) {",
             '  printf("%d %d %d %d %d %d %u\\n", P0_F8_ROW, P0_F8_TILE, P0_F8EPI_F16, P0_F8EPI_F32, P0_F8EPI_SWIGLU, P0_F8EPI_GEGLU, P0_F8_MAX_D);']
    for s in STRUCTS:
        lines.append('  printf("%s %%zu\\n", sizeof(%s));' % (s, s))
        for f, _ in getattr(L, s)._fields_:
            lines.append('  printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (s, f, s, f))
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines()
    E, K = L.F8EPI, L.F8BLOCK
    assert out[0] == "%d %d %d %d %d %d %d" % (K["row"], K["tile"], E["f16"], E["f32"], E["swiglu"], E["geglu"], L.P0_F8_MAX_D)
    got = dict(x.rsplit(" ", 1) for x in out[1:])
    for s in STRUCTS:
        cls = getattr(L, s)
        assert int(got[s]) == ctypes.sizeof(cls), s
        for f, _ in cls._fields_:
            assert int(got["%s.%s" % (s, f)]) == getattr(cls, f).offset, (s, f)


def sent(op, a):
    g = FakeGpu()
    op(g, a)
    (name, rec), = g._lib.calls
    return name, rec[0]


def f8(i, **more):
    return {"buf": FakeBuf(i), "off": 32, "ld": 256, "s": {"buf": FakeBuf(i + 1), "off": 5, "ld": 9}, **more}


def same8(m, i):
    return (m.buf.id, m.off, m.ld, m.s.id, m.s_off, m.s_ld) == (i, 32, 256, i + 1, 5, 9)


def test_pack_arguments():
    name, s = sent(p0.packF8, {"x": {"buf": FakeBuf(1), "off": 3, "ld": 700}, "type": "f16", "M": 5, "K": 200, "block": "tile", "y": f8(2)})
    assert name == "p0_pack_f8" and (s.x.id, s.x_off, s.x_ld, s.type, s.M, s.K, s.block) == (1, 3, 700, 1, 5, 200, 1) and same8(s.y, 2)
    _, s = sent(p0.packF8, {"x": {"buf": FakeBuf(1)}, "M": 5, "K": 200, "y": {"buf": FakeBuf(2), "s": {"buf": FakeBuf(3)}}})
    assert (s.x_off, s.x_ld, s.type, s.block, s.y.off, s.y.ld, s.y.s_off, s.y.s_ld) == (0,) * 8
    with pytest.raises(p0.P0Error, match="packF8: type bf16"):
        sent(p0.packF8, {"x": {"buf": FakeBuf(1)}, "type": "bf16", "M": 5, "K": 200, "y": f8(2)})
    with pytest.raises(p0.P0Error, match="packF8: block column"):
        sent(p0.packF8, {"x": {"buf": FakeBuf(1)}, "M": 5, "K": 200, "block": "column", "y": f8(2)})


def test_norm_arguments():
    name, s = sent(p0.normF8, {"x": {"buf": FakeBuf(1), "off": 3, "ld": 700}, "type": "f16", "t": {"buf": FakeBuf(2), "off": 4, "ld": 1 << 33, "ldm": 650,
                               "type": "f32", "n": 3}, "pw": {"buf": FakeBuf(3), "off": 6}, "h": {"buf": FakeBuf(4), "off": 7, "ld": 600},
                               "w": {"buf": FakeBuf(5), "off": 8}, "y": f8(6), "st": {"buf": FakeBuf(8), "off": 9}, "M": 10, "D": 512, "eps": 0.5, "scale": 0.25})
    assert name == "p0_norm_f8" and same8(s.y, 6)
    assert (s.x.id, s.x_off, s.x_ld, s.type, s.t.id, s.t_off, s.t_ld, s.t_ldm, s.t_type, s.t_n, s.pw.id, s.pw_off, s.h.id, s.h_off, s.h_ld, s.w.id, s.w_off,
            s.st.id, s.st_off, s.M, s.D, s.eps, s.scale) == (1, 3, 700, 1, 2, 4, 1 << 33, 650, 0, 3, 3, 6, 4, 7, 600, 5, 8, 8, 9, 10, 512, 0.5, 0.25)
    _, s = sent(p0.normF8, {"x": {"buf": FakeBuf(1)}, "w": {"buf": FakeBuf(5)}, "y": f8(6), "M": 1, "D": 64})
    assert (s.type, s.t.id, s.t_type, s.t_n, s.pw.id, s.h.id, s.st.id, s.eps, s.scale) == (0, 0, 0, 0, 0, 0, 0, 0.0, 1.0)
    with pytest.raises(p0.P0Error, match="normF8: type f64"):
        sent(p0.normF8, {"x": {"buf": FakeBuf(1)}, "t": {"buf": FakeBuf(2), "type": "f64"}, "w": {"buf": FakeBuf(5)}, "y": f8(6), "M": 1, "D": 64})


def test_gemm_arguments():
    name, s = sent(p0.gemmF8, {"x": f8(1), "w": f8(3), "u": f8(5), "M": 7, "N": 8, "K": 9, "epi": "geglu", "y": f8(7)})
    assert name == "p0_gemm_f8" and same8(s.x, 1) and same8(s.w, 3) and same8(s.u, 5) and same8(s.y, 7)
    assert (s.M, s.N, s.K, s.epi, s.bv.id, s.bv_off) == (7, 8, 9, 3, 0, 0)
    _, s = sent(p0.gemmF8, {"x": f8(1), "w": f8(3), "M": 7, "N": 8, "K": 9, "bv": {"buf": FakeBuf(5), "off": 2}, "y": {"buf": FakeBuf(6), "off": 3, "ld": 20}})
    assert (s.epi, s.u.buf.id, s.bv.id, s.bv_off, s.y.buf.id, s.y.off, s.y.ld, s.y.s.id) == (0, 0, 5, 2, 6, 3, 20, 0)
    with pytest.raises(p0.P0Error, match="gemmF8: epilogue relu"):
        sent(p0.gemmF8, {"x": f8(1), "w": f8(3), "M": 7, "N": 8, "K": 9, "epi": "relu", "y": f8(6)})
    g = FakeGpu()
    call = p0.bound(p0.gemmF8, g, {"x": f8(1), "w": f8(3), "M": 7, "N": 8, "K": 9, "y": {"buf": FakeBuf(6)}})
    call()
    call()
    assert [n for n, _ in g._lib.calls] == ["p0_gemm_f8"] * 2


# ---------------------------------------------------------------- refusals: the library's own checks, without a device
class HostGpu:
    """calls the library on a context without a device; every call made through it has to be refused"""

    def __init__(self, lib):
        self.host, self._lib = lib, L.load()
        lib.host_ctx.restype = ctypes.c_void_p
        self.ctx = ctypes.c_void_p(lib.host_ctx())
        self.n = 0

    def buf(self, size, at=None):
        self.n += 1
        self.host.host_buf(self.ctx, ctypes.c_uint64(self.n), ctypes.c_uint64(at or self.n << 32), ctypes.c_uint64(size))
        return FakeBuf(self.n)

    def _check(self, st):
        b = ctypes.create_string_buffer(512)
        self._lib.p0_last_error(self.ctx, b, 512)
        raise p0.P0Error(st, b.value.decode())


@pytest.fixture(scope="module")
def hg(tmp_path_factory):
    if not shutil.which("g++") or not os.path.exists("/usr/local/cuda/include/cuda_runtime.h"):
        pytest.skip("needs g++ and CUDA's headers")
    so = tmp_path_factory.mktemp("host") / "host.so"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I/usr/local/cuda/include", os.path.join(ROOT, "tests", "f8_host.cc"), "-o", str(so)], check=True)
    g = HostGpu(ctypes.CDLL(str(so)))
    yield g
    g.host.host_free(g.ctx)


def put(a, path, v):
    a = dict(a)
    at = a
    keys = path.split(".")
    for k in keys[:-1]:
        at[k] = dict(at[k])
        at = at[k]
    if v is None:
        at.pop(keys[-1], None)
    else:
        at[keys[-1]] = v
    return a


FakeNone = FakeBuf(0)


def refused(hg, op, a, match, status=L.P0_EINVAL):
    with pytest.raises(p0.P0Error, match=match) as e:
        op(hg, a)
    assert e.value.status == status


def mat(hg, rows, cols, tile=False):
    kb, nb = R.blocks(cols), R.blocks(rows)
    return {"buf": hg.buf((rows - 1) * (-(-cols // 16) * 16) + cols), "s": {"buf": hg.buf((nb * kb if tile else (kb - 1) * (-(-rows // 4) * 4) + rows) * 4)}}


def test_pack_refusals(hg):
    M, K = 6, 200
    a = {"x": {"buf": hg.buf(M * K * 4)}, "M": M, "K": K, "y": mat(hg, M, K)}
    small = hg.buf(M * K * 4 - 4)
    for path, v, match, st in [
            ("x.buf", small, "packF8: x range", 1), ("x.ld", 199, "x row stride 199 < 200", 1), ("x.ld", 201, "x range", 1), ("x.off", 1, "x range", 1),
            ("x.off", 1 << 62, "x offset", 1), ("x.buf", hg.buf(M * K * 4, 0x7000000000002), "x must be 4-byte aligned", 2), ("x.buf", FakeBuf(999), "not a live buffer", 1),
            ("x.buf", FakeNone, "missing binding x", 1),
            ("y.ld", 192, "y row stride 192 < 200", 1), ("y.ld", 200, "ld % 16", 2), ("y.ld", 224, "y range", 1), ("y.off", 16, "y range", 1), ("y.off", (1 << 64) - 16, "y range", 1),
            ("y.buf", hg.buf(M * 208, 0x7000000000008), "16-byte boundaries", 2), ("y.s.ld", 5, "y.s row stride 5 < 6", 1), ("y.s.ld", 9, "y.s range", 1),
            ("y.s.off", 1, "y.s range", 1), ("y.s.off", 1 << 62, "y.s offset", 1), ("y.s.buf", FakeNone, "missing binding y.s", 1),
            ("y.s.buf", hg.buf(64, 0x7000000000002), "y.s must be 4-byte aligned", 2),
            ("K", (1 << 24) + 1, "packF8: 6 x 16777217", 1), ("M", 1 << 31, "packF8: 2147483648 x", 1), ("y.buf", a["x"]["buf"], "must not lie over", 1),
            ("y.s.buf", a["x"]["buf"], "must not lie over", 1)]:
        refused(hg, p0.packF8, put(a, path, v), match, st)


def test_norm_refusals(hg):
    M, D = 5, 200
    a = {"x": {"buf": hg.buf(M * D * 2)}, "type": "f16", "t": {"buf": hg.buf(2 * M * D * 4), "n": 2}, "h": {"buf": hg.buf(M * D * 2)}, "w": {"buf": hg.buf(D * 4)},
         "pw": {"buf": hg.buf(D * 4)}, "y": mat(hg, M, D), "st": {"buf": hg.buf(M * 4)}, "M": M, "D": D}
    for path, v, match, st in [
            ("D", L.P0_F8_MAX_D + 1, "D > 16384", 1), ("x.ld", 100, "x row stride 100 < 200", 1), ("x.off", 1, "x range", 1), ("t.n", 3, "t range", 1), ("t.n", 2000, "2000 partial", 1),
            ("t.ld", 1001, "t range", 1), ("t.ld", 1 << 41, "apart", 1), ("t.ldm", 199, "t row stride 199", 1), ("t.ldm", 201, "t range", 1), ("t.off", 1, "t range", 1),
            ("h.ld", 201, "h range", 1), ("h.off", 1, "h range", 1), ("w.off", 1, "w range", 1), ("w.buf", FakeNone, "missing binding w", 1), ("pw.off", 1, "pw range", 1),
            ("st.off", 1, "st range", 1), ("y.ld", 64, "y row stride", 1), ("y.s.ld", 4, "y.s row stride", 1), ("h", {"buf": a["t"]["buf"]}, "lies over", 1),
            ("h", {"buf": a["w"]["buf"]}, "h range", 1), ("y.buf", a["x"]["buf"], "lies over", 1), ("y.buf", a["t"]["buf"], "lies over", 1),
            ("st.buf", a["w"]["buf"], "lies over", 1), ("st.buf", a["h"]["buf"], "lie over one another", 1), ("t", None, "pw without t", 1), ("M", 1 << 31, "rows", 1),
            ("st.buf", hg.buf(64, 0x7100000000001), "4-byte aligned", 2), ("x.buf", hg.buf(M * D * 2, 0x7200000000001), "2-byte aligned", 2)]:
        refused(hg, p0.normF8, put(a, path, v), match, st)
    shifted = hg.buf(M * D * 2 + 400)   # h over x, but not the same rows
    refused(hg, p0.normF8, {**a, "x": {"buf": shifted}, "h": {"buf": shifted, "off": 200}}, "lies over")
    refused(hg, p0.normF8, {**a, "x": {"buf": shifted}, "h": {"buf": shifted, "ld": 201}}, "lies over")


def test_gemm_refusals(hg):
    M, N, K = 9, 140, 200
    a = {"x": mat(hg, M, K), "w": mat(hg, N, K, True), "M": M, "N": N, "K": K, "y": {"buf": hg.buf(M * N * 2)}, "bv": {"buf": hg.buf(N * 4)}}
    for path, v, match, st in [
            ("x.ld", 192, "x row stride", 1), ("x.ld", 224, "x range", 1), ("x.ld", 201, "ld % 16", 2), ("x.off", 16, "x range", 1), ("x.s.ld", 8, "x.s row stride 8 < 9", 1), ("x.s.ld", 13, "x.s range", 1),
            ("w.ld", 224, "w range", 1), ("w.s.ld", 1, "w.s row stride 1 < 2", 1), ("w.s.ld", 3, "w.s range", 1), ("w.buf", FakeNone, "missing binding w", 1),
            ("y.ld", 139, "y row stride 139", 1), ("y.ld", 141, "y range", 1), ("y.off", 1, "y range", 1), ("bv.off", 1, "bv range", 1), ("K", 0, "K is 0", 1), ("N", 1 << 25, "N 33554432", 1),
            ("epi", "swiglu", "needs u", 1), ("u", a["w"], "u without", 1), ("y.buf", a["x"]["buf"], "range", 1), ("M", (1 << 24) + 1, "M 16777217", 1)]:
        refused(hg, p0.gemmF8, put(a, path, v), match, st)
    big = hg.buf(1 << 20)
    refused(hg, p0.gemmF8, {**a, "x": put(a["x"], "buf", big), "y": {"buf": big, "off": 800}}, "must not lie over")
    refused(hg, p0.gemmF8, {**a, "w": put(a["w"], "s.buf", big), "y": {"buf": big}}, "must not lie over")
    gated = {**a, "u": mat(hg, N, K, True), "epi": "geglu", "y": mat(hg, M, N)}
    refused(hg, p0.gemmF8, gated, "bv with a gated")
    gated.pop("bv")
    for path, v, match, st in [("y.ld", 140, "ld % 16", 2), ("y.s.ld", 8, "y.s row stride", 1), ("y.s.buf", FakeNone, "missing binding y.s", 1), ("u.s.ld", 1, "u.s row stride", 1),
                               ("y.buf", gated["u"]["buf"], "must not lie over", 1), ("y.s.buf", gated["y"]["buf"], "must not lie over", 1)]:
        refused(hg, p0.gemmF8, put(gated, path, v), match, st)


def test_empty_calls_do_nothing(hg):
    # no rows or columns: accepted before anything is looked at, as gemm's
    a = {"x": {"buf": FakeNone}, "y": {"buf": FakeNone}, "w": {"buf": FakeNone}}
    p0.packF8(hg, {**a, "M": 0, "K": 5})
    p0.normF8(hg, {**a, "M": 0, "D": 5})
    p0.gemmF8(hg, {**a, "M": 0, "N": 5, "K": 5})


# ---------------------------------------------------------------- the tests' own statements
def test_ref_codes():
    import torch
    v = np.concatenate([R.VALUE[:127], (R._POS[1:] + R._POS[:-1]) / 2, [0.0, 1e-30, 448, 463.9]]).astype(np.float32)
    v = np.concatenate([v, -v, np.random.default_rng(1).standard_normal(4000).astype(np.float32) * 100])
    assert (R.encode(v) == torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()).all()
    assert (R.encode([np.nan, np.inf, -np.inf, 1e9]) == [0x7f, 0x7e, 0xfe, 0x7e]).all()
    assert (torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()[:127] == R.VALUE[:127]).all()


def test_ref_quantise_by_hand():
    x = np.zeros((2, 130), np.float32)
    x[0, :3] = [1.0, -0.5, 0.3]
    x[1, 129] = np.nan
    x[1, 128] = -np.inf
    q, s = R.quantise(x)
    assert s[0, 0] == np.float32(1 / 448) and q[0, :2].tolist() == [0x7e, 0xf6] and abs(R.values(q, s)[0, 2] - 0.3) <= 0.3 / 16
    assert s[0, 1] == np.float32(2.0 ** -100) / np.float32(448) and not q[1, :128].any()
    assert q[1, 128:].tolist() == [0xfe, 0x7f] and s[1, 1] == R.MOST / np.float32(448)
    q, s = R.quantise(np.array([[3.0] * 129] * 129, np.float32), tile=True)
    assert s.shape == (2, 2) and (R.values(q, s, True) == np.float32(3 / 448) * np.float64(448)).all()
