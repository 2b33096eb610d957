"""packF8, normF8 and gemmF8 against the 64-bit statements of tests/f8_ref.py, over types, lengths, odd sizes, strides, offsets
and values that hurt; outputs beyond what a call writes stay as they were."""
import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import f8_ref as R

pytestmark = pytest.mark.gpu
TYPE = {"f32": np.float32, "f16": np.float16}
FILL = 0x5b          # what outputs hold before a call


class Rows:
    """rows in a buffer with an offset, a stride and something else between and behind them"""

    def __init__(self, g, x, ld=0, off=0, fill=None):
        M, K = x.shape
        self.g, self.dt, self.shape, self.ld, self.off = g, x.dtype, x.shape, ld or K, off
        n = off + (M - 1) * self.ld + K + 24
        host = np.full(n * x.dtype.itemsize, FILL, np.uint8).view(x.dtype) if fill is None else np.full(n, fill, x.dtype)
        self.at = (off + np.arange(M)[:, None] * self.ld + np.arange(K)).ravel()
        host[self.at] = x.ravel()
        self.before, self.buf = host, g.upload(host)

    def arg(self, **more):
        return {"buf": self.buf, "off": self.off, "ld": self.ld, **more}

    def read(self):
        """the rows; what lies between them has to be as it was"""
        host = self.g.read(self.buf).view(self.dt)[:self.before.size]
        other = np.ones(host.size, bool)
        other[self.at] = False
        assert host[other].tobytes() == self.before[other].tobytes()
        return host[self.at].reshape(self.shape)


class Mat:
    """a matrix in 8 bits: from codes and scales, or an output"""

    def __init__(self, g, q, s, ld=0, off=0, s_ld=0, s_off=0, poison=True):
        self.q = Rows(g, q, ld or -(-q.shape[1] // 16) * 16, off, 0x7f if poison else None)              # NaN codes
        self.s = Rows(g, s, s_ld or s.shape[1], s_off, np.nan if poison else None)

    def arg(self):
        return self.q.arg(s=self.s.arg())

    def read(self):
        return self.q.read(), self.s.read()


def out_mat(g, M, K, tile=False, ld=0, off=0, s_ld=0, s_off=0):
    s = np.full((R.blocks(M), R.blocks(K)) if tile else (R.blocks(K), M), -1, np.float32)
    return Mat(g, np.full((M, K), FILL, np.uint8), s, ld, off, s_ld, s_off, poison=False)


def rand_mat(g, rng, M, K, tile=False, **lay):
    """a quantised random matrix on the device, and the values it stands for"""
    x = rng.standard_normal((M, K)).astype(np.float32)
    if not tile:
        x *= np.exp(rng.standard_normal((M, 1))).astype(np.float32)
    q, s = R.quantise(x, tile)
    return Mat(g, q, s, **lay), R.values(q, s, tile)


# ---------------------------------------------------------------- packF8
PACK = [(1, 1), (1, 16), (3, 127), (2, 128), (5, 129), (128, 300), (129, 256), (33, 1000), (260, 143), (1, 5000), (1000, 8)]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("M,K", PACK)
def test_pack(g, M, K, block, kind):
    rng = np.random.default_rng(M * 1000 + K)
    x = (rng.standard_normal((M, K)) * np.exp(3 * rng.standard_normal((M, 1)))).astype(TYPE[kind])
    src, tile = Rows(g, x), block == "tile"
    y = out_mat(g, M, K, tile)
    p0.packF8(g, {"x": src.arg(), "type": kind, "M": M, "K": K, "block": block, "y": y.arg()})
    q, s = y.read()
    wq, ws = R.quantise(x, tile)
    assert (s == ws).all() and (q == wq).all()            # the same steps in f32, bit for bit
    src.read()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("ld,off", [(208, 0), (208, 8), (201, 0), (208, 3)])   # 16-byte rows, an odd stride, an odd start
def test_pack_layouts(g, block, kind, ld, off):
    M, K, tile = 140, 200, block == "tile"
    x = np.random.default_rng(ld + off).standard_normal((M, K)).astype(TYPE[kind])
    src = Rows(g, x, ld, off)
    y = out_mat(g, M, K, tile, ld=240, off=32, s_ld=(7 if tile else 151), s_off=5)
    p0.packF8(g, {"x": src.arg(), "type": kind, "M": M, "K": K, "block": block, "y": y.arg()})
    q, s = y.read()
    wq, ws = R.quantise(x, tile)
    assert (s == ws).all() and (q == wq).all()


@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_pack_hard_values(g, block, kind):
    M, K, tile = 6, 400, block == "tile"
    x = np.random.default_rng(0).standard_normal((M, K)).astype(np.float32)
    if kind == "f32":
        x[0] *= 1e-38          # below the floor of a block's maximum
        with np.errstate(over="ignore"):
            x[1] *= 1e38
    x[2] = 0
    x[3, 5], x[3, 300] = np.nan, -np.nan
    x[4, 7], x[4, 399] = np.inf, -np.inf
    x[5] = -0.0
    with np.errstate(over="ignore"):
        x = x.astype(TYPE[kind])
    y = out_mat(g, M, K, tile)
    p0.packF8(g, {"x": Rows(g, x).arg(), "type": kind, "M": M, "K": K, "block": block, "y": y.arg()})
    q, s = y.read()
    wq, ws = R.quantise(x, tile)
    assert (s == ws).all() and (q == wq).all() and np.isfinite(s).all()


# ---------------------------------------------------------------- normF8
# a sum of n squares by 16 at a lane, then trees and up to 32 in order: 60 roundings of 2^-24, halved by the root; rsqrtf 2^-22, three products
SLACK = 60 * 2.0 ** -25 + 2.0 ** -22 + 4 * 2.0 ** -24


def run_norm(g, M, D, kind="f32", t=None, parts=1, post=False, h="own", st=True, scale=1.0, eps=0.0, ld=0, off=0, seed=0, x=None, misalign=0):
    rng = np.random.default_rng(M * 7 + D + seed)
    if x is None:
        x = (rng.standard_normal((M, D)) * np.exp(rng.standard_normal((M, 1)))).astype(TYPE[kind])
    xs = Rows(g, x, ld, off)
    w = (1 + 0.3 * rng.standard_normal((1, D))).astype(np.float32)
    wb, pb = Rows(g, w, off=misalign), None
    y = out_mat(g, M, D, ld=-(-D // 16) * 16 + 16, s_ld=M + 3, s_off=2)
    a = {"x": xs.arg(), "type": kind, "w": wb.arg(), "y": y.arg(), "M": M, "D": D, "scale": scale, "eps": eps}
    tv = pw = None
    if t:
        tv = rng.standard_normal((parts, M, D)).astype(TYPE[t])
        tb = Rows(g, tv.reshape(parts * M, D), ld, off)
        a["t"] = tb.arg(type=t, n=parts, ld=M * tb.ld, ldm=tb.ld)
        if post:
            pw = (1 + 0.3 * rng.standard_normal((1, D))).astype(np.float32)
            pb = Rows(g, pw, off=misalign)
            a["pw"] = pb.arg()
    hs = xs
    if h == "own" and t:
        hs = Rows(g, np.zeros_like(x), ld and ld + 16, off)
        a["h"] = hs.arg()
    sb = Rows(g, np.full((1, M), -1, np.float32), off=3)
    if st:
        a["st"] = sb.arg()
    p0.normF8(g, a)
    got = hs.read()
    want, _, _ = R.norm(x, tv, pw[0] if pw is not None else None, w[0], eps or 1e-6, scale)
    if t or scale != 1.0:
        size = np.abs(x.astype(np.float64)) + (np.abs(tv.astype(np.float64)).sum(0) * (4 if post else 1) if t else 0)
        half = 2.0 ** -11 if kind == "f16" else 2.0 ** -24
        assert (np.abs(got.astype(np.float64) - want) <= np.abs(want) * half + 2.0 ** -25 + np.abs(scale) * size * (SLACK + (parts + 2) * 2.0 ** -24)).all()
    else:
        assert got.tobytes() == x.tobytes()
    if hs is not xs:
        xs.read()
    _, wst, wy = R.norm(x, tv, pw, w[0], eps or 1e-6, scale, got)
    if st:
        assert (np.abs(sb.read()[0] - wst) <= wst * SLACK).all()
    q, s = y.read()
    R.check_codes(q, s, wy, SLACK)
    return q, s


@pytest.mark.parametrize("D", [1, 8, 100, 127, 128, 129, 256, 264, 500, 512, 1536, 2240, 8192, 8200, 16384])
@pytest.mark.parametrize("M", [1, 5])
def test_norm_plain(g, M, D):
    run_norm(g, M, D)


@pytest.mark.parametrize("kind,t", [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("M,D,parts,post,h", [(1, 2560, 2, True, "x"), (3, 136, 1, False, "own"), (7, 1000, 3, True, "own"), (301, 520, 1, False, "x"), (300, 250, 1, True, "own"),
                                              (310, 60, 2, True, "x"), (299, 2240, 1, True, "own"), (1, 9000, 1, False, "x"), (2, 16383, 2, True, "own"),
                                              (320, 16384, 1, True, "x"), (450, 9216, 2, False, "own"), (1700, 1536, 1, True, "x"), (2900, 264, 1, False, "own")])
def test_norm_residual(g, kind, t, M, D, parts, post, h):
    run_norm(g, M, D, kind, t, parts, post, h)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("ld,off,misalign", [(208, 8, 0), (201, 0, 0), (208, 3, 0), (208, 8, 1)])
def test_norm_layouts(g, kind, ld, off, misalign):
    run_norm(g, 9, 200, kind, kind, 2, True, "own", ld=ld, off=off, misalign=misalign)
    run_norm(g, 400, 200, kind, kind, 1, False, "x", ld=ld, off=off, misalign=misalign)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_norm_scale_eps_no_st(g, kind):
    run_norm(g, 4, 300, kind, kind, 1, True, scale=0.125, eps=0.5)
    run_norm(g, 4, 300, kind, None, scale=-2.0, st=False)
    run_norm(g, 4, 300, kind, None, st=False)


def test_norm_rows_of_zeros_and_nan(g):
    x = np.random.default_rng(3).standard_normal((3, 300)).astype(np.float32)
    x[0] = 0
    x[1, 17] = np.nan
    xs, w, y, st = Rows(g, x), Rows(g, np.ones((1, 300), np.float32)), out_mat(g, 3, 300), Rows(g, np.zeros((1, 3), np.float32))
    p0.normF8(g, {"x": xs.arg(), "w": w.arg(), "y": y.arg(), "st": st.arg(), "M": 3, "D": 300})
    q, s = y.read()
    assert not q[0].any() and (s[:, 0] == np.float32(2.0 ** -100) / np.float32(448)).all() and abs(st.read()[0, 0] - 1e3) < 1
    assert ((q[1] & 127) == 127).all() and np.isnan(st.read()[0, 1])
    R.check_codes(q[2:], s[:, 2:], R.norm(x[2:], None, None, np.ones(300), 1e-6, 1.0)[2], SLACK)


def test_norm_is_that_of_the_stored_stream(g):
    # the codes of a call that adds equal those of a plain call on the stream that it left
    rng = np.random.default_rng(9)
    x, t = rng.standard_normal((40, 700)).astype(np.float16), rng.standard_normal((40, 700)).astype(np.float16)
    w, xs = Rows(g, np.ones((1, 700), np.float32)), Rows(g, x)
    got = []
    for more in ({"t": Rows(g, t).arg(type="f16")}, {}):
        y = out_mat(g, 40, 700)
        p0.normF8(g, {"x": xs.arg(), "type": "f16", "w": w.arg(), "y": y.arg(), "M": 40, "D": 700, **more})
        got.append(y.read())
    assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all()


# ---------------------------------------------------------------- gemmF8
ACT_SLACK = 2.0 ** -19       # the gate in f32: __expf (2 + 1.2 |x| units), a division, three products; exp's error counts where e^-x does


def run_gemm(g, M, N, K, epi="f16", bias=False, seed=0, lay=None, ylay=None, mats=None):
    rng = np.random.default_rng(M * 31 + N * 7 + K + seed)
    lay = lay or {}
    x, xv = mats[0] if mats else rand_mat(g, rng, M, K, **lay.get("x", {}))
    w, wv = mats[1] if mats else rand_mat(g, rng, N, K, True, **lay.get("w", {}))
    a = {"x": x.arg(), "w": w.arg(), "M": M, "N": N, "K": K, "epi": epi}
    want, size = R.product(xv, wv)
    err = size * R.sum_bound(K)
    if epi in ("swiglu", "geglu"):
        u, uv = mats[2] if mats else rand_mat(g, rng, N, K, True, **lay.get("u", {}))
        a["u"] = u.arg()
        up, usize = R.product(xv, uv)
        y = out_mat(g, M, N, **(ylay or {}))
        a["y"] = y.arg()
        p0.gemmF8(g, a)
        act = R.gate(want, epi)
        # |act'| <= 1.2 for both gates
        R.check_codes(*y.read(), act * up, ACT_SLACK, off=1.2 * err * np.abs(up) + (np.abs(act) + 1.2 * err) * usize * R.sum_bound(K) + np.abs(want * up) * 2.0 ** -22)
        return y.read()
    y = Rows(g, np.zeros((M, N), TYPE[epi]), **(ylay or {}))
    a["y"] = y.arg()
    if bias:
        bv = rng.standard_normal((1, N)).astype(np.float32)
        a["bv"] = Rows(g, bv, off=3).arg()
        want = want + bv.astype(np.float64)
    p0.gemmF8(g, a)
    got = y.read().astype(np.float64)
    tol = err + np.abs(want) * (2.0 ** -11 if epi == "f16" else 2.0 ** -24) + 2.0 ** -25 + np.abs(want) * 2.0 ** -23
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
    return got


SIZES = [(1, 1, 1), (1, 16, 16), (1, 17, 100), (2, 15, 128), (7, 128, 129), (8, 129, 256), (9, 300, 300), (16, 64, 1000), (17, 140, 127), (32, 16, 2240), (33, 300, 400),
         (64, 129, 520), (65, 64, 384), (100, 400, 640), (127, 127, 127), (128, 128, 128), (129, 257, 129), (200, 1000, 260), (257, 513, 384), (300, 64, 5000), (1, 2048, 2048),
         (500, 260, 1111)]


@pytest.mark.parametrize("epi", ["f16", "f32", "swiglu", "geglu"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_gemm(g, M, N, K, epi):
    run_gemm(g, M, N, K, epi, bias=(M + N) % 2 == 1 and epi in ("f16", "f32"))


LAY = {"x": dict(ld=464, off=48, s_ld=1031, s_off=3), "w": dict(ld=448, off=16, s_ld=9, s_off=1), "u": dict(ld=416, off=64, s_ld=4, s_off=7)}


@pytest.mark.parametrize("M", [1, 12, 40, 150, 1029])
@pytest.mark.parametrize("epi", ["f16", "f32", "swiglu"])
@pytest.mark.parametrize("ld,off", [(0, 0), (288, 32), (293, 1), (284, 4)])
def test_gemm_layouts(g, M, epi, ld, off):
    ylay = dict(ld=ld, off=off) if epi != "swiglu" else dict(ld=-(-(ld or 280) // 16) * 16, off=off // 16 * 16, s_ld=M + (ld & 7), s_off=off & 7)
    run_gemm(g, M, 280, 400, epi, lay=LAY, ylay=ylay)


@pytest.mark.parametrize("epi", ["f16", "f32", "geglu"])
@pytest.mark.parametrize("ld,off", [(1120, 32), (1109, 3), (1116, 4)])     # rows of y on 16 bytes, on none, f32 alone
def test_gemm_layouts_many_tokens(g, epi, ld, off):
    M, N, K = 2100, 1101, 400
    lay = {"x": dict(ld=464, off=48, s_ld=2107, s_off=3), "w": dict(ld=448, off=16, s_ld=9, s_off=1), "u": dict(ld=416, off=64, s_ld=4, s_off=7)}
    run_gemm(g, M, N, K, epi, bias=epi == "f32", lay=lay, ylay=dict(ld=ld, off=off) if epi != "geglu" else dict(ld=-(-ld // 16) * 16, off=off // 16 * 16, s_ld=M + 5, s_off=off & 7))


@pytest.mark.parametrize("M,N,K", [(1100, 1300, 700), (2100, 520, 2240), (300, 4000, 1024)])
@pytest.mark.parametrize("epi", ["f16", "f32", "geglu"])
def test_gemm_large(g, M, N, K, epi):
    run_gemm(g, M, N, K, epi, bias=epi == "f32")


@pytest.mark.parametrize("M", [1, 3, 20, 130, 600])
def test_gemm_scales_far_apart(g, M):
    # blocks of very different sizes: a sum that went through one accumulator unscaled would lose the small ones
    rng = np.random.default_rng(M)
    N, K = 200, 640
    x = rng.standard_normal((M, K)).astype(np.float32) * np.repeat(np.float32([1e-6, 1e4, 1e-3, 1e8, 1.0]), 128)
    w = rng.standard_normal((N, K)).astype(np.float32) * np.repeat(np.float32([1e6, 1e-4, 1e3, 1e-8, 1.0]), 128)
    (xq, xs), (wq, ws) = R.quantise(x), R.quantise(w, True)
    run_gemm(g, M, N, K, "f32", mats=[(Mat(g, xq, xs), R.values(xq, xs)), (Mat(g, wq, ws), R.values(wq, ws, True))])


@pytest.mark.parametrize("M", [2, 40, 400])
def test_gemm_largest_and_smallest_codes(g, M):
    # every product 448 * 448, or the smallest subnormal's: sums beyond f16, below its subnormals
    N, K = 130, 300
    for code in (0x7e, 0x01, 0x81):
        q, s = np.full((M, K), code, np.uint8), np.ones((3, M), np.float32)
        wq, ws = np.full((N, K), 0x7e if code == 0x7e else 0x01, np.uint8), np.ones((2, 3), np.float32)
        run_gemm(g, M, N, K, "f32", mats=[(Mat(g, q, s), R.values(q, s)), (Mat(g, wq, ws), R.values(wq, ws, True))])


@pytest.mark.parametrize("M", [4, 60, 500])
@pytest.mark.parametrize("epi", ["f16", "f32", "swiglu"])
def test_gemm_nan_stays_in_its_row(g, M, epi):
    rng = np.random.default_rng(M)
    N, K = 260, 300
    q, s = R.quantise(rng.standard_normal((M, K)).astype(np.float32))
    wq, ws = R.quantise(rng.standard_normal((N, K)).astype(np.float32), True)
    q[1, 299] = 0x7f
    x, w = Mat(g, q, s), Mat(g, wq, ws)
    a = {"x": x.arg(), "w": w.arg(), "M": M, "N": N, "K": K, "epi": epi}
    if epi == "swiglu":
        y = out_mat(g, M, N)
        p0.gemmF8(g, {**a, "u": w.arg(), "y": y.arg()})
        nan = (y.read()[0] & 127) == 127
        assert np.isfinite(y.read()[1]).all()
    else:
        y = Rows(g, np.zeros((M, N), TYPE[epi]))
        p0.gemmF8(g, {**a, "y": y.arg()})
        nan = np.isnan(y.read())
    assert nan[1].all() and not nan[[0] + list(range(2, M))].any()


@pytest.mark.parametrize("epi", ["f16", "swiglu"])
@pytest.mark.parametrize("M", [1, 16, 100, 700])
def test_gemm_repeats_bit_for_bit(g, M, epi):
    rng = np.random.default_rng(M)
    x, w, u = rand_mat(g, rng, M, 900), rand_mat(g, rng, 600, 900, True), rand_mat(g, rng, 600, 900, True)
    first = run_gemm(g, M, 600, 900, epi, mats=[x, w, u])
    for _ in range(4):
        again = run_gemm(g, M, 600, 900, epi, mats=[x, w, u])
        assert all((np.asarray(p) == np.asarray(q)).all() for p, q in zip(first, again))


@pytest.mark.parametrize("M", [3, 50, 400])
@pytest.mark.parametrize("epi", ["swiglu", "geglu"])
def test_gemm_gates_far_out(g, M, epi):
    # gates from -2000 to 2000: the exponentials leave f32 on either side
    N, K = 150, 128
    q, s = np.full((M, K), 0x38, np.uint8), np.repeat(np.float32(2.0) ** np.linspace(-12, 4, M, dtype=np.float32)[None], 1, 0).astype(np.float32)
    wq, ws = np.where(np.arange(N)[:, None] % 2, 0x38, 0xb8) + np.zeros((1, K), np.int64), np.ones((2, 1), np.float32)
    w = (Mat(g, wq.astype(np.uint8), ws), R.values(wq.astype(np.uint8), ws, True))
    u = (Mat(g, np.full((N, K), 0x38, np.uint8), ws), R.values(np.full((N, K), 0x38, np.uint8), ws, True))
    codes, scales = run_gemm(g, M, N, K, epi, mats=[(Mat(g, q, s), R.values(q, s)), w, u])
    assert np.isfinite(scales).all() and not ((codes & 127) == 127).any()


# ---------------------------------------------------------------- together, on streams and in graphs
def layer(g, M, D, F, seed):
    """an MLP's buffers: x, norm weights, gate / up / down weights, and the calls that run it: normF8 -> gemmF8 (gated, codes) -> gemmF8 (f16) -> normF8"""
    rng = np.random.default_rng(seed)
    b = {"x": Rows(g, rng.standard_normal((M, D)).astype(np.float32)), "w1": Rows(g, (1 + 0.2 * rng.standard_normal((1, D))).astype(np.float32)),
         "pw": Rows(g, (1 + 0.2 * rng.standard_normal((1, D))).astype(np.float32)), "h": Rows(g, np.zeros((M, D), np.float32)), "xn": out_mat(g, M, D), "mid": out_mat(g, M, F),
         "down": Rows(g, np.zeros((M, D), np.float16)), "out": out_mat(g, M, D), "st": Rows(g, np.zeros((1, M), np.float32))}
    for name, n, k in (("gate", F, D), ("up", F, D), ("proj", D, F)):      # weights as a program makes them: packed on the device
        src, b[name] = Rows(g, (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)), out_mat(g, n, k, True)
        p0.packF8(g, {"x": src.arg(), "M": n, "K": k, "block": "tile", "y": b[name].arg()})
        b[name + "_f32"] = src
    a = [(p0.normF8, {"x": b["x"].arg(), "w": b["w1"].arg(), "y": b["xn"].arg(), "M": M, "D": D}),
         (p0.gemmF8, {"x": b["xn"].arg(), "w": b["gate"].arg(), "u": b["up"].arg(), "M": M, "N": F, "K": D, "epi": "geglu", "y": b["mid"].arg()}),
         (p0.gemmF8, {"x": b["mid"].arg(), "w": b["proj"].arg(), "M": M, "N": D, "K": F, "y": b["down"].arg()}),
         (p0.normF8, {"x": b["x"].arg(), "t": b["down"].arg(type="f16"), "pw": b["pw"].arg(), "h": b["h"].arg(), "w": b["w1"].arg(), "y": b["out"].arg(), "st": b["st"].arg(),
                      "M": M, "D": D})]
    return b, [p0.bound(op, g, x) for op, x in a]


def check_layer(b, M, D, F):
    """every step against 64 bits on what the step before left"""
    val = lambda m, tile=False: R.values(*m.read(), tile)
    for name in ("gate", "up", "proj"):
        q, s = R.quantise(b[name + "_f32"].read(), True)
        assert (b[name].read()[0] == q).all() and (b[name].read()[1] == s).all()
    R.check_codes(*b["xn"].read(), R.norm(b["x"].read(), None, None, b["w1"].read()[0], 1e-6, 1.0)[2], SLACK)
    xv = val(b["xn"])
    (g1, s1), (u1, s2) = R.product(xv, val(b["gate"], True)), R.product(xv, val(b["up"], True))
    e, act = R.sum_bound(D), R.gate(g1, "geglu")
    R.check_codes(*b["mid"].read(), act * u1, ACT_SLACK, off=1.2 * e * s1 * np.abs(u1) + (np.abs(act) + 1.2 * e * s1) * s2 * e + np.abs(g1 * u1) * 2.0 ** -22)
    want, size = R.product(val(b["mid"]), val(b["proj"], True))
    down = b["down"].read().astype(np.float64)
    assert (np.abs(down - want) <= size * R.sum_bound(F) + np.abs(want) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all()
    h = b["h"].read()
    wh, wst, wy = R.norm(b["x"].read(), b["down"].read()[None], b["pw"].read()[0], b["w1"].read()[0], 1e-6, 1.0, h)
    assert (np.abs(h - wh) <= np.abs(wh) * 2.0 ** -23 + (np.abs(b["x"].read()) + 4 * np.abs(down)) * (SLACK + 2.0 ** -22)).all()
    assert (np.abs(b["st"].read()[0] - wst) <= wst * SLACK).all()
    R.check_codes(*b["out"].read(), wy, SLACK)


@pytest.mark.parametrize("M,D,F", [(1, 256, 512), (9, 520, 1100), (70, 520, 1100), (400, 640, 1300)])
def test_layer(g, M, D, F):
    b, calls = layer(g, M, D, F, M)
    for c in calls:
        c()
    check_layer(b, M, D, F)
    # and what it comes to: the whole in 64 bits without codes. Each rounding to e4m3 is up to 2^-4 of a value, 2^-4 / sqrt(3) of it on
    # average; four roundings (x, weights, gated results, weights) meet in the sums: 4 * 2^-4 / sqrt(3) < 0.15 of the result's size
    x, w = b["x"].read().astype(np.float64), {k: b[k + "_f32"].read().astype(np.float64) for k in ("gate", "up", "proj")}
    xn = R.norm(x, None, None, b["w1"].read()[0], 1e-6, 1.0)[2]
    want = (R.gate(xn @ w["gate"].T, "geglu") * (xn @ w["up"].T)) @ w["proj"].T
    got = b["down"].read().astype(np.float64)
    assert np.linalg.norm(got - want) <= 0.15 * np.linalg.norm(want)


def test_layer_on_torch_streams_and_in_graphs(g):
    """the calls on a stream of torch's; captured, replayed with other inputs; two captured graphs side by side on streams of their own"""
    import torch
    own = p0.Gpu(0)
    try:
        shapes = [(5, 264, 520), (300, 520, 700)]
        side = torch.cuda.Stream()
        own.set_stream(side.cuda_stream)
        made = [layer(own, M, D, F, 50 + M) for M, D, F in shapes]
        for _, calls in made:
            for c in calls:
                c()
        for (b, _), s in zip(made, shapes):
            check_layer(b, *s)
        graphs = []
        for b, calls in made:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                for c in calls:
                    c()
            graphs.append(graph)
        rng = np.random.default_rng(1)
        for (b, _), (M, D, F) in zip(made, shapes):
            new = b["x"].before.copy()
            new[b["x"].at] = rng.standard_normal(M * D).astype(np.float32)
            own.write(b["x"].buf, new)
            b["x"].before = new
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(3):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for (b, _), s in zip(made, shapes):
            check_layer(b, *s)
        del graphs
    finally:
        own.close()


def test_calls_back_to_back_overlap_rightly(g):
    # programmatic launches: each call reads what the one before wrote, in place, many times over
    M, D = 20, 640
    x = np.random.default_rng(2).standard_normal((M, D)).astype(np.float32)
    xs, t, w, y = Rows(g, x), Rows(g, np.full((M, D), 0.25, np.float32)), Rows(g, np.ones((1, D), np.float32)), out_mat(g, M, D)
    call = p0.bound(p0.normF8, g, {"x": xs.arg(), "t": t.arg(), "w": w.arg(), "y": y.arg(), "M": M, "D": D})
    for _ in range(64):
        call()
    want = x.copy()
    for _ in range(64):
        want = (want + np.float32(0.25)).astype(np.float32)
    assert (xs.read() == want).all()
    R.check_codes(*y.read(), R.norm(want, None, None, np.ones(D), 1e-6, 1.0)[2], SLACK)


def test_refused_calls_leave_the_context_usable(g):
    x, w = rand_mat(g, np.random.default_rng(0), 4, 64)[0], rand_mat(g, np.random.default_rng(1), 16, 64, True)[0]
    y = Rows(g, np.zeros((4, 16), np.float16))
    with pytest.raises(p0.P0Error, match="gemmF8: K is 0"):
        p0.gemmF8(g, {"x": x.arg(), "w": w.arg(), "M": 4, "N": 16, "K": 0, "y": y.arg()})
    with pytest.raises(p0.P0Error, match="x range"):
        p0.gemmF8(g, {"x": {**x.arg(), "off": 1 << 20}, "w": w.arg(), "M": 4, "N": 16, "K": 64, "y": y.arg()})
    run_gemm(g, 4, 16, 64)
    g.done()
