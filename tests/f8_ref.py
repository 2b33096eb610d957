"""Plain statements of the 8-bit operators on the host, for the tests: the quantiser's steps in f32 as the operator defines
them, everything else in 64 bits, and how far a right answer may be off."""
import numpy as np

B, TOP, LEAST, MOST = 128, np.float32(448), np.float32(2.0 ** -100), np.finfo(np.float32).max


def _table():
    v = np.zeros(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v[c] = (f / 8 * 2.0 ** -6) if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        if c & 127 == 127:
            v[c] = np.nan
        if c & 128:
            v[c] = -v[c]
    return v


VALUE = _table()                       # of each code
_POS = VALUE[:127]                     # 0 .. 448, in order


def encode(v):
    """f32 values -> codes: nearest, halves to the even code, held at 448"""
    v = np.asarray(v, np.float64)
    a = np.minimum(np.abs(v), 448.0)
    a = np.where(np.isnan(v), 0.0, a)
    hi = np.searchsorted(_POS, a).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    c = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    c = np.where(np.signbit(v), c + 128, c)
    return np.where(np.isnan(v), 127, c).astype(np.uint8)


def blocks(n):
    return -(-n // B)


def quantise(x, tile=False):
    """[M][K] f32 -> codes u8 [M][K], scales f32 [KB][M] (or [MB][KB])"""
    x = np.asarray(x, np.float32)
    M, K = x.shape
    q = np.zeros((M, K), np.uint8)
    s = np.zeros((blocks(M), blocks(K)) if tile else (blocks(K), M), np.float32)
    step = B if tile else 1
    with np.errstate(invalid="ignore", over="ignore"):
        for m in range(0, M, step):
            for b in range(blocks(K)):
                v = x[m:m + step, b * B:(b + 1) * B]
                a = np.abs(v)
                a = np.float32(np.where(np.isnan(a), 0, a).max())
                a = min(max(a, LEAST), MOST)
                inv = np.float32(TOP / a)
                q[m:m + step, b * B:(b + 1) * B] = encode((v * inv).astype(np.float32))
                s[(m // B, b) if tile else (b, m)] = np.float32(a / TOP)
    return q, s


def values(q, s, tile=False):
    """what codes and scales stand for, f64 [M][K]"""
    M, K = q.shape
    s = s.astype(np.float64)
    if tile:
        f = np.repeat(np.repeat(s, B, 0)[:M], B, 1)[:, :K]
    else:
        f = np.repeat(s[:, :M].T, B, 1)[:, :K]
    return VALUE[q] * f


def check_codes(q, s, y, slack, off=0.0):
    """q, s against y (f64 [M][K]) whose computation in f32 may be off by slack * |y| + off: scales by that and two roundings,
    values by half a step of e4m3 (2^-4 of the value, 2^-10 scales below 2^-6) besides"""
    M, K = y.shape
    off = np.broadcast_to(off, y.shape)
    for b in range(blocks(K)):
        v, o = np.abs(y[:, b * B:(b + 1) * B]), off[:, b * B:(b + 1) * B]
        a = v.max(1)
        tol = (v * slack + o).max(1) + a * 2.0 ** -22
        assert (np.abs(s[b, :M].astype(np.float64) * 448 - np.maximum(a, 2.0 ** -100)) <= tol + 2.0 ** -120).all()
    got = values(q, s)
    sc = np.repeat(s[:, :M].T.astype(np.float64), B, 1)[:, :K]
    err = np.abs(got - y)
    # y itself may lie past the border between two codes by what its computation is off (twice: its scale is off as well); 2^-22: the
    # rounded product with 448 / a and the scale
    tol = np.maximum(np.abs(y) * (2.0 ** -4 + 2.0 ** -22), sc * 2.0 ** -10) + 2 * (np.abs(y) * slack + off)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())


def gate(x, epi):
    z = x if epi == "swiglu" else 2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)
    with np.errstate(over="ignore"):
        return x / (1 + np.exp(-z))


def sum_bound(K):
    """of sum |x w|: how far a product's sums in f32 may be off. Products of codes are exact. A block's 128 are summed by the tensor cores
    in f32, at worst cut off at each of 128 additions (2^-23), then scaled (the scales' product and the fma, 2^-24 each) and added
    to as many blocks before and, by parts, in up to 16 more additions"""
    return 128 * 2.0 ** -23 + (blocks(K) + 18) * 2.0 ** -24


def product(x, w):
    """(sum x w, sum |x w|) in f64 of values [M][K], [N][K]"""
    return x @ w.T, np.abs(x) @ np.abs(w).T


def norm(x, tv, pw, w, eps, scale, h=None):
    """(h, st, y) in f64; the norm is of `h` if given (the rounded stream as the operator left it)"""
    x = x.astype(np.float64)
    if tv is not None:
        tv = tv.astype(np.float64).sum(0)
        if pw is not None:
            tv = tv / np.sqrt((tv ** 2).mean(1, keepdims=True) + eps) * pw.astype(np.float64)
        x = x + tv
    want = x * scale
    h = want if h is None else h.astype(np.float64)
    st = 1 / np.sqrt((h ** 2).mean(1) + eps)
    return want, st, h * st[:, None] * w.astype(np.float64)
