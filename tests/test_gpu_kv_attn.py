"""kv4Attn on the GPU against softmax attention in 64 bits over the same codes (tests/kv_ref.py): every element within the
bound that kv_ref.attention_bound derives from the roundings of the kernel's arithmetic."""
import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import kv_ref as R
from .test_gpu_kv import kv_args

pytestmark = pytest.mark.gpu


def run(g, c, q, counts, nh, type_, window=0, sinks=0, scale=0.0, lay=(0, 0, 0), out_lay=(0, 0, 0), bufs=None):
    """out [n][nh][D] as the call wrote it; every other element of the output buffer must keep its fill"""
    dt = np.float32 if type_ == "f32" else np.float16
    n = sum(counts)
    bufs, kv = kv_args(g, c, bufs)

    def rows(x, lay):
        ld, ldh, off = lay[0] or nh * c.D, lay[1] or c.D, lay[2]
        at = off + np.arange(n)[:, None, None] * ld + np.arange(nh)[None, :, None] * ldh + np.arange(c.D)
        buf = np.full(at.max() + 1, -77, dt)
        if x is not None:
            buf[at] = x
        return buf, at, {"off": off, "ld": ld, "ldh": ldh}

    (qb, _, qa), (ob, oi, oa) = rows(q, lay), rows(None, out_lay)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    new = {"n": n, "T": counts[0]} if len(set(counts)) == 1 else {"n": n, "cu": {"buf": g.upload(np.concatenate([[9], cu]).astype(np.uint32)), "off": 1}}
    o = g.upload(ob)
    p0.kv4Attn(g, {"kv": kv, "q": {"buf": g.upload(qb), **qa}, "out": {"buf": o, **oa}, "type": type_, "nh": nh, "window": window, "sinks": sinks,
                   "scale": scale, **new})
    g.done()
    got = g.read(o, 0, ob.nbytes, dt)
    keep = np.ones(ob.size, bool)
    keep[oi] = False
    assert np.all(got[keep] == -77)
    return got[oi]


def check(got, c, q, counts, nh, type_, window=0, sinks=0, scale=1.0, ref=R.attention):
    want, spread, size = ref(c, q, counts, nh, window, sinks, scale)
    tol = R.attention_bound(spread, size, want, c.D, int(c.table.shape[1]), type_ == "f16")
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= tol), (float((err / tol).max()), np.unravel_index((err / tol).argmax(), err.shape))
    seen = spread.any(-1)
    assert not got[~seen].any()                                      # rows that see nothing are zeros
    return want


CASES = [
    # lens, new tokens, nh, nkv, D, window, sinks
    ([1], [1], 8, 1, 256, 0, 0),
    ([63, 64, 65, 0, 1000], [1] * 5, 8, 2, 128, 0, 0),               # page borders; an empty sequence
    ([700, 3, 129], [1] * 3, 6, 2, 64, 100, 4),                      # window and sinks, three heads a group
    ([900], [1], 4, 4, 512, 64, 70),                                 # sinks over two pages; no shared heads
    ([600, 128], [1] * 2, 3, 1, 256, 1, 0),                          # a window of one key
    ([500, 40], [5, 5], 8, 2, 256, 0, 0),
    ([300, 8, 5], [8, 8, 8], 8, 1, 128, 40, 2),                      # the last sequence is shorter than its tokens: rows that see nothing
    ([200, 90, 64], [33, 7, 64], 4, 2, 64, 0, 0),                    # ragged
    ([130, 260], [130, 1], 2, 1, 512, 50, 3),
    ([64 * 5], [3], 16, 1, 256, 0, 0),
    ([2000] + [1] * 20, [1] * 21, 2, 2, 64, 0, 0),                   # one long, many short
]


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("lens,counts,nh,nkv,D,window,sinks", CASES)
def test_attn(g, lens, counts, nh, nkv, D, window, sinks, type_):
    rng = np.random.default_rng(D + len(lens))
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    q = (rng.standard_normal((sum(counts), nh, D)) * (3.0 / D ** 0.5)).astype(np.float32 if type_ == "f32" else np.float16)
    got = run(g, c, q, counts, nh, type_, window, sinks)
    check(got, c, q, counts, nh, type_, window, sinks)


# contexts (and tables) long enough that whole pages go to warps
LONG = [
    # lens, nh, nkv, D, window, sinks
    ([9000, 700, 0, 4097, 64, 1], 8, 1, 256, 0, 0),
    ([5000, 12000], 8, 2, 256, 6000, 70),
    ([70, 8000, 3333, 10], 4, 4, 128, 0, 0),
    ([6000, 2500, 7777], 16, 2, 64, 4000, 4),
]


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("lens,nh,nkv,D,window,sinks", LONG)
def test_attn_long(g, lens, nh, nkv, D, window, sinks, type_):
    rng = np.random.default_rng(D + len(lens))
    c = R.Cache(rng, lens, nkv, D, ld=2500)
    c.fill_fast(rng)
    c.table[0, 3], c.table[-1, 0] = c.pages + 1, R.NONE if lens[-1] > 100 else c.table[-1, 0]
    for b, n in enumerate(lens):
        seen = set(np.nonzero(R.visible(n - 1, n, window, sinks))[0].tolist())
        c.poison_unseen(b, seen)
    q = (rng.standard_normal((len(lens), nh, D)) * (3.0 / D ** 0.5)).astype(np.float32 if type_ == "f32" else np.float16)
    got = run(g, c, q, [1] * len(lens), nh, type_, window, sinks)
    want, spread, size = R.attention(c, q, [1] * len(lens), nh, window, sinks)
    tol = R.attention_bound(spread, size, want, D, 200, type_ == "f16")
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= tol), float((err / tol).max())
    assert not got[~spread.any(-1)].any()
    assert np.array_equal(run(g, c, q, [1] * len(lens), nh, type_, window, sinks).view(np.uint8), got.view(np.uint8))


PROMPTS = [
    # lens, new tokens, nh, nkv, D, window, sinks, scale
    ([1900], [700], 8, 1, 256, 0, 0, 0.0),                           # several key tiles a run, parts of units joined
    ([900, 64, 1300], [900, 64, 40], 8, 1, 256, 0, 0, 0.0),          # from the first token on; units of one tile; an odd page
    ([1500, 700], [500, 300], 4, 1, 256, 200, 70, -0.7),             # window, sinks over two pages, a negative scale
    ([1300, 500, 260], [640, 100, 260], 8, 2, 128, 0, 0, 0.3),
    ([2000, 300], [600, 300], 6, 2, 128, 300, 4, 0.0),
    ([1100, 900], [700, 64], 16, 4, 64, 0, 0, 0.0),
    ([100, 20, 640], [130, 30, 100], 8, 1, 64, 90, 1, 2.0),          # sequences shorter than their tokens: rows that see nothing
    ([1500, 64, 700], [400, 64, 40], 8, 1, 512, 0, 0, 0.0),          # 512 dims: the output in two parts
    ([1300, 30], [300, 60], 4, 2, 512, 250, 70, -0.5),
]


@pytest.mark.parametrize("lens,counts,nh,nkv,D,window,sinks,scale", PROMPTS)
def test_prompt(g, lens, counts, nh, nkv, D, window, sinks, scale):
    rng = np.random.default_rng(D + counts[0])
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    q = (rng.standard_normal((sum(counts), nh, D)) * (3.0 / D ** 0.5)).astype(np.float16)
    got = run(g, c, q, counts, nh, "f16", window, sinks, scale)
    check(got, c, q, counts, nh, "f16", window, sinks, float(np.float32(scale or 1.0)), ref=R.attention_prompt)


@pytest.mark.parametrize("D,nh,nkv,lay,out_lay,scale", [
    (64, 8, 1, (8 * 72 + 8, 72, 16), (8 * 72, 72, 8), 0.4),          # rows apart, 16 bytes at a time
    (128, 6, 2, (6 * 136, 136, 8), (0, 0, 0), -0.3),                 # three heads a group: no box of 128 rows
    (256, 4, 2, (4 * 257 + 3, 257, 5), (4 * 259 + 1, 259, 3), -0.2), # odd offsets and strides, a negative scale
    (512, 4, 1, (4 * 513, 513, 1), (0, 0, 2), 0.0),
    (64, 256, 1, (0, 0, 0), (0, 0, 0), 0.0),                         # more heads a group than a block has rows
    (128, 2, 2, (128, 128 * 330, 0), (128, 128 * 330, 0), 0.0),      # head-major rows
])
def test_prompt_strides(g, D, nh, nkv, lay, out_lay, scale):
    rng = np.random.default_rng(17 + D)
    lens, counts = ([700, 300, 80], [200, 30, 100]) if nh < 256 else ([300, 70], [5, 2])
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    q = (rng.standard_normal((sum(counts), nh, D)) * (3.0 / D ** 0.5)).astype(np.float16)
    got = run(g, c, q, counts, nh, "f16", 90, 3, scale, lay=lay, out_lay=out_lay)
    check(got, c, q, counts, nh, "f16", 90, 3, float(np.float32(scale or 1.0)), ref=R.attention_prompt)
    again = run(g, c, q, counts, nh, "f16", 90, 3, scale, lay=lay, out_lay=out_lay)
    assert np.array_equal(again.view(np.uint16), got.view(np.uint16))


def test_prompt_units_in_a_row_d512(g):
    # several whole units after one another in every run, where the output of one stands in the place of the next one's q
    rng = np.random.default_rng(31)
    lens, counts, nh = [300, 270, 256, 290] * 3, [256, 200, 256, 100] * 3, 16
    c = R.Cache(rng, lens, nh, 512)
    c.fill_fast(rng)
    q = (rng.standard_normal((sum(counts), nh, 512)) * (3.0 / 512 ** 0.5)).astype(np.float16)
    got = run(g, c, q, counts, nh, "f16")
    check(got, c, q, counts, nh, "f16", ref=R.attention_prompt)
    for _ in range(20):
        assert np.array_equal(run(g, c, q, counts, nh, "f16").view(np.uint16), got.view(np.uint16))


@pytest.mark.parametrize("D,nh,nkv", [(64, 16, 8), (128, 16, 4), (256, 8, 4)])
def test_prompt_same_bits(g, D, nh, nkv):
    # many tiles and units a run: what either CTA of a pair copied is there when the pair's products read it, each time
    rng = np.random.default_rng(32 + D)
    lens, counts = [1100, 700, 900, 1000], [300, 520, 410, 256]
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    q = (rng.standard_normal((sum(counts), nh, D)) * (3.0 / D ** 0.5)).astype(np.float16)
    got = run(g, c, q, counts, nh, "f16")
    check(got, c, q, counts, nh, "f16", ref=R.attention_prompt)
    for _ in range(20):
        assert np.array_equal(run(g, c, q, counts, nh, "f16").view(np.uint16), got.view(np.uint16))


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("T", [1, 400])
def test_attn_growing_scores(g, D, T):
    # every later page holds larger scores, by more than 2^8 in P: what was summed before has to follow the maximum
    rng = np.random.default_rng(15)
    c = R.Cache(rng, [900], 1, D)
    c.fill_fast(rng)
    for j in range(c.ld):
        if c.table[0, j] < c.pages:
            rec = c.pool[c.table[0, j], :c.part].reshape(-1, 1280)
            rec[:, 1024:] = np.tile(np.array([0.0, 0.02 * j], np.float16).view(np.uint8), 64)   # k = 0.02 j in every dim
    q = (np.ones((T, 2, D)) * (600.0 / D) + rng.standard_normal((T, 2, D)) * 0.01).astype(np.float16)
    check(run(g, c, q, [T], 2, "f16"), c, q, [T], 2, "f16", ref=R.attention_prompt)
    if T == 1:
        check(run(g, c, q.astype(np.float32), [T], 2, "f32"), c, q, [T], 2, "f32", ref=R.attention_prompt)


@pytest.mark.parametrize("type_,lay,out_lay", [("f32", (0, 0, 3), (901, 129, 1)), ("f16", (1153, 131, 7), (0, 0, 0)), ("f16", (128, 128 * 21, 0), (128, 128 * 21, 8))])
def test_attn_strides_layers_scale(g, type_, lay, out_lay):
    # odd offsets and strides, head-major rows, the last layer of a page, a scale; the other layers hold NaN
    rng = np.random.default_rng(8)
    lens, counts, nh, nkv, D = [150, 400, 77], [7, 7, 7], 4, 2, 128
    part = nkv * 2 * D // 32 * 1280
    c = R.Cache(rng, lens, nkv, D, stride=3 * part, off=2 * part)
    c.pool[:] = 0xFF
    c.fill_fast(rng)
    q = rng.standard_normal((21, nh, D)).astype(np.float32 if type_ == "f32" else np.float16)
    got = run(g, c, q, counts, nh, type_, scale=0.11, lay=lay, out_lay=out_lay)
    check(got, c, q, counts, nh, type_, scale=float(np.float32(0.11)))


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("T,window,sinks", [(1, 0, 0), (1, 70, 5), (6, 70, 5), (90, 70, 66)])
def test_attn_ignores_what_nobody_sees(g, type_, T, window, sinks):
    # NaN scales and infinite minima in every slot outside what some row of the call sees, and pages that are not there
    rng = np.random.default_rng(9)
    lens, nh, nkv, D = [333, 200], 4, 1, 128
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    for b, n in enumerate(lens):
        seen = set()
        for i in range(T):
            seen |= set(np.nonzero(R.visible(n - T + i, n, window, sinks))[0].tolist())
        c.poison_unseen(b, seen)
    c.table[0, -1] = c.pages + 9
    q = (rng.standard_normal((2 * T, nh, D)) * 0.3).astype(np.float32 if type_ == "f32" else np.float16)
    check(run(g, c, q, [T, T], nh, type_, window, sinks), c, q, [T, T], nh, type_, window, sinks)


@pytest.mark.parametrize("type_,T", [("f32", 1), ("f16", 3), ("f16", 100)])
def test_attn_missing_pages(g, type_, T):
    # a page that was given back, one beyond the pool, and a sequence without any: their keys are not there
    rng = np.random.default_rng(10)
    lens, nh, nkv, D = [400, 300, 130], 2, 1, 64
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    c.table[0, 2], c.table[1, 0], c.table[2, :] = R.NONE, c.pages, R.NONE
    q = rng.standard_normal((3 * T, nh, D)).astype(np.float32 if type_ == "f32" else np.float16) * np.float16(0.4)
    check(run(g, c, q, [T] * 3, nh, type_), c, q, [T] * 3, nh, type_)


def test_attn_long_table_offsets(g):
    # a length beyond the table counts as the table's; pool offsets past 32 bits: pages 400 MB apart
    rng = np.random.default_rng(11)
    c = R.Cache(rng, [64 * 15], 1, 64, spare=0, ld=15)
    c.fill_fast(rng)
    q = rng.standard_normal((1, 2, 64)).astype(np.float32)
    stride = 400 << 20
    pool = g.buffer((c.pages - 1) * stride + c.stride, "pool")
    for p in range(c.pages):
        g.write(pool, c.pool[p], p * stride)
    lens = np.array([1 << 31], np.uint32)
    bufs = {"pool": pool, "table": g.upload(c.table), "len": g.upload(lens)}
    _, kv = kv_args(g, c, bufs)
    kv["pool"]["stride"] = stride
    o = g.buffer(2 * 64 * 4)
    p0.kv4Attn(g, {"kv": kv, "q": {"buf": g.upload(q)}, "out": {"buf": o}, "type": "f32", "nh": 2, "n": 1, "T": 1})
    got = g.read(o, 0, 512, np.float32).reshape(1, 2, 64)
    check(got, c, q, [1], 2, "f32")
    g.free(pool)


def test_attn_same_bits_and_other_stream(g):
    # the same call gives the same bits, and so does it on another stream of the caller's
    import torch
    rng = np.random.default_rng(12)
    lens, nh, D = [3000, 10, 700], 8, 256
    c = R.Cache(rng, lens, 1, D)
    c.fill_fast(rng)
    q = (rng.standard_normal((3, nh, D)) * 0.2).astype(np.float32)
    first = run(g, c, q, [1] * 3, nh, "f32")
    for _ in range(3):
        assert np.array_equal(run(g, c, q, [1] * 3, nh, "f32").view(np.uint32), first.view(np.uint32))
    s = torch.cuda.Stream()
    g.done()
    g.set_stream(s.cuda_stream)
    try:
        assert np.array_equal(run(g, c, q, [1] * 3, nh, "f32").view(np.uint32), first.view(np.uint32))
    finally:
        g.done()
        g.set_stream(0)


def test_attn_cu_out_of_order(g):
    # a cu that decreases or passes n gives no tokens out of range: rows of no sequence keep what they held
    rng = np.random.default_rng(13)
    c = R.Cache(rng, [100, 50, 70], 1, 64)
    c.fill_fast(rng)
    q = rng.standard_normal((10, 2, 64)).astype(np.float32) * 0.4
    bufs, kv = kv_args(g, c)
    o = g.upload(np.full(10 * 128, -77, np.float32))
    p0.kv4Attn(g, {"kv": kv, "q": {"buf": g.upload(q)}, "out": {"buf": o}, "type": "f32", "nh": 2, "n": 10,
                   "cu": {"buf": g.upload(np.array([4, 2, 4000000000, 4000000000], np.uint32))}})
    got = g.read(o, 0, 10 * 512, np.float32).reshape(10, 2, 64)
    assert np.all(got[:2] == -77)
    c2 = R.Cache(rng, [50], 1, 64)
    c2.table, c2.pool, c2.pages, c2.ld = c.table[1:2], c.pool, c.pages, c.ld
    check(got[2:], c2, q[2:], [8], 2, "f32")                         # sequence 1 has tokens 2 .. 9, the others none


@pytest.mark.parametrize("D,T,nh", [(64, 1, 8), (256, 1, 8), (128, 6, 4), (256, 8, 8), (512, 4, 4)])
@pytest.mark.parametrize("size", [2.0 ** 17, 3e9, 2.0 ** 100, 1e-6, 3e-12, 2.0 ** -105])
def test_attn_f32_queries_of_any_size(g, D, T, nh, size):
    # q far outside f16's range, and the scale that makes ordinary scores of it; rows of sizes of their own, a row of zeros, one
    # element that stands out (its keys' dim is small)
    rng = np.random.default_rng(34 + D)
    c = R.Cache(rng, [700, 90], 1, D)
    c.fill_fast(rng)
    scale = float(np.float32(1.0 / size))
    q = rng.standard_normal((2 * T, nh, D)) * (3.0 / D ** 0.5)
    q[0, 1] *= 2.0 ** -9
    q[0, 2] = 0.0
    q[-1, 3] *= 8.0
    q[-1, 0, 5] = 40.0
    q = (q * size).astype(np.float32)
    check(run(g, c, q, [T, T], nh, "f32", scale=scale), c, q, [T, T], nh, "f32", scale=scale, ref=R.attention_prompt)


def test_attn_f32_queries_beyond_f16(g):
    # a query beyond 65504 in a dim where every key is 0: its scores are the other dims'
    rng = np.random.default_rng(35)
    c = R.Cache(rng, [200], 1, 64)
    c.fill_fast(rng)
    for page in c.table[0, :4]:
        rec = c.pool[page, :1280]
        rec[0:1024:16] &= 0xF0                                       # K's dim 0: code 0
        sm = np.ascontiguousarray(rec[1024:]).view(np.float16).reshape(64, 2)
        sm[:, 1] = 0.0                                               # and minimum 0
        rec[1024:] = sm.view(np.uint8).reshape(-1)
    q = (rng.standard_normal((1, 4, 64)) * 0.3).astype(np.float32)
    q[0, :, 0] = [65520.0, -7e4, 1e9, 6e4]
    got = run(g, c, q, [1], 4, "f32")
    assert np.isfinite(got).all()
    want, spread, size = R.attention(c, q, [1], 4)
    # the low part of the other dims is held to 2^-25 at a row's largest of 2^14 or more: 2^-39 of it
    lost = np.abs(q).max(-1) * 2.0 ** -38 * 64 * 4.0
    tol = R.attention_bound(spread, size, want, 64, 5, False) + 2 * lost[..., None] * spread
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("lens,counts,nh,nkv,D,lay", [
    ([900, 130, 40], [1, 1, 1], 8, 1, 256, (0, 0, 0)),
    ([700, 300], [40, 9], 4, 2, 128, (4 * 130, 130, 3)),
    ([700, 300, 90], [300, 200, 90], 8, 2, 256, (0, 0, 0)),
    ([700, 300, 90], [300, 200, 90], 8, 4, 512, (0, 0, 0)),          # prompts of 512 dims: the output in two parts
    ([700, 300], [300, 200], 4, 4, 512, (4 * 513, 513, 1)),
    ([700, 300], [300, 200], 2, 2, 512, (512, 512 * 501, 0)),
])
def test_attn_in_place(g, type_, lens, counts, nh, nkv, D, lay):
    # out = q gives what a call with an output of its own gives
    rng = np.random.default_rng(37)
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    n = sum(counts)
    q = (rng.standard_normal((n, nh, D)) * (3.0 / D ** 0.5)).astype(np.float32 if type_ == "f32" else np.float16)
    want = run(g, c, q, counts, nh, type_, 200, 3, lay=lay, out_lay=lay)
    check(want, c, q, counts, nh, type_, 200, 3, ref=R.attention_prompt)
    ld, ldh, off = lay[0] or nh * D, lay[1] or D, lay[2]
    at = off + np.arange(n)[:, None, None] * ld + np.arange(nh)[None, :, None] * ldh + np.arange(D)
    host = np.full(at.max() + 1, -77, q.dtype)
    host[at] = q
    _, kv = kv_args(g, c)
    x = g.upload(host)
    rows = {"buf": x, "off": off, "ld": ld, "ldh": ldh}
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    new = {"T": counts[0]} if len(set(counts)) == 1 else {"cu": {"buf": g.upload(cu)}}
    p0.kv4Attn(g, {"kv": kv, "q": rows, "out": rows, "type": type_, "nh": nh, "n": n, "window": 200, "sinks": 3, **new})
    g.done()
    got = g.read(x, 0, host.nbytes, q.dtype)
    assert np.array_equal(got[at].view(np.uint8), want.view(np.uint8))
    got[at] = -77
    assert np.all(got == -77)


def test_prompt_without_memory_for_wide_pages(g):
    # a device too full for the pages as f16 (2 GB here): the call is served by the form for few rows (two launches), and by the
    # other one (three) once there is room
    import torch
    rng = np.random.default_rng(38)
    c = R.Cache(rng, [400, 130], 1, 256, ld=16384)
    c.fill_fast(rng)
    counts = [80, 80]
    q = (rng.standard_normal((160, 2, 256)) * (3.0 / 256 ** 0.5)).astype(np.float16)
    own = p0.Gpu(0)
    try:
        check(run(own, c, q, counts, 2, "f16", 100, 3), c, q, counts, 2, "f16", 100, 3, ref=R.attention_prompt)
        full = own.buffer(torch.cuda.mem_get_info()[0] - (1 << 30), "what fills the device")
        for launches in (2, 2, 3):
            if launches == 3:
                own.free(full)
            before = own.stats["dispatches"]
            got = run(own, c, q, counts, 2, "f16")
            assert own.stats["dispatches"] - before == launches
            check(got, c, q, counts, 2, "f16", ref=R.attention_prompt)
    finally:
        own.close()


def test_prompt_window_in_a_wide_table(g):
    # what the window lets a call see bounds the pages held as f16, not what the table could hold
    rng = np.random.default_rng(39)
    lens, counts = [3000, 500, 64, 900], [300, 200, 64, 1]
    c = R.Cache(rng, lens, 1, 64, ld=70000)
    c.fill_fast(rng)
    q = (rng.standard_normal((sum(counts), 2, 64)) * (3.0 / 8)).astype(np.float16)
    before = g.stats["dispatches"]
    got = run(g, c, q, counts, 2, "f16", 130, 70)
    assert g.stats["dispatches"] - before == 3
    want, spread, size = R.attention_prompt(c, q, counts, 2, 130, 70)
    assert np.all(np.abs(got - want) <= R.attention_bound(spread, size, want, 64, 50, True))


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("T,nh,nkv", [(7, 8, 1), (9, 12, 2), (3, 7, 1)])
def test_attn_fragments_at_once(g, type_, D, T, nh, nkv):
    # 56, 54 and 21 rows a KV head: up to four fragments of rows on each dequantised page, the last ones not full
    rng = np.random.default_rng(41 + D)
    lens = [900, 64, 333, 7]
    c = R.Cache(rng, lens, nkv, D)
    c.fill_fast(rng)
    q = (rng.standard_normal((4 * T, nh, D)) * (3.0 / D ** 0.5)).astype(np.float32 if type_ == "f32" else np.float16)
    for window, sinks in ((0, 0), (100, 66)):
        check(run(g, c, q, [T] * 4, nh, type_, window, sinks), c, q, [T] * 4, nh, type_, window, sinks, ref=R.attention_prompt)


@pytest.mark.parametrize("gap", [10.0, 13.3, 17.4])
@pytest.mark.parametrize("type_,D,R_,T,nh,at", [("f32", 64, 1, 1, 1, 0), ("f32", 64, 1024, 1, 1, 0), ("f32", 256, 600, 1, 8, 40000), ("f32", 128, 200, 8, 4, 0),
                                                ("f32", 512, 300, 2, 4, 7), ("f16", 64, 1024, 1, 2, 0), ("f16", 256, 200, 8, 4, 0), ("f16", 64, 127, 64, 1, 0),
                                                ("f16", 256, 60, 70, 1, 200), ("f16", 512, 30, 130, 1, 30)])
def test_attn_long_flat_tail(g, type_, D, R_, T, nh, at, gap):
    # one key holds the maximum, 65499 others of one score lie `gap` below it and weigh e^-gap each: up to 3 of its 1 together.
    # Each exp(-gap) has to reach O as it reaches the sum, though f16 by itself ends at 2^-24. The sequences are one and the same,
    # so many that a run holds most of one's pages (each run has a maximum of its own)
    n = 65500
    rng = np.random.default_rng(36)
    c = R.Cache(rng, [n], 1, D, ld=1024)
    G = D // 32
    rec = np.zeros((c.pages, 2, G, 1280), np.uint8)                  # codes 0: a row's value is its minimum
    mn = np.zeros((c.pages, 2, G, 64, 2), np.float16)
    mn[..., 0] = 1.0
    mn[:, 1, :, :, 1] = 1.0 + 0.25 * rng.random((c.pages, G, 64))
    top = c.table[0, at // 64], slice(None), slice(None), at % 64, 1
    mn[top] = np.array([[1.0], [-1.0]])
    rec[..., 1024:] = mn.reshape(c.pages, 2, G, 128).view(np.uint8)
    c.pool[:] = rec.reshape(c.pages, -1)
    dt = np.float32 if type_ == "f32" else np.float16
    q = np.full((T, nh, D), gap / D, dt)
    want, spread, size = R.attention_prompt(c, q, [T], nh)
    # attention_bound's sums and scores; what P loses: 2^-22 of it as two halves, and 2^-40 (f32, f16) or 2^-32 (prompts) a key
    e = (D / 16 + D / 32 + 4) * 2.0 ** -23 * size[..., None]
    tol = (2 * e + 2.0 ** -20 + (c.ld + 8) * 2.0 ** -23) * spread + n * 2.0 ** (-32 if T * nh >= 64 else -40) * 2
    if type_ == "f16":
        tol += 2.0 ** -11 * spread + 2.0 ** -11 * np.abs(want)
    c.table, c.lens = np.repeat(c.table, R_, 0), np.full(R_, n, np.uint32)
    got = run(g, c, np.tile(q, (R_, 1, 1)), [T] * R_, nh, type_).reshape(R_, T, nh, D)
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("type_,R_,n", [("f32", 1024, 40), ("f16", 1024, 40), ("f16", 200, 13000)])
def test_attn_cu_up_and_down(g, type_, R_, n):
    # 0, n, 0, n, ...: half of the sequences claim every token. More than the call has: nothing is computed (few rows, and prompts)
    rng = np.random.default_rng(33)
    c = R.Cache(rng, [70], 1, 64)
    c.fill_fast(rng)
    c.table, c.lens = np.repeat(c.table, R_, 0), np.full(R_, 70, np.uint32)
    _, kv = kv_args(g, c)
    dt = np.float32 if type_ == "f32" else np.float16
    q, o = g.upload(np.ones(n * 64, dt)), g.upload(np.full(n * 64, -77, dt))
    cu = np.tile(np.array([0, n], np.uint32), R_)[:R_ + 1]
    p0.kv4Attn(g, {"kv": kv, "q": {"buf": q}, "out": {"buf": o}, "type": type_, "nh": 1, "n": n, "cu": {"buf": g.upload(cu)}})
    g.done()
    assert np.all(g.read(o, 0, n * 64 * dt().itemsize, dt) == -77)
    cu = np.minimum(np.arange(R_ + 1) * (n // R_ + 1), n).astype(np.uint32)
    p0.kv4Attn(g, {"kv": kv, "q": {"buf": q}, "out": {"buf": o}, "type": type_, "nh": 1, "n": n, "cu": {"buf": g.upload(cu)}})
    g.done()
    assert not np.any(g.read(o, 0, n * 64 * dt().itemsize, dt) == -77)   # every token of a sequence is written


def test_attn_refusals(g):
    rng = np.random.default_rng(14)
    c = R.Cache(rng, [100, 70], 2, 64)
    _, kv = kv_args(g, c)
    x = g.buffer(2 * 4 * 64 * 4)
    a = {"kv": kv, "q": {"buf": x}, "out": {"buf": x}, "type": "f32", "nh": 4, "n": 2, "T": 1}
    for msg, change in (("3 query heads over 2 KV heads", {"nh": 3}), ("0 query heads", {"nh": 0}), ("D 32 must be", {"kv": {**kv, "D": 32}}),
                        ("q range", {"q": {"buf": x, "off": 1}}), ("out range", {"out": {"buf": x, "ld": 257}}), ("type bf16", {"type": "bf16"}),
                        ("cu range", {"cu": {"buf": g.buffer(4), "off": 2}}), ("n 4 is not", {"n": 4}), ("1025 sequences", {"kv": {**kv, "rows": 1025}})):
        with pytest.raises(p0.P0Error, match=msg):
            p0.kv4Attn(g, {**a, **change})
    p0.kv4Attn(g, {**a, "n": 0})                                     # no tokens: nothing to do
    g.done()
