"""The paged 4-bit cache's writer, reader and page operators (kv4Put, kv4Get, kvStep, kvCompact) on the GPU against the
host statements in tests/kv_ref.py. Everything here is exact: codes, tables, counts and copied bytes are compared whole."""
import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import kv_ref as R

pytestmark = pytest.mark.gpu


def kv_args(g, c, bufs=None):
    bufs = bufs or {"pool": g.upload(c.pool), "table": g.upload(c.table), "len": g.upload(c.lens)}
    return bufs, {"pool": {"buf": bufs["pool"], "off": c.off, "stride": c.stride}, "pages": c.pages, "table": {"buf": bufs["table"], "ld": c.ld},
                  "len": {"buf": bufs["len"]}, "rows": len(c.lens), "D": c.D, "nkv": c.nkv}


def rows_of(rng, n, heads, D, type_, ld=0, ldh=0, off=0, big=False):
    """(host buffer, [n][heads][D] view of it as f32, the rows' arguments)"""
    ldh = ldh or D
    ld = ld or heads * D
    buf = np.zeros(off + (n - 1) * ld + (heads - 1) * ldh + D if n else off + 1, np.float32 if type_ == "f32" else np.float16)
    at = off + np.arange(n)[:, None, None] * ld + np.arange(heads)[None, :, None] * ldh + np.arange(D)
    x = rng.standard_normal((n, heads, D)).astype(buf.dtype)
    if big:
        x = x * (rng.random((n, heads, 1)) < 0.5) * 3.0
        x[0, 0, :7] = [np.nan, np.inf, -np.inf, 6e4, -6.1e4, 1e-7, -0.0]
    buf[at] = x
    return buf, at, {"off": off, "ld": ld, "ldh": ldh}


CASES = [
    # lens, new tokens, nkv, D, type, row layout (ld, ldh, off)
    ([1], [1], 1, 64, "f32", (0, 0, 0)),
    ([64, 65, 0, 700], [1, 1, 1, 1], 2, 256, "f16", (0, 0, 0)),
    ([130, 40, 5], [70, 40, 9], 1, 128, "f32", (0, 0, 0)),           # the last two sequences are shorter than, or as long as, their tokens
    ([63, 200], [63, 3], 3, 512, "f16", (0, 0, 0)),
    ([90, 33], [17, 33], 2, 128, "f32", (301, 129, 5)),              # odd strides: element by element
    ([90, 33], [17, 33], 2, 64, "f16", (150, 77, 3)),
    ([90, 33], [17, 33], 2, 64, "f16", (96, 1000, 8)),               # heads outside tokens
]


@pytest.mark.parametrize("lens,counts,nkv,D,type_,lay", CASES)
def test_put_get(g, lens, counts, nkv, D, type_, lay):
    rng = np.random.default_rng(len(lens) * 1000 + D)
    part = nkv * 2 * D // 32 * 1280
    c = R.Cache(rng, lens, nkv, D, stride=3 * part, off=part)        # the middle one of three layers
    c.pool[:] = 0xAB
    n = sum(counts)
    ld, ldh, off = lay
    if ldh > ld > 0:
        ldh = n * ld
    (kb, ki, ka), (vb, vi, va) = (rows_of(rng, n, nkv, D, type_, ld, ldh, off, big) for big in (True, False))
    bufs, kv = kv_args(g, c)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    rows = {"n": n, "T": counts[0]} if len(set(counts)) == 1 else {"n": n, "cu": {"buf": g.upload(cu)}}
    p0.kv4Put(g, {"kv": kv, "k": {"buf": g.upload(kb), **ka}, "v": {"buf": g.upload(vb), **va}, "type": type_, **rows})
    place = []
    for b, T in enumerate(counts):
        for i in range(T):
            pos = int(lens[b]) - T + i
            place.append((b, pos))
            if pos >= 0:
                for h in range(nkv):
                    c.write(b, pos, 0, h, kb[ki[cu[b] + i, h]])
                    c.write(b, pos, 1, h, vb[vi[cu[b] + i, h]])
    assert np.array_equal(g.read(bufs["pool"], 0, c.pool.nbytes).reshape(c.pool.shape), c.pool)
    for gt, dt in (("f16", np.float16), ("f32", np.float32)):
        outs = [g.upload(np.full(x.size, 77, dt)) for x in (kb, vb)]
        p0.kv4Get(g, {"kv": kv, "k": {"buf": outs[0], **ka}, "v": {"buf": outs[1], **va}, "type": gt, **rows})
        for i, (o, at, host) in enumerate(zip(outs, (ki, vi), (kb, vb))):
            got = g.read(o, 0, host.size * dt().itemsize, dt)
            want = np.full(host.size, 77, dt)
            for t, (b, pos) in enumerate(place):
                for h in range(nkv):
                    want[at[t, h]] = c.values(b, i, h, int(lens[b]))[0][pos] if pos >= 0 else 0
            assert np.array_equal(got, want)


def test_put_page_equals_packed_weights_layout(g):
    # a full page of one head is a [64][D] q4g32a.t64 tensor: the weights' own dequantiser reads it
    rng = np.random.default_rng(3)
    c = R.Cache(rng, [64], 1, 256)
    bufs, kv = kv_args(g, c)
    x = rng.standard_normal((64, 256)).astype(np.float32)
    xb = g.upload(x)
    p0.kv4Put(g, {"kv": kv, "k": {"buf": xb}, "v": {"buf": xb}, "type": "f32", "n": 64, "T": 64})
    page = int(c.table[0, 0])
    out = g.buffer(64 * 256 * 2)
    p0.dequant_f16(g, {"buf": bufs["pool"], "off": page * c.stride, "enc": "q4g32a.t64", "rows": 64, "cols": 256}, out)
    q, s, mn = R.quantise(x.reshape(64, 8, 32))
    want = R.stands_for(q, s, mn).reshape(64, 256)
    assert np.array_equal(g.read(out, 0, 64 * 256 * 2, np.float16).reshape(64, 256).astype(np.float64), want)


def test_put_halves_and_scales(g):
    # quotients on, and next to, halves: groups whose scale is exactly 2^k, values at (n + 1/2) * 2^k and their neighbours
    rng = np.random.default_rng(6)
    c = R.Cache(rng, [640], 1, 64)
    x = np.zeros((640, 2, 32), np.float32)
    for t in range(640):
        k = np.float32(2.0 ** rng.integers(-12, 8))
        v = (rng.integers(0, 16, (2, 32)) + rng.choice([0.0, 0.5, 0.25], (2, 32))).astype(np.float32) * k
        v = np.nextafter(v, np.where(rng.random((2, 32)) < 0.5, np.float32(-np.inf), np.float32(np.inf)), dtype=np.float32) if t % 2 else v
        v[:, 0], v[:, 1] = 0, 15 * k
        x[t] = np.clip(v, 0, 15 * k) + (rng.integers(-8, 8) * k if t % 3 == 0 else 0)
    x = x.reshape(640, 64)
    bufs, kv = kv_args(g, c)
    xb = g.upload(x)
    p0.kv4Put(g, {"kv": kv, "k": {"buf": xb}, "v": {"buf": xb}, "type": "f32", "n": 640, "T": 640})
    for t in range(640):
        c.write(0, t, 0, 0, x[t])
        c.write(0, t, 1, 0, x[t])
    assert np.array_equal(g.read(bufs["pool"], 0, c.pool.nbytes).reshape(c.pool.shape), c.pool)


def test_put_drops_tokens_without_a_page(g):
    rng = np.random.default_rng(4)
    c = R.Cache(rng, [100, 70], 1, 64)
    c.table[0, 1] = R.NONE
    c.table[1, 0] = c.pages + 5                                      # no such page
    before = c.pool.copy()
    bufs, kv = kv_args(g, c)
    x = rng.standard_normal((2 * 70, 64)).astype(np.float32)
    xb, o = g.upload(x), [g.upload(np.full(140 * 64, 9, np.float32)) for _ in range(2)]
    p0.kv4Put(g, {"kv": kv, "k": {"buf": xb}, "v": {"buf": xb}, "type": "f32", "n": 140, "T": 70})
    for b, n in ((0, 100), (1, 70)):
        for i in range(70):
            for s in (0, 1):
                c.write(b, n - 70 + i, s, 0, x[b * 70 + i])
    assert not np.array_equal(before, c.pool)
    assert np.array_equal(g.read(bufs["pool"], 0, c.pool.nbytes).reshape(c.pool.shape), c.pool)
    p0.kv4Get(g, {"kv": kv, "k": {"buf": o[0]}, "v": {"buf": o[1]}, "type": "f32", "n": 140, "T": 70})
    k = g.read(o[0], 0, 140 * 256, np.float32).reshape(2, 70, 64)
    assert not k[0, 64 - 30:].any() and k[0, :34].any() and not k[1, :64].any() and k[1, 64:].any()


# ------------------------------------------------------------------------------------------------ pages
def batch(rng, lens, shares, ld, spare):
    """groups of rows that share their first pages: (table, len, ref, pages)"""
    rows = []
    at = 0
    for n, (beams, shared) in zip(lens, shares):
        np_ = -(-n // R.PAGE)
        shared = min(shared, max(0, np_ - 1))
        head = list(range(at, at + shared))
        at += shared
        for _ in range(beams):
            rows.append((n, head + list(range(at, at + np_ - shared))))
            at += np_ - shared
    pages = at + spare
    ids = rng.permutation(pages)
    table, ref = np.full((len(rows), ld), R.NONE, np.uint32), np.zeros(pages, np.uint32)
    for i, (_, t) in enumerate(rows):
        for j, p in enumerate(t):
            table[i, j] = ids[p]
            ref[ids[p]] += 1
    return table, np.array([n for n, _ in rows], np.uint32), ref, pages


def run_step(g, table, lens, ref, pages, stride, pool, **a):
    up = g.upload
    b = {k: up(v) for k, v in (("table", table), ("len", lens), ("ref", ref), ("pool", pool))}
    to = {k: up(np.full_like(v, 0x5a5a)) for k, v in (("table", table), ("len", lens), ("ref", ref))}
    stat = g.buffer(16)
    kv = {"pool": {"buf": b["pool"], "stride": stride}, "pages": pages, "table": {"buf": b["table"], "ld": table.shape[1]}, "len": {"buf": b["len"]},
          "rows": table.shape[0]}
    args = {"kv": kv, "ref": {"buf": b["ref"]}, "to": {k: {"buf": v} for k, v in to.items()}, "stat": {"buf": stat}}
    for k in ("parent", "add"):
        if a.get(k) is not None and not np.isscalar(a[k]):
            a[k] = {"buf": up(np.asarray(a[k], np.uint32))}
    p0.kvStep(g, {**args, **{k: v for k, v in a.items() if v is not None}})
    return (g.read(to["table"], 0, table.nbytes, np.uint32).reshape(table.shape), g.read(to["len"], 0, lens.nbytes, np.uint32),
            g.read(to["ref"], 0, ref.nbytes, np.uint32), tuple(g.read(stat, 0, 8, np.uint32).tolist()),
            g.read(b["pool"], 0, pool.nbytes).reshape(pool.shape))


@pytest.mark.parametrize("seed,lens,shares,parent,add,window,sinks,spare", [
    (0, [130], [(4, 1)], [0, 0, 0, 2], 1, 0, 0, 9),                    # a fork: two copies of one tail
    (1, [128, 1], [(3, 2), (2, 0)], [1, 1, 2, 3, 3], 1, 0, 0, 9),      # a full last page needs no copy, one of a single token does
    (2, [700, 64, 0], [(4, 9), (4, 1), (1, 0)], None, [1, 0, 64, 65, 2, 0, 200, 1, 3], 0, 0, 40),
    (3, [700, 300], [(3, 8), (3, 3)], [2, 2, 0, R.NONE, 77, 5], 1, 200, 4, 20),   # freed rows; the window gives pages back
    (4, [700, 300], [(3, 8), (3, 3)], [0, 0, 0, 3, 3, 3], 1, 1, 70, 20),          # a window of one token, sinks over two pages
    (5, [129], [(2, 0)], [R.NONE, R.NONE], 5, 0, 0, 1),                # everything freed
    (6, [100], [(5, 0)], [0, 0, 0, 0, 0], 1, 0, 0, 0),                 # its own old rows' pages make the room
    (7, [64 * 6], [(2, 5)], [0, 1], 1, 0, 0, 1),                       # one page short
    (8, [64 * 6], [(2, 5)], [0, 0], 129, 0, 0, 40),                    # longer than the table
])
def test_step(g, seed, lens, shares, parent, add, window, sinks, spare):
    rng = np.random.default_rng(seed)
    ld = max(-(-n // 64) for n in lens) + (2 if seed != 2 else 4)
    table, ln, ref, pages = batch(rng, lens, shares, ld, spare)
    stride = 48 if seed % 2 else 16 * 1024 + 16
    pool = rng.integers(0, 256, (pages, stride), dtype=np.uint8)
    want = R.step(table, ln, ref, pages, parent, add, window, sinks)
    expect = pool.copy()
    for s, d in want[4]:
        expect[d] = pool[s]
    got = run_step(g, table, ln, ref, pages, stride, pool, parent=parent, add=add, window=window, sinks=sinks)
    assert got[3] == want[3]
    if seed in (7, 8):
        assert want[3][0] != 0
    for a, b in zip(got[:3], want[:3]):
        assert np.array_equal(a, b)
    assert np.array_equal(got[4], expect)


def test_step_many_random(g):
    # one batch taken through random steps: every state against the host's, counts against the table at the end
    rng = np.random.default_rng(20)
    table, ln, ref, pages = batch(rng, [900, 333, 64], [(16, 10), (16, 4), (8, 0)], 40, 6000)
    pool = rng.integers(0, 256, (pages, 32), dtype=np.uint8)
    for step in range(12):
        parent = rng.integers(0, 40, 40)
        parent[rng.random(40) < 0.1] = R.NONE
        add = rng.integers(0, 90, 40)
        window, sinks = ((0, 0), (150, 4), (64, 100))[step % 3]
        want = R.step(table, ln, ref, pages, parent, add, window, sinks)
        got = run_step(g, table, ln, ref, pages, 32, pool, parent=parent, add=add, window=window, sinks=sinks)
        assert got[3] == want[3]
        for s, d in want[4]:
            pool[d] = pool[s]
        for a, b in zip(got[:3], want[:3]):
            assert np.array_equal(a, b)
        assert np.array_equal(got[4], pool)
        table, ln, ref = want[:3]
    used = table[table < pages]
    assert np.array_equal(np.bincount(used, minlength=pages), ref)


def lowered_step(table, lens, ref, pages, *a):
    """R.step of a state whose tables may hold pages beyond the lengths: those are references, which the step ends"""
    clean, counts = table.copy(), ref.astype(np.int64)
    for b, n in enumerate(lens):
        for j in range(-(-int(n) // R.PAGE), table.shape[1]):
            if clean[b, j] < pages:
                counts[clean[b, j]] -= 1
                clean[b, j] = R.NONE
    got = R.step(clean, lens, counts.astype(np.uint32), pages, *a)
    return got if got[3][0] == 0 else (table, lens, ref, (got[3][0], int((ref == 0).sum())), [])


@pytest.mark.parametrize("spare", [60, 6000])                        # one CTA plans, and a cluster
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_step_after_a_lowered_length(g, spare, window, sinks):
    # rounds of: every row takes up to 200 drafted tokens, keeps some of them, and goes on; rows end and fork now and then. No page
    # is lost: the counts are the table's at every step
    rng = np.random.default_rng(21)
    table, ln, ref, pages = batch(rng, [300, 65], [(3, 2), (3, 0)], 30, spare)
    rows = len(ln)
    pool = rng.integers(0, 256, (pages, 32), dtype=np.uint8)
    for step in range(14):
        parent = np.arange(rows)
        if step % 4 == 3:
            parent = np.where(rng.random(rows) < 0.2, R.NONE, rng.integers(0, rows, rows))
        add = rng.integers(0, 200, rows) if step != 9 else np.full(rows, 64 * 30)   # once more than the tables hold: nothing changes
        want = lowered_step(table, ln, ref, pages, parent, add, window, sinks)
        got = run_step(g, table, ln, ref, pages, 32, pool, parent=parent, add=add, window=window, sinks=sinks)
        assert (want[3][0] != 0) == (step == 9)
        assert got[3] == want[3]
        for s, d in want[4]:
            pool[d] = pool[s]
        for a, b in zip(got[:3], want[:3]):
            assert np.array_equal(a, b)
        assert np.array_equal(got[4], pool)
        before, (table, ln, ref) = ln, want[:3]
        assert np.array_equal(np.bincount(table[table < pages], minlength=pages), ref)
        if step != 9:                                                # the drafts that are not accepted: never below the length before
            keep = rng.integers(0, add + 1)
            ln = np.where(ln >= add, ln - np.minimum(add, ln) + keep, ln).astype(np.uint32)


@pytest.mark.parametrize("seed,pages,live,rows", [(0, 1, 0.0, 1), (1, 1, 1.0, 2), (2, 300, 0.5, 7), (3, 5000, 0.3, 33), (4, 20011, 0.9, 3), (5, 64, 1.0, 4)])
def test_compact(g, seed, pages, live, rows):
    rng = np.random.default_rng(seed)
    ref = (rng.random(pages) < live).astype(np.uint32) * rng.integers(1, 5, pages).astype(np.uint32)
    ids = np.nonzero(ref)[0]
    ld = 50
    table = np.full((rows, ld), R.NONE, np.uint32)
    if len(ids):
        table[:, :40] = rng.choice(ids, (rows, 40))
        table[:, 41] = pages + 7                                     # no such page: kept as it is
    stride = 16 * (1 + 1300 * (seed == 3))
    pool = rng.integers(0, 256, (pages, stride), dtype=np.uint8)
    t, r, stat, moves = R.compact(table, ref, pages)
    b = {k: g.upload(v) for k, v in (("table", table), ("ref", ref), ("pool", pool), ("len", np.zeros(rows, np.uint32)))}
    to = {k: g.upload(np.full_like(v, 0x5a5a)) for k, v in (("table", table), ("ref", ref))}
    sb = g.buffer(16)
    p0.kvCompact(g, {"kv": {"pool": {"buf": b["pool"], "stride": stride}, "pages": pages, "table": {"buf": b["table"], "ld": ld}, "len": {"buf": b["len"]},
                            "rows": rows}, "ref": {"buf": b["ref"]}, "to": {k: {"buf": v} for k, v in to.items()}, "stat": {"buf": sb}})
    expect = pool.copy()
    for s, d in moves:
        expect[d] = pool[s]
    assert tuple(g.read(sb, 0, 8, np.uint32).tolist()) == stat
    assert np.array_equal(g.read(to["table"], 0, table.nbytes, np.uint32).reshape(table.shape), t)
    assert np.array_equal(g.read(to["ref"], 0, ref.nbytes, np.uint32), r)
    assert np.array_equal(g.read(b["pool"], 0, pool.nbytes).reshape(pool.shape), expect)


def test_refusals(g):
    rng = np.random.default_rng(5)
    c = R.Cache(rng, [100, 70], 1, 64)
    bufs, kv = kv_args(g, c)
    x = g.buffer(2 * 64 * 4)
    a = {"kv": kv, "k": {"buf": x}, "v": {"buf": x}, "type": "f32", "n": 2, "T": 1}
    for msg, change in (("D 96 must be", {"kv": {**kv, "D": 96}}), ("n 3 is not T 1 x 2", {"n": 3}), ("T .new tokens per sequence. or cu is missing", {"T": 0}),
                        ("0 sequences", {"kv": {**kv, "rows": 0}}), ("pool range", {"kv": {**kv, "pages": c.pages + 1}}),
                        ("table range", {"kv": {**kv, "rows": 3}}), ("16-byte aligned", {"kv": {**kv, "pool": {"buf": bufs["pool"], "off": 8}, "pages": 1}}),
                        ("below the layer's", {"kv": {**kv, "pool": {"buf": bufs["pool"], "stride": 16}}}), ("k range", {"k": {"buf": x, "ld": 65}}),
                        ("type f64", {"type": "f64"}), ("missing binding v", {"v": {"buf": None}})):
        with pytest.raises(p0.P0Error, match=msg):
            p0.kv4Put(g, {**a, **change})
    ref, stat = g.buffer(c.pages * 4), g.buffer(8)
    to = {"table": {"buf": g.buffer(c.table.nbytes)}, "len": {"buf": g.buffer(8)}, "ref": {"buf": g.buffer(c.pages * 4)}}
    s = {"kv": kv, "ref": {"buf": ref}, "to": to, "stat": {"buf": stat}, "add": 1}
    for msg, change in (("must not lie over", {"to": {**to, "table": kv["table"]}}), ("must not lie over", {"to": {**to, "ref": {"buf": ref}}}),
                        ("page stride is missing", {"kv": {**kv, "pool": {"buf": bufs["pool"]}}}), ("missing binding stat", {"stat": {"buf": None}})):
        with pytest.raises(p0.P0Error, match=msg):
            p0.kvStep(g, {**s, **change})
    with pytest.raises(p0.P0Error, match="must not lie over"):
        p0.kvCompact(g, {"kv": kv, "ref": {"buf": ref}, "to": {"table": to["table"], "ref": {"buf": ref}}, "stat": {"buf": stat}})
    g.done()


def test_refuses_pools_beyond_64_bits(g):
    # (pages - 1) * stride wraps to 0 here: the pool would seem to fit its buffer
    rng = np.random.default_rng(7)
    c = R.Cache(rng, [100], 1, 64)
    bufs, kv = kv_args(g, c)
    huge = {**kv, "pages": (1 << 24) + 1, "pool": {"buf": bufs["pool"], "stride": 1 << 40}}
    x = g.buffer(64 * 4)
    with pytest.raises(p0.P0Error, match="pass 64 bits"):
        p0.kv4Put(g, {"kv": huge, "k": {"buf": x}, "v": {"buf": x}, "type": "f32", "n": 1, "T": 1})
    with pytest.raises(p0.P0Error, match="pass 64 bits"):
        p0.kv4Attn(g, {"kv": huge, "q": {"buf": x}, "out": {"buf": x}, "type": "f32", "nh": 1, "n": 1, "T": 1})
    with pytest.raises(p0.P0Error, match="pool range"):              # the largest that does not wrap is still beyond the buffer
        p0.kv4Put(g, {"kv": {**huge, "pages": 1 << 24}, "k": {"buf": x}, "v": {"buf": x}, "type": "f32", "n": 1, "T": 1})
    g.done()
