"""The failure path of the in-kernel waits, exercised without a GPU fault: a kernel's bounded mbarrier wait that
nothing completes gives up after a short limit, records its code in the context's error word and returns; p0_done
reports P0_ETIMEOUT (the reference surfaces device failures at done(), engine/core/gpu.js:141-147) and the same
context then runs GEMV calls that match the oracle.
"""
import numpy as np
import pytest

import p0pc0rn_b200 as p0
from p0pc0rn_b200 import _lib as L
from oracle import ref

from .test_gpu_parity import assert_close, nan_buf, wview

pytestmark = pytest.mark.gpu


def _gemv_ok(g, seed):
    N, K = 256, 2048
    b, _ = ref.pack_q4(ref.randn(N * K, seed, 0.02), N, K)
    X = ref.randn(K, seed + 1)
    yb = nan_buf(g, N * 4)
    p0.gemv(g, {"w": wview(g.upload(b), N, K), "x": {"buf": g.upload(X)}, "N": N, "K": K, "y": {"buf": yb}})
    g.done()
    want, _, _ = ref.gemv(b, X, N, K)
    assert_close(g.read(yb, 0, N * 4, np.float32), want)


def test_bounded_wait_gives_up_and_context_stays_usable(g):
    _gemv_ok(g, 500)
    g.wait_selftest(4096)
    with pytest.raises(p0.P0Error) as ei:
        g.done(10000)
    assert ei.value.status == L.P0_ETIMEOUT
    assert "0x7e1" in str(ei.value)
    # the error word was cleared by the report: the next done() is clean, and the kernels still compute
    g.done()
    _gemv_ok(g, 510)
    # twice in a row behaves the same
    g.wait_selftest(1)
    with pytest.raises(p0.P0Error):
        g.done(10000)
    _gemv_ok(g, 520)


def test_wait_selftest_rejects_bad_limits(g):
    for polls in (0, (1 << 20) + 1):
        with pytest.raises(p0.P0Error, match="polls"):
            g.wait_selftest(polls)


@pytest.mark.parametrize("type_", ["f32", "f16"])
@pytest.mark.parametrize("lens,T,nh,D", [([9000, 700, 30], 1, 8, 256), ([40000] * 4, 1, 2, 64), ([3000, 200], 7, 4, 128), ([2000, 900], 5, 4, 512)])
def test_attention_gives_up_and_context_stays_usable(g, type_, lens, T, nh, D, monkeypatch):
    # every wait of kv4Attn for its copies gives up at once, while they are on their way: the call reports it, and the next one is right
    from . import kv_ref as R
    from .test_gpu_kv import kv_args
    from .test_gpu_kv_attn import check, run
    rng = np.random.default_rng(40 + D)
    c = R.Cache(rng, lens, 1, D)
    c.fill_fast(rng)
    n, dt = T * len(lens), np.float32 if type_ == "f32" else np.float16
    q = (rng.standard_normal((n, nh, D)) * (3.0 / D ** 0.5)).astype(dt)
    _, kv = kv_args(g, c)
    qb, o = g.upload(q), g.buffer(q.nbytes)
    a = {"kv": kv, "q": {"buf": qb}, "out": {"buf": o}, "type": type_, "nh": nh, "n": n, "T": T}
    for _ in range(3):
        monkeypatch.setenv("P0MM_KV4_POLLS", "0")
        p0.kv4Attn(g, a)
        with pytest.raises(p0.P0Error, match="0x4a1") as ei:
            g.done(10000)
        assert ei.value.status == L.P0_ETIMEOUT
        monkeypatch.delenv("P0MM_KV4_POLLS")
        check(run(g, c, q, [T] * len(lens), nh, type_), c, q, [T] * len(lens), nh, type_)
