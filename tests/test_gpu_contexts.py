"""Two contexts, a thread each, with calls of one kernel that need different amounts of shared memory: neither is refused, and both compute what
they compute alone."""
import threading

import numpy as np
import pytest

import p0pc0rn_b200 as p0
from oracle import ref

from . import kv_ref as R
from .test_gpu_kv import kv_args
from .test_gpu_parity import wview

pytestmark = pytest.mark.gpu


def gemv(g, N, K):
    b, _ = ref.pack_q4(ref.randn(N * K, N, 0.02), N, K)
    y = g.buffer(N * 4)
    a = {"w": wview(g.upload(b), N, K), "x": {"buf": g.upload(ref.randn(K, 1))}, "N": N, "K": K, "y": {"buf": y}}
    return lambda: p0.gemv(g, a), y


def normadd(g, D, _):
    x, st = g.upload(ref.randn(D, 2)), g.buffer(4)       # the sum of t's sources is zero: x stays what it is
    a = {"t": {"buf": g.upload(np.zeros(D, np.float32))}, "x": {"buf": x}, "st": {"buf": st}, "M": 1, "D": D, "mode": 1}
    return lambda: p0.normadd(g, a), st


def attention(g, seqs, length):
    rng = np.random.default_rng(seqs)
    c = R.Cache(rng, [length] * seqs, 1, 128)
    c.fill_fast(rng)
    _, kv = kv_args(g, c)
    q = rng.standard_normal((seqs, 4, 128)).astype(np.float16)
    o = g.buffer(q.nbytes)
    return p0.bound(p0.kv4Attn, g, {"kv": kv, "q": {"buf": g.upload(q)}, "out": {"buf": o}, "type": "f16", "nh": 4, "n": seqs, "T": 1}), o


@pytest.mark.parametrize("make,one,two", [(gemv, (2048, 512), (2048, 2048)), (gemv, (64, 512), (64, 2048)),
                                          (normadd, (12288, 0), (16384, 0)), (attention, (2, 70), (400, 70))])
def test_two_threads(make, one, two):
    gpus, errors = [p0.Gpu(0) for _ in range(2)], []
    try:
        calls = [make(g, *size) for g, size in zip(gpus, (one, two))]
        alone = []
        for g, (run, out) in zip(gpus, calls):
            run()
            g.done()
            alone.append(g.read(out).tobytes())
        start = threading.Barrier(2)

        def work(g, run):
            try:
                start.wait()
                for i in range(5000):
                    run()
                    if i % 250 == 249:
                        g.done()
            except Exception as e:
                errors.append(e)

        threads = [threading.Thread(target=work, args=(g, run)) for g, (run, _) in zip(gpus, calls)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors
        assert [g.read(out).tobytes() for g, (_, out) in zip(gpus, calls)] == alone
    finally:
        for g in gpus:
            g.close()
