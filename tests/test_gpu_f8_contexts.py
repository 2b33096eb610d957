"""Two contexts, a thread each, with calls of one kernel that need different amounts of shared memory."""
import threading

import numpy as np
import pytest

import p0pc0rn_b200 as p0

from . import f8_ref as R
from .test_gpu_f8 import SLACK, Rows, out_mat

pytestmark = pytest.mark.gpu
M = 160       # more rows than SMs: rows come through shared memory


def call(g, D):
    x = np.random.default_rng(D).standard_normal((M, D)).astype(np.float16)
    w, y = np.ones((1, D), np.float32), out_mat(g, M, D)
    a = {"x": Rows(g, x).arg(), "type": "f16", "w": Rows(g, w).arg(), "y": y.arg(), "M": M, "D": D}
    return p0.bound(p0.normF8, g, a), lambda: R.check_codes(*y.read(), R.norm(x, None, None, w[0], 1e-6, 1.0)[2], SLACK)


def test_norm_in_two_threads():
    made, errors = [], []
    gpus = [p0.Gpu(0) for _ in range(2)]
    try:
        made = [call(g, D) for g, D in zip(gpus, (1536, 9216))]
        start = threading.Barrier(2)

        def work(g, run):
            try:
                start.wait()
                for i in range(20000):
                    run()
                    if i % 500 == 499:
                        g.done()
            except Exception as e:
                errors.append(e)

        threads = [threading.Thread(target=work, args=(g, run)) for g, (run, _) in zip(gpus, made)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors
        for _, check in made:
            check()
    finally:
        for g in gpus:
            g.close()
