"""Beam search over the paged 4-bit cache (p0pc0rn_b200.beam) with a small model of full and sliding layers, against the
same search on the host: the oracle's decode operators per hypothesis, K and V through tests/kv_ref.py's quantiser, its
attention in 64 bits and its selection. Logits agree within the decode parity tolerance, so the host's selections are used
where their runner-up is clear, and the test asserts that it is."""
import numpy as np
import pytest

from oracle import ref
from p0pc0rn_b200 import beam, decode

from . import kv_ref as R
from .test_gpu_decode_step import host_model, upload_model

pytestmark = pytest.mark.gpu

CFG = {"D": 512, "layers": 3, "NH": 4, "NKV": 1, "hd": 128, "FF": 2304, "vocab": 4096, "window": 40, "sinks": 3, "kinds": ["full", "sliding", "full"],
       "embed_scale": 22.627417, "softcap": 30.0, "eps": 1e-6, "beams": 4, "eos": 11}


class Host:
    """hypotheses as lists of quantised (k, v) rows per layer"""

    def __init__(self, cfg, h):
        self.cfg, self.h = cfg, h

    def logits(self, tok, pos, kv):
        c, h = self.cfg, self.h
        D, NH, NKV, hd, FF, V, eps = c["D"], c["NH"], c["NKV"], c["hd"], c["FF"], c["vocab"], c["eps"]
        nq, nqkv = NH * hd, NH * hd + 2 * NKV * hd
        x, st = ref.embed(h["embed"], np.array([tok], np.uint32), D, scale=float(np.float32(c["embed_scale"])), eps=eps, st_off=0)
        for l, W in enumerate(h["layers"]):
            kind = c["kinds"][l]
            qkv, _, _ = ref.gemv(W["qkv"], x, nqkv, D, pro="rms", norm=W["in_norm"], stat_buf=st, stat_off=0)
            Q, kc, vc = ref.qkrope(qkv, 1, nqkv, W["qk_norm"], h["rope"][kind], hd, NH, nkv=NKV, pos=pos, eps=eps, qw=0, kw=hd, npairs=hd // 2, kv_row=0,
                                   kv_len=1, KC=np.zeros(NKV * hd, np.uint16), VC=np.zeros(NKV * hd, np.uint16))
            rows = [R.stands_for(*R.quantise(np.asarray(ref.h2f(a), np.float32).reshape(NKV, hd // 32, 32))).reshape(NKV, hd) for a in (kc, vc)]
            kv[l].append(rows)
            k, v = (np.stack([r[i][0] for r in kv[l]]) for i in (0, 1))
            see = R.visible(pos, pos + 1, c["window"] if kind == "sliding" else 0, c["sinks"])
            s = Q.reshape(NH, hd).astype(np.float64) @ k[see].T
            p = np.exp(s - s.max(-1, keepdims=True))
            ao = ((p / p.sum(-1, keepdims=True)) @ v[see]).astype(np.float32).reshape(-1)
            t, _, ns = ref.gemv(W["o"], ao, D, nq, kPer=decode.KP)
            ref.normadd(t, ns, D, W["post_attn"], 0, x, st, 0, D, 1, eps=eps, scale=1.0)
            mb, _, _ = ref.gemv(W["gu"], x, FF, D, pro="rms", epi="geglu", norm=W["pre_ff"], stat_buf=st, stat_off=0)
            t, _, ns = ref.gemv(W["down"], mb, D, FF, kPer=decode.KP)
            ref.normadd(t, ns, D, W["post_ff"], 0, x, st, 0, D, 1, eps=eps, scale=1.0)
        mx = np.zeros(V // 64 * 2 + 2, np.float32)
        mx[V // 64 * 2] = st[0]
        out, _, _ = ref.gemv(h["embed"], x, V, D, pro="rms", epi="softcap", norm=h["final_norm"], stat_off=V // 64 * 2, mx=mx, cap=c["softcap"])
        return out


def rope_table(npos, npairs, seed):
    ang = ref.randn(npos * npairs, seed, 2.0).astype(np.float64)
    rp = np.zeros(2 * npos * npairs, np.float32)
    rp[0::2], rp[1::2] = np.cos(ang), np.sin(ang)
    return rp


def test_beam_search(g):
    c, M, npos = CFG, CFG["beams"], 160
    h = host_model(c, 900)
    h["rope"] = {k: rope_table(npos, c["hd"] // 2, 77 + i) for i, k in enumerate(("full", "sliding"))}
    prompt = [(7 * i * i + 13) % c["vocab"] for i in range(60)]       # the hypotheses fork inside a page and grow into the next
    steps = 9
    host = Host(c, h)
    kv = [[] for _ in h["layers"]]
    for pos, tok in enumerate(prompt):
        x = host.logits(tok, pos, kv)
    # the host's search
    logits = np.full((M, c["vocab"]), -np.inf, np.float32)
    logits[0] = x
    score, fin = np.array([0.0] + [-np.inf] * (M - 1), np.float32), np.zeros(M, np.uint32)
    hyps = [kv] + [None] * (M - 1)
    hist, margins = [], []
    for t in range(steps + 1):
        parent, token, score2, fin2 = R.beam(logits, score, 1, M, c["eos"], fin)
        with np.errstate(all="ignore"):
            allc = np.concatenate([[score[b]] if fin[b] else score[b] + (logits[b] - np.logaddexp.reduce(logits[b].astype(np.float64))) for b in range(M)])
        top = np.sort(allc[np.isfinite(allc)])[::-1][:M + 1]
        margins.append(float((top[:-1] - top[1:]).min()))
        hist.append((parent, token))
        score, fin = score2, fin2
        if t == steps:
            break
        hyps = [[list(layer) for layer in hyps[int(p)]] for p in parent]
        logits = np.stack([host.logits(int(token[i]), len(prompt) + t, hyps[i]) for i in range(M)])
    assert min(margins) > 2e-3, margins                               # no selection hangs on the decode tolerance
    want = []
    for i in range(M):
        seq, at = [], i
        for parent, token in hist[::-1]:
            seq.append(int(token[at]))
            at = int(parent[at])
        want.append(seq[::-1])
    # the device's
    m = upload_model(g, h)
    s = beam.BeamSearch(g, c, m, npos)
    s.prompt(prompt)
    for t in range(steps):
        s.step()
        if t == 4:
            for cache in s.cache.values():
                cache.compact()
    got, sc, f = s.result()
    g.done()
    s.close()
    assert got == want
    assert np.all(np.abs(sc - score) <= 2e-2) and np.array_equal(f, fin)
    # the sliding layers gave back what their window has passed: one row's pages at most reach from the sinks to the end
    ref_counts = g.read(s.cache["sliding"].state[s.cache["sliding"].now]["ref"], 0, s.cache["sliding"].pages * 4, np.uint32)
    assert 0 < (ref_counts > 0).sum() <= 2 * M + 1
