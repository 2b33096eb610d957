"""Beam search with a Gemma-4-style decoder over a paged 4-bit cache: the decode token of p0pc0rn_b200.decode for up to 8
hypotheses at once, on the device from one step to the next.

  step:  kvStep      the rows continue the hypotheses that the last selection chose (pages shared, last ones copied), + 1 token
         embed       the chosen tokens
         per layer   gemvM rms QKV -> qkrope per row -> kv4Put -> kv4Attn -> gemvM O -> normadd -> gemvM rms GeGLU -> gemvM
                     down -> normadd
         head        gemvM rms softcap over the vocabulary
         beamSelect  the best continuations: parent, token, score, finished

Layers of one kind (full, sliding) share a page table; a page holds every layer of the kind. Sliding layers see the last
`window` tokens and the first `sinks`; kvStep gives back the pages that no later token sees. The prompt goes through row 0
alone (the other rows are empty: nothing is stored or seen for them); the first selection then forks it to every row.
Nothing is read back but the chosen (parent, token) pairs at the end, from which the sequences follow, and what the steps
were short of (then, and every LOG steps)."""
import numpy as np

from . import _lib as L
from . import ops
from .decode import KP, model_sizes

PAGE = L.P0_KV_PAGE
LOG = 4096                  # steps whose shortages a cache holds before it looks at them


class PagedCache:
    """the pages of the layers of one kind, and two states (tables, lengths, reference counts) that steps alternate between"""

    def __init__(self, g, rows, layers, nkv, D, pages, max_pages):
        self.g, self.rows, self.layers, self.pages, self.ld = g, rows, layers, pages, max_pages
        self.D, self.nkv, self.part = D, nkv, nkv * 2 * (D // 32) * 1280
        self.pool = g.buffer(pages * layers * self.part, "kv pages")
        none = np.full(rows * max_pages, L.P0_KV_NONE, np.uint32)
        self.state = [{"table": g.upload(none), "len": g.buffer(rows * 4), "ref": g.buffer(pages * 4)} for _ in range(2)]
        self.now, self.moved = 0, g.buffer(16, "moved")
        # what each step was short of, and left free: kept until ran_short() has looked at it
        self.log, self.steps, self.first_short = g.buffer(8 * LOG, "steps"), 0, 0

    def view(self, layer=0):
        s = self.state[self.now]
        return {"pool": {"buf": self.pool, "off": layer * self.part, "stride": self.layers * self.part}, "pages": self.pages,
                "table": {"buf": s["table"], "ld": self.ld}, "len": {"buf": s["len"]}, "rows": self.rows, "D": self.D, "nkv": self.nkv}

    def step(self, **a):
        """kvStep into the other state, which becomes the current one"""
        if self.steps and self.steps % LOG == 0:
            self.ran_short()
        to = self.state[1 - self.now]
        kv = self.view()
        stat = self.g.wrap(self.log.ptr + 8 * (self.steps % LOG), 8, "stat")
        ops.kvStep(self.g, {"kv": kv, "ref": {"buf": self.state[self.now]["ref"]}, "to": {k: {"buf": to[k]} for k in to}, "stat": {"buf": stat}, **a})
        self.g.free(stat)
        self.steps += 1
        self.now = 1 - self.now

    def compact(self):
        """the pages in use into the lowest ones"""
        s, to = self.state[self.now], self.state[1 - self.now]
        ops.kvCompact(self.g, {"kv": self.view(), "ref": {"buf": s["ref"]}, "to": {"table": {"buf": to["table"]}, "ref": {"buf": to["ref"]}},
                               "stat": {"buf": self.moved}})
        self.g.copy(s["len"], 0, to["len"], 0, self.rows * 4)
        self.now = 1 - self.now

    def short(self):
        """pages that the last step was short of (0: none; its state is otherwise the one before it). Waits for the device"""
        return int(self.g.read(self.log, 8 * ((self.steps - 1) % LOG), 4, np.uint32)[0]) if self.steps else 0

    def ran_short(self):
        """pages that a step was short of, however long ago (0: no step was). Waits for the device"""
        if not self.first_short and self.steps:
            logged = self.g.read(self.log, 0, 8 * min(self.steps, LOG), np.uint32)[0::2]   # beyond LOG steps: of some that were looked at before
            self.first_short = int(logged[logged != 0][0]) if logged.any() else 0
        return self.first_short


    def close(self, tables=True):
        """gives back the pages and, with tables, the states (which can be read until then)"""
        for b in [self.pool, self.log, self.moved] + ([b for s in self.state for b in s.values()] if tables else []):
            self.g.free(b)


class BeamSearch:
    """cfg as p0pc0rn_b200.decode's, plus beams (<= 8), eos, sinks (default 0); model m as decode_token's"""

    def __init__(self, g, cfg, m, max_pos, spare_pages=16):
        self.g, self.cfg, self.m, self.max_pos = g, cfg, m, max_pos
        M, D, NH, NKV, hd, FF, V = cfg["beams"], cfg["D"], cfg["NH"], cfg["NKV"], cfg["hd"], cfg["FF"], cfg["vocab"]
        if not 1 <= M <= 8:
            raise ValueError("beams: 1 to 8 (gemvM's rows)")
        mp = -(-max_pos // PAGE)
        self.kinds = [k for k in ("full", "sliding") if k in cfg["kinds"]]
        self.cache = {k: PagedCache(g, M, cfg["kinds"].count(k), NKV, hd, M * mp + spare_pages, mp) for k in self.kinds}
        nq, nqkv = NH * hd, NH * hd + 2 * NKV * hd
        b = {"x": M * D * 4, "st": 64, "qkvp": M * nqkv * 4, "q": M * nq * 4, "k": M * NKV * hd * 2, "v": M * NKV * hd * 2, "ao": M * nq * 4,
             "tpart": max(-(-nq // KP), -(-FF // KP)) * M * D * 4, "mbuf": M * FF * 4, "logits": M * V * 4, "mx": (M * (V // 64) + 1) * 8,
             "parent": M * 4, "token": M * 4, "score": M * 4, "fin": M * 4, "add": M * 4, "hist": 2 * M * 4 * max_pos}
        self.b = {k: g.buffer(n, k) for k, n in b.items()}
        # qkrope binds its buffers from their start: each row's part of the shared ones as a buffer of its own
        part = lambda k, n, i: g.wrap(self.b[k].ptr + i * n, n, k)
        self.rows = [{"s": part("qkvp", nqkv * 4, i), "q": part("q", nq * 4, i), "k": part("k", NKV * hd * 2, i), "v": part("v", NKV * hd * 2, i)}
                     for i in range(M)]
        self.pos, self.chosen = 0, 0
        g.write(self.b["score"], np.array([0.0] + [-np.inf] * (M - 1), np.float32))

    def close(self):
        """gives back the buffers and the caches' pages; the caches' tables, lengths and counts stay until PagedCache.close()"""
        for r in self.rows:
            for w in r.values():
                self.g.free(w)
        self.rows = []
        for b in self.b.values():
            self.g.free(b)
        for c in self.cache.values():
            c.close(tables=False)

    def _layers(self, ids):
        """one token of every row (ids: a device buffer) at position self.pos - 1 of the current caches"""
        g, c, m, b = self.g, self.cfg, self.m, self.b
        M, D, NH, NKV, hd, FF = c["beams"], c["D"], c["NH"], c["NKV"], c["hd"], c["FF"]
        nq, nqkv, eps, sz, pos = NH * hd, NH * hd + 2 * NKV * hd, c.get("eps", 1e-6), model_sizes(c), self.pos - 1
        w = lambda buf, shape: {"buf": buf, "off": 0, "enc": "q4g32a.t64", "rows": shape[0], "cols": shape[1]}
        rms = lambda norm: {"pro": "rms", "stat": {"buf": b["st"], "off": 0, "ld": 1}, "norm": {"buf": norm, "off": 0}}
        buf = lambda k: {"buf": b[k]}
        ops.embed(g, {"w": w(m["embed"], sz["head"]), "ids": {"buf": ids}, "x": buf("x"), "st": {"buf": b["st"], "off": 0}, "K": D, "n": M,
                      "scale": float(np.float32(c["embed_scale"])), "eps": eps})
        seen = {k: 0 for k in self.kinds}
        for l, W in enumerate(m["layers"]):
            kind = c["kinds"][l]
            kv = self.cache[kind].view(seen[kind])
            seen[kind] += 1
            ops.gemvM(g, {"w": w(W["qkv"], sz["qkv"]), "x": buf("x"), "M": M, "N": nqkv, "K": D, "y": buf("qkvp"), **rms(W["in_norm"])})
            for r in self.rows:
                ops.qkrope(g, {"s": {"buf": r["s"], "n": 1, "ld": nqkv}, "norm": {"buf": W["qk_norm"]}, "qw": 0, "kw": hd,
                               "rope": {"buf": m["rope"][kind], "off": 0}, "q": {"buf": r["q"]}, "kc": {"buf": r["k"]}, "vc": {"buf": r["v"]}, "D": hd,
                               "nq": NH, "hasKV": True, "pos": pos, "npairs": c.get("npairs", hd // 2), "kvRow": 0, "nkv": NKV, "kvLen": 1, "eps": eps})
            ops.kv4Put(g, {"kv": kv, "k": buf("k"), "v": buf("v"), "type": "f16", "n": M, "T": 1})
            ops.kv4Attn(g, {"kv": kv, "q": buf("q"), "out": buf("ao"), "type": "f32", "nh": NH, "n": M, "T": 1,
                            "window": c["window"] if kind == "sliding" else 0, "sinks": c.get("sinks", 0)})
            ns = ops.gemvM(g, {"w": w(W["o"], sz["o"]), "x": buf("ao"), "M": M, "N": D, "K": nq, "kPer": KP, "y": buf("tpart")})
            add = lambda ns, norm: ops.normadd(g, {"t": {"buf": b["tpart"], "n": ns, "ld": M * D}, "w": {"buf": norm, "off": 0}, "x": buf("x"),
                                                   "st": {"buf": b["st"], "off": 0}, "D": D, "M": M, "eps": eps, "scale": 1.0})
            add(ns, W["post_attn"])
            ops.gemvM(g, {"w": w(W["gu"], sz["gu"]), "x": buf("x"), "M": M, "N": FF, "K": D, "epi": "geglu", "y": buf("mbuf"), **rms(W["pre_ff"])})
            ns = ops.gemvM(g, {"w": w(W["down"], sz["down"]), "x": buf("mbuf"), "M": M, "N": D, "K": FF, "kPer": KP, "y": buf("tpart")})
            add(ns, W["post_ff"])

    def _select(self):
        g, c, m, b = self.g, self.cfg, self.m, self.b
        M, D, V = c["beams"], c["D"], c["vocab"]
        buf = lambda k: {"buf": b[k]}
        ops.gemvM(g, {"w": {"buf": m["embed"], "off": 0, "enc": "q4g32a.t64", "rows": V, "cols": D}, "x": buf("x"), "M": M, "N": V, "K": D, "pro": "rms",
                      "stat": {"buf": b["st"], "off": 0, "ld": 1}, "norm": {"buf": m["final_norm"], "off": 0}, "epi": "softcap",
                      "cap": c.get("softcap", 30.0), "mx": buf("mx"), "y": buf("logits")})
        ops.beamSelect(g, {"logits": buf("logits"), "score": buf("score"), "fin": buf("fin"), "groups": 1, "beams": M, "V": V, "eos": c["eos"],
                           "parent": buf("parent"), "token": buf("token"), "scoreOut": buf("score"), "finOut": buf("fin")})
        for i, k in enumerate(("parent", "token")):
            g.copy(b[k], 0, b["hist"], (2 * self.chosen + i) * M * 4, M * 4)
        self.chosen += 1

    def _advance(self, **a):
        if self.pos >= self.max_pos:
            raise ValueError("the caches hold %d positions" % self.max_pos)
        for k, cache in self.cache.items():
            cache.step(window=self.cfg["window"] if k == "sliding" else 0, sinks=self.cfg.get("sinks", 0), **a)
        self.pos += 1

    def prompt(self, tokens):
        """the prompt's tokens through row 0, then the first selection. Once: the other rows are empty until then"""
        M = self.cfg["beams"]
        if self.pos:
            raise ValueError("the search has its prompt")
        if not 1 <= len(tokens) <= self.max_pos:
            raise ValueError("a prompt of %d tokens: 1 to %d" % (len(tokens), self.max_pos))
        self.g.write(self.b["add"], np.array([1] + [0] * (M - 1), np.uint32))
        ids = self.g.upload(np.repeat(np.asarray(tokens, np.uint32)[:, None], M, 1))
        one = [self.g.wrap(ids.ptr + 4 * M * i, 4 * M, "ids") for i in range(len(tokens))]
        for w in one:
            self._advance(add={"buf": self.b["add"]})
            self._layers(w)
        self._select()
        for w in one:
            self.g.free(w)
        self.g.free(ids)

    def step(self):
        """one more token for every hypothesis"""
        self._advance(parent={"buf": self.b["parent"]}, add=1)
        self._layers(self.b["token"])
        self._select()

    def result(self):
        """(sequences, best first, without the prompt; scores; finished). A finished hypothesis goes on with eos"""
        M = self.cfg["beams"]
        for c in self.cache.values():
            if c.ran_short():
                raise RuntimeError("the cache is short of %d pages" % c.ran_short())
        h = self.g.read(self.b["hist"], 0, 2 * M * 4 * self.chosen, np.uint32).reshape(self.chosen, 2, M)
        score = self.g.read(self.b["score"], 0, 4 * M, np.float32)
        out = []
        for i in range(M):
            seq, at = [], i
            for t in range(self.chosen - 1, -1, -1):
                if at >= M:
                    break
                seq.append(int(h[t, 1, at]))
                at = int(h[t, 0, at])
            out.append(seq[::-1])
        return out, score, self.g.read(self.b["fin"], 0, 4 * M, np.uint32)
