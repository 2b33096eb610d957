"""Measured cases of the paged 4-bit cache and beam search operators: kv4Put / kv4Get (K and V rows quantised into pages
of 64 tokens, and read back), kv4Attn (attention over the pages: whole context or a sliding window with a few first
tokens that stay visible; one new token per sequence, a few to verify, or a prompt's), kvStep / kvCompact (fork,
reorder, extend, trim, free and compact the pages of a batch of sequences) and beamSelect.

Where `own` is false `run` computes an operator in elementary torch operations in 32 bits; where it is true it makes the
framework's calls. Lengths and the shapes of the page tables follow from the case alone; page numbers and values from
the seed.

A page holds 64 tokens: per layer and KV head K then V, each as D / 32 records of 1280 bytes (64 rows x 16 bytes of
codes, low nibble first, then 64 x (f16 scale, f16 minimum)). A code q stands for f16(q * scale + minimum).
"""
import math
import random
import weakref

import torch

own = False

DEV = "cuda"
PAGE = 64
NONE = -1            # a table entry without a page (0xffffffff)
HOLD = 60000.0       # K and V values beyond it are held at it


def listed():
    return [
        # one decode step of eight beams of one request on a sliding-window layer with four first tokens kept: small
        # enough that the call's latency is what counts
        _attn("decode_beams_window", "f32", 8, 1, 6000, 8, 1, 256, window=512, sinks=4),
        # a serving batch of ragged contexts on full-attention layers, one slot waiting (empty): the bandwidth case
        _attn("decode_batch_long", "f32", 32, 1, 65500, 8, 1, 256),
        # eight drafted tokens verified at once, wide heads, two KV heads
        _attn("verify_wide_heads", "f32", 4, 8, 8190, 8, 2, 512),
        # a batch of prompts of different lengths on top of earlier context, whole attention
        _attn("prompt_full", "f16", 3, 2048, 5003, 8, 1, 256),
        # the same on a sliding-window layer with narrow heads
        _attn("prompt_window", "f16", 4, 1500, 6001, 16, 4, 128, window=1024, sinks=4),
        # the cache write (and reading back) of one decode step of eight beams, and of a prompt
        _put("put_step", "f16", 8, 1, 700, 1, 256),
        _put("put_prompt", "f32", 2, 4096, 5000, 2, 256),
        # a decode step's reorder of eight beams; of a batch of long contexts, every layer's part in the page
        _step("step_beams", 1, 8, 3011, 4, 1, 128, 200),
        _step("step_batch", 8, 8, 9000, 26, 1, 256, 2300),
        # a cache half of whose pages were given back, made dense
        _step("compact_batch", 3, 8, 6000, 26, 1, 256, 1400, compact=True),
        # beams of a small vocabulary; a batch over the 262144-row head
        _beam("beam_small", 1, 4, 4099),
        _beam("beam_batch", 16, 8, 262144),
    ]


def _attn(name, kind, B, T, ctx, nh, nkv, D, window=0, sinks=0):
    return {"name": name, "op": "attn", "type": kind, "B": B, "T": T, "ctx": ctx, "nh": nh, "nkv": nkv, "D": D, "window": window, "sinks": sinks}


def _put(name, kind, B, T, ctx, nkv, D):
    return {"name": name, "op": "put", "type": kind, "B": B, "T": T, "ctx": ctx, "nkv": nkv, "D": D}


def _step(name, groups, beams, ctx, layers, nkv, D, pages, window=0, compact=False):
    return {"name": name, "op": "compact" if compact else "step", "groups": groups, "beams": beams, "ctx": ctx, "layers": layers, "nkv": nkv,
            "D": D, "pages": pages, "window": window, "sinks": 4 if window else 0}


def _beam(name, groups, beams, V):
    return {"name": name, "op": "beam", "groups": groups, "beams": beams, "V": V}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        top = {k: max(top.get(k, 0), w[k]) for k in w}
    while True:
        kind = rng.choice(["decode", "decode", "verify", "prompt", "prompt", "put", "step", "compact", "beam", "beam"])
        D = rng.choice([64, 128, 256, 512])
        nh, nkv = rng.choice([(8, 1), (8, 2), (8, 4), (4, 4), (16, 2), (6, 2)])
        window, sinks = rng.choice([(0, 0), (0, 0), (rng.randint(40, 2048), rng.choice([0, 1, 4, 70]))])
        if kind == "decode":
            c = _attn("", rng.choice(["f32", "f32", "f16"]), _log(rng, 1, 48), 1, _log(rng, 1, 65536), nh, nkv, D, window, sinks)
        elif kind == "verify":
            c = _attn("", rng.choice(["f32", "f16"]), _log(rng, 1, 8), rng.randint(2, 8), _log(rng, 8, 32768), nh, nkv, D, window, sinks)
        elif kind == "prompt":
            T = _log(rng, 32, 2048)
            c = _attn("", "f16", _log(rng, 1, 6), T, T + _log(rng, 1, 6000), nh, nkv, D, window, sinks)
        elif kind == "put":
            T = _log(rng, 1, 4096)
            c = _put("", rng.choice(["f32", "f16"]), _log(rng, 1, 8), T, T + rng.randint(0, 3000), nkv, D)
        elif kind in ("step", "compact"):
            c = _step("", _log(rng, 1, 16), rng.randint(1, 8), _log(rng, 20, 9000), _log(rng, 1, 26), nkv, D, 0, window, kind == "compact")
            c["pages"] = _page_need(c) + rng.randint(8, 400)
        else:
            c = _beam("", _log(rng, 1, 16), rng.randint(1, 16), rng.choice([_log(rng, 1000, 262144), 262144]))
        del c["name"]
        w = work(c)
        if all(w[k] <= top[k] for k in w) and _state_bytes(c) < 6e9:
            return c


# ------------------------------------------------------------------------------------------------ shapes of a case
def _rng(c):
    return random.Random(",".join("%s=%s" % (k, c[k]) for k in sorted(c) if k != "name"))


def _lens(c):
    """(length, new tokens) of every sequence: the first at the full sizes; one of eight or more is an empty slot"""
    r, got = _rng(c), []
    for b in range(c["B"]):
        f = 1.0 if b == 0 else r.uniform(0.3, 1.0)
        T = c["T"] if c["T"] <= 8 or b == 0 else max(1, int(c["T"] * r.uniform(0.4, 1.0)))
        got.append((max(T, int(c["ctx"] * f)), T))
    if c["B"] >= 8 and c["op"] == "attn":
        got[-1] = (0, 1)
    return got


def _visible(c, n, T):
    """visible (new token, key) pairs of one sequence, and the keys that some new token sees"""
    W, S, pairs = c.get("window", 0), c.get("sinks", 0), 0
    lo = n - T
    for p in range(max(lo, 0), n):
        if not W or p - W < 0:
            pairs += p + 1
        else:
            pairs += W + min(S, p - W + 1)
    first = 0 if not W else max(0, lo - W + 1)
    return pairs, (n - first) + min(S, first)


def _page_bytes(c):
    return c.get("layers", 1) * c["nkv"] * 2 * (c["D"] // 32) * 1280


def _beam_shapes(c):
    """per group (length, pages that all its beams share)"""
    r = _rng(c)
    return [(max(2, int(c["ctx"] * (1.0 if g == 0 else r.uniform(0.5, 1.0)))), r.uniform(0.7, 0.98)) for g in range(c["groups"])]


def _beam_pages(c, n, share):
    """(pages, pages shared by the group) of a beam's row"""
    np_ = -(-n // PAGE)
    return np_, min(np_ - 1, int(np_ * share))


def _page_need(c):
    need = 0
    for n, share in _beam_shapes(c):
        np_, shared = _beam_pages(c, n, share)
        need += shared + (np_ - shared) * c["beams"]
    return need + c["groups"] * c["beams"] * 2


def _parents(c):
    """a step's parents: most beams continue, some twice; now and then a finished request frees its rows"""
    r, got = _rng(c), []
    for g in range(c["groups"]):
        free = c["groups"] > 3 and g % 7 == 5
        for i in range(c["beams"]):
            got.append(NONE if free else g * c["beams"] + min(c["beams"] - 1, int(c["beams"] * r.random() ** 1.5)))
    return got


def _state_bytes(c):
    if c["op"] in ("step", "compact"):
        return c["pages"] * _page_bytes(c) * 3
    if c["op"] == "beam":
        return c["groups"] * c["beams"] * c["V"] * 24
    most = max(n for n, T in _lens(c))
    t = max(T for n, T in _lens(c))
    scores = c["B"] * c["nh"] * t * most * 12 if c["op"] == "attn" else 0
    return scores / 4 + c["B"] * most * c["nkv"] * c["D"] * 8


def work(c):
    if c["op"] == "attn":
        e, flops, size = 4 if c["type"] == "f32" else 2, 0, 0
        for n, T in _lens(c):
            pairs, keys = _visible(c, n, T)
            flops += 4 * c["D"] * c["nh"] * pairs
            size += keys * c["nkv"] * c["D"] * 2 * 0.625 + 2 * T * c["nh"] * c["D"] * e + -(-n // PAGE) * 4
        return {"bytes": size, "flops": flops}
    if c["op"] == "put":
        n = sum(T for _, T in _lens(c)) * c["nkv"] * c["D"] * 2
        return {"bytes": n * ((4 if c["type"] == "f32" else 2) + 0.625 * 2 + 2), "flops": n * 6}
    if c["op"] == "beam":
        n = c["groups"] * c["beams"]
        return {"bytes": 4 * n * c["V"] + n * 28, "flops": 4 * n * c["V"]}
    rows = c["groups"] * c["beams"]
    table = sum(-(-n // PAGE) * c["beams"] for n, _ in _beam_shapes(c)) * 4
    if c["op"] == "step":
        seen, copies = set(), 0
        for i, p in enumerate(_parents(c)):
            if p >= 0:
                copies += p in seen and _beam_shapes(c)[p // c["beams"]][0] % PAGE != 0
                seen.add(p)
        return {"bytes": copies * _page_bytes(c) * 2 + 2 * table + rows * 12 + c["pages"] * 8, "flops": rows}
    live = _page_need(c) - rows * 2
    moves = live * max(0, c["pages"] - live) // c["pages"]          # live pages beyond the first `live`, on average
    return {"bytes": moves * _page_bytes(c) * 2 + 2 * table + c["pages"] * 8, "flops": rows}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _cache(c, seed, pages):
    """one layer's pool [pages, nkv, 2, D / 32, 1280] of bell-shaped codes, values within about +-1.5"""
    g, G = _gen(seed), c["D"] // 32
    pool = torch.empty(pages, c["nkv"], 2, G, 1280, dtype=torch.uint8, device=DEV)
    nib = lambda: torch.randint(0, 8, (pages, c["nkv"], 2, G, 1024), generator=g, device=DEV, dtype=torch.uint8) + \
        torch.randint(0, 9, (pages, c["nkv"], 2, G, 1024), generator=g, device=DEV, dtype=torch.uint8)
    pool[..., :1024] = nib() | (nib() << 4)
    s = (0.2 * (0.75 + 0.5 * torch.rand(pages, c["nkv"], 2, G, 64, generator=g, device=DEV))).half()
    mn = (-7.5 * s.float() + 0.1 * torch.randn(pages, c["nkv"], 2, G, 64, generator=g, device=DEV)).half()
    pool[..., 1024:] = torch.stack([s, mn], -1).reshape(pages, c["nkv"], 2, G, 128).view(torch.uint8)
    return pool


class State(dict):
    """what a user's program has in hand; with the framework's own calls, its buffer registrations go when it goes"""


def prepare(c, seed):
    s = State(case=c)
    g = _gen(seed + 7)
    if c["op"] in ("attn", "put"):
        lens = _lens(c)
        B, ld = c["B"], max(1, max(-(-n // PAGE) for n, _ in lens)) + 1
        used = sum(-(-n // PAGE) for n, _ in lens)
        pages = used + 3
        ids = torch.randperm(pages, generator=g, device=DEV).int()
        table = torch.full((B, ld), NONE, dtype=torch.int32, device=DEV)
        at = 0
        for b, (n, _) in enumerate(lens):
            k = -(-n // PAGE)
            table[b, :k] = ids[at:at + k]
            at += k
        n = sum(T for _, T in lens)
        cu = [0]
        for _, T in lens:
            cu.append(cu[-1] + T)
        s.update(table=table, len=torch.tensor([n for n, _ in lens], dtype=torch.int32, device=DEV), cu=torch.tensor(cu, dtype=torch.int32, device=DEV),
                 n=n, pages=pages, most=max(n for n, _ in lens), tmax=max(T for _, T in lens), same=len({T for _, T in lens}) == 1)
        dt = torch.float32 if c["type"] == "f32" else torch.float16
        if c["op"] == "attn":
            s["pool"] = _cache(c, seed, pages)
            s["q"] = (torch.randn(n, c["nh"], c["D"], generator=g, device=DEV) * (3.0 / math.sqrt(c["D"]))).to(dt)
            s["out"] = torch.empty(n, c["nh"], c["D"], dtype=dt, device=DEV)
        else:
            s["pool"] = torch.zeros(pages, c["nkv"], 2, c["D"] // 32, 1280, dtype=torch.uint8, device=DEV)
            for x in ("k", "v"):
                s[x] = torch.randn(n, c["nkv"], c["D"], generator=g, device=DEV).to(dt)
                s[x + "_out"] = torch.empty(n, c["nkv"], c["D"], dtype=torch.float16, device=DEV)
    elif c["op"] == "beam":
        R = c["groups"] * c["beams"]
        z = torch.randn(R, c["V"], generator=g, device=DEV) * 4.0
        s["logits"] = 30.0 * torch.tanh(z / 30.0)                    # the head's soft cap
        s["score"] = -20.0 * torch.rand(R, generator=g, device=DEV)
        fin = torch.rand(R, generator=g, device=DEV) < 0.05
        if c["groups"] > 1:
            s["score"][R - c["beams"] + 1:] = -math.inf              # a request's first step: one live beam
            fin[R - c["beams"]:] = False
        s["fin"] = fin.int()
        for x in ("parent", "token", "fin_out"):
            s[x] = torch.empty(R, dtype=torch.int32, device=DEV)
        s["score_out"] = torch.empty(R, dtype=torch.float32, device=DEV)
    else:
        shapes, rows = _beam_shapes(c), c["groups"] * c["beams"]
        ld = max(-(-n // PAGE) for n, _ in shapes) + 2
        ids = torch.randperm(c["pages"], generator=g, device=DEV).int()
        table = torch.full((rows, ld), NONE, dtype=torch.int32, device=DEV)
        at = 0
        for i, (n, share) in enumerate(shapes):
            np_, shared = _beam_pages(c, n, share)
            r0 = i * c["beams"]
            table[r0:r0 + c["beams"], :shared] = ids[at:at + shared]
            at += shared
            k = (np_ - shared) * c["beams"]
            table[r0:r0 + c["beams"], shared:np_] = ids[at:at + k].view(c["beams"], np_ - shared)
            at += k
        ref = torch.zeros(c["pages"], dtype=torch.int32, device=DEV)
        flat = table[table >= 0].long()
        ref.index_add_(0, flat, torch.ones_like(flat, dtype=torch.int32))
        lens = torch.tensor([n for n, _ in shapes], dtype=torch.int32, device=DEV).repeat_interleave(c["beams"])
        # one page more than the cache has: where the plain form copies what need not be copied
        pool = torch.randint(0, 256, (c["pages"] + 1, _page_bytes(c)), generator=g, device=DEV, dtype=torch.uint8)
        s.update(table=table, len=lens, ref=ref, pool=pool, parent=torch.tensor(_parents(c), dtype=torch.int32, device=DEV),
                 add=torch.ones(rows, dtype=torch.int32, device=DEV), table_out=torch.empty_like(table), len_out=torch.empty_like(lens),
                 ref_out=torch.empty_like(ref), stat=torch.empty(2, dtype=torch.int32, device=DEV))
    if own:
        _bind(s)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
_GPU = []


def _bind(s):
    """registers the tensors with the framework's context and keeps the calls' checked arguments, as a serving loop does"""
    import p0pc0rn_b200 as p0
    if not _GPU:
        _GPU.append(p0.Gpu(0))
        _GPU[0].set_stream(1)                                        # the stream that torch's work is on
    g, c = _GPU[0], s["case"]
    bufs = {k: g.wrap(v.data_ptr(), v.numel() * v.element_size(), k) for k, v in s.items() if isinstance(v, torch.Tensor)}
    weakref.finalize(s, lambda: [g.free(b) for b in bufs.values()])
    b = lambda k: {"buf": bufs[k]}
    if c["op"] in ("attn", "put"):
        kv = {"pool": b("pool"), "pages": s["pages"], "table": {"buf": bufs["table"], "ld": s["table"].shape[1]}, "len": b("len"), "rows": c["B"],
              "D": c["D"], "nkv": c["nkv"]}
        rows = {"n": s["n"], "T": s["tmax"]} if s["same"] else {"n": s["n"], "cu": b("cu")}
        if c["op"] == "attn":
            s["calls"] = [p0.bound(p0.kv4Attn, g, {"kv": kv, "q": b("q"), "out": b("out"), "type": c["type"], "nh": c["nh"], "window": c["window"],
                                                   "sinks": c["sinks"], **rows})]
        else:
            s["calls"] = [p0.bound(p0.kv4Put, g, {"kv": kv, "k": b("k"), "v": b("v"), "type": c["type"], **rows}),
                          p0.bound(p0.kv4Get, g, {"kv": kv, "k": b("k_out"), "v": b("v_out"), "type": "f16", **rows})]
    elif c["op"] == "beam":
        s["calls"] = [p0.bound(p0.beamSelect, g, {"logits": b("logits"), "score": b("score"), "fin": b("fin"), "groups": c["groups"],
                                                  "beams": c["beams"], "V": c["V"], "eos": 1, "parent": b("parent"), "token": b("token"),
                                                  "scoreOut": b("score_out"), "finOut": b("fin_out")})]
    else:
        kv = {"pool": {"buf": bufs["pool"], "stride": _page_bytes(c)}, "pages": c["pages"], "table": {"buf": bufs["table"], "ld": s["table"].shape[1]},
              "len": b("len"), "rows": c["groups"] * c["beams"]}
        a = {"kv": kv, "ref": b("ref"), "to": {"table": b("table_out"), "len": b("len_out"), "ref": b("ref_out")}, "stat": b("stat")}
        if c["op"] == "step":
            s["calls"] = [p0.bound(p0.kvStep, g, {**a, "parent": b("parent"), "add": b("add"), "window": c["window"], "sinks": c["sinks"]})]
        else:
            s["calls"] = [p0.bound(p0.kvCompact, g, a)]


def run(s):
    op = s["case"]["op"]
    if own:
        for call in s["calls"]:
            call()
    else:
        {"attn": _plain_attn, "put": _plain_put, "beam": _plain_beam, "step": _plain_step, "compact": _plain_compact}[op](s)
    if op == "attn":
        return {"out": s["out"]}
    if op == "put":
        return {"k": s["k_out"], "v": s["v_out"]}
    if op == "beam":
        return {"parent": s["parent"], "token": s["token"], "score": s["score_out"], "fin": s["fin_out"]}
    if op == "step":
        return {"table": s["table_out"], "len": s["len_out"], "ref": s["ref_out"], "stat": s["stat"], "pool": s["pool"]}
    return {"table": s["table_out"], "ref": s["ref_out"], "stat": s["stat"], "pool": s["pool"]}


# ------------------------------------------------------------------------------------------------ the plain forms
def _values(rec, dt):
    """records [..., G, 1280] -> the values of their codes [..., 64, G * 32] in dt, each rounded to f16"""
    codes = rec[..., :1024].unflatten(-1, (64, 16))
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(dt)
    sm = rec[..., 1024:].contiguous().view(torch.float16).unflatten(-1, (64, 2)).to(dt)
    x = (q * sm[..., :1] + sm[..., 1:]).half().to(dt)
    return x.transpose(-3, -2).flatten(-2)


def _pairs(s, b):
    """new token t of sequence b: its position [T] and its row of q, for sequences padded to the longest"""
    t = torch.arange(s["tmax"], device=DEV)
    T = (s["cu"][1:] - s["cu"][:-1])[b]
    live = t < T[:, None]
    pos = s["len"][b, None] - T[:, None] + t
    return live, pos, torch.where(live, s["cu"][:-1][b, None] + t, 0).long()


def _plain_attn(s):
    c = s["case"]
    B, nkv, D, hpg = c["B"], c["nkv"], c["D"], c["nh"] // c["nkv"]
    np_ = max(1, -(-s["most"] // PAGE))
    live, pos, row = _pairs(s, torch.arange(B, device=DEV))
    kv = _values(s["pool"][s["table"][:, :np_].clamp(min=0).long()], torch.float32)          # [B, np, nkv, 2, 64, D]
    k, v = (kv[:, :, :, i].transpose(1, 2).flatten(2, 3) for i in (0, 1))                      # [B, nkv, keys, D]
    del kv
    j = torch.arange(np_ * PAGE, device=DEV)
    see = live[..., None] & (j <= pos[..., None])
    if c["window"]:
        see &= (j > pos[..., None] - c["window"]) | (j < c["sinks"])
    v = torch.where((j < s["len"][:, None])[:, None, :, None], v, 0.0)
    q = s["q"].float()[row].view(B, s["tmax"], nkv, hpg, D).permute(0, 2, 1, 3, 4).reshape(B, nkv, s["tmax"] * hpg, D)
    x = (q @ k.transpose(-1, -2)).view(B, nkv, s["tmax"], hpg, -1)
    x = torch.where(see[:, None, :, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    o = (p.view(B, nkv, s["tmax"] * hpg, -1) @ v).view(B, nkv, s["tmax"], hpg, D).permute(0, 2, 1, 3, 4).reshape(B * s["tmax"], c["nh"], D)
    # every live row is read from its place among the padded ones
    at = torch.searchsorted(s["cu"], torch.arange(s["n"], device=DEV, dtype=torch.int32), right=True) - 1
    s["out"].copy_(o[at * s["tmax"] + torch.arange(s["n"], device=DEV) - s["cu"][at]])


def _places(s):
    """(page, slot) of every new row"""
    i = torch.arange(s["n"], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["cu"], i, right=True) - 1
    pos = s["len"][b] - s["cu"][b + 1] + i
    return s["table"][b, (pos // PAGE).long()].long(), (pos % PAGE).long()


def _plain_put(s):
    c = s["case"]
    page, slot = _places(s)
    codes, sms = s["pool"][..., :1024].unflatten(-1, (64, 16)), s["pool"][..., 1024:].unflatten(-1, (64, 4))
    fifteen = torch.full((), 15.0, device=DEV)
    for i, x in enumerate((s["k"], s["v"])):
        x = x.float().nan_to_num(0.0, HOLD, -HOLD).clamp(-HOLD, HOLD).unflatten(-1, (c["D"] // 32, 32))
        mn, mx = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        low = mn.half()
        sc = ((mx - low.float()) / fifteen).half()
        sc = torch.where(sc == 0, torch.ones_like(sc), sc)
        q = ((x - low.float()) / sc.float()).round().clamp(0, 15).to(torch.uint8).unflatten(-1, (16, 2))
        codes[page, :, i, :, slot] = q[..., 0] | (q[..., 1] << 4)
        sms[page, :, i, :, slot] = torch.cat([sc, low], -1).view(torch.uint8)
    q = codes[page, :, :, :, slot]                                                            # [n, nkv, 2, G, 16]
    q = torch.stack([q & 15, q >> 4], -1).flatten(-2).float()
    sm = sms[page, :, :, :, slot].contiguous().view(torch.float16).float()
    x = (q * sm[..., :1] + sm[..., 1:]).half().flatten(-2)
    s["k_out"].copy_(x[:, :, 0])
    s["v_out"].copy_(x[:, :, 1])


def _plain_beam(s):
    c = s["case"]
    k, V = c["beams"], c["V"]
    x = s["logits"]
    m = x.amax(-1, keepdim=True)
    lse = m + (x - m).exp().sum(-1, keepdim=True).log()
    cand = s["score"][:, None] + (x - lse)
    fin = s["fin"][:, None] != 0
    v = torch.arange(V, device=DEV)
    cand = torch.where(fin, torch.where(v == 1, s["score"][:, None], -math.inf), cand)
    cand = torch.where(torch.isnan(cand), -math.inf, cand).view(c["groups"], k * V) + 0.0
    # one whole number per candidate: the value's order above the lowest index first
    bits = cand.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    key = (order << 32) + (k * V - 1 - torch.arange(k * V, device=DEV))
    at = k * V - 1 - (key.topk(k, -1).values & 0xffffffff)
    score = cand.gather(-1, at)
    none = score == -math.inf
    parent = at // V + torch.arange(c["groups"], device=DEV)[:, None] * k
    token = at % V
    s["fin_out"].copy_(torch.where(none, 0, ((token == 1) | (s["fin"][parent] != 0)).int()).flatten())
    s["parent"].copy_(torch.where(none, NONE, parent).flatten())
    s["token"].copy_(torch.where(none, NONE, token).flatten())
    s["score_out"].copy_(score.flatten())


def _plain_step(s):
    c = s["case"]
    table, n, ref, pages = s["table"], s["len"], s["ref"], c["pages"]
    rows, ld = table.shape
    j = torch.arange(ld, device=DEV)
    held = lambda t: (t >= 0) & (t < pages)
    count = lambda r, t, m, sign: r.index_add_(0, torch.where(m, t, 0).flatten().long(), sign * m.flatten().int())
    old = (j < ((n + 63) // PAGE)[:, None]) & held(table)
    now = count(ref.clone(), table, old, -1)
    valid = (s["parent"] >= 0) & (s["parent"] < rows)
    par = torch.where(valid, s["parent"], 0).long()
    lp = torch.where(valid, n[par], 0)
    row = table[par]
    keep = (j < ((lp + 63) // PAGE)[:, None]) & held(row)
    if c["window"]:
        keep &= ~((j * PAGE + 63 <= (lp - c["window"])[:, None]) & (j * PAGE >= c["sinks"]))
    same = (s["parent"][:, None] == s["parent"][None]) & torch.ones(rows, rows, dtype=torch.bool, device=DEV).tril(-1)
    tail = keep & (valid & same.any(-1) & (lp % PAGE != 0))[:, None] & (j == (lp // PAGE)[:, None])
    keep &= ~tail
    now = count(now, row, keep, 1)
    to = torch.where(valid, lp + s["add"], 0)
    want = tail | ((j >= ((lp + 63) // PAGE)[:, None]) & (j < ((to + 63) // PAGE)[:, None]))
    free = now == 0
    ids = torch.sort(free.int(), descending=True, stable=True).indices.int()
    total, left = want.sum(), free.sum()
    long = (to > ld * PAGE).any()
    ok = (total <= left) & ~long
    rank = (want.flatten().long().cumsum(0) - 1).clamp(0, pages - 1)
    new = torch.where(keep, row, torch.where(want, ids[rank].view(rows, ld), NONE))
    after = count(now.clone(), new, want & ok, 1)
    s["table_out"].copy_(torch.where(ok, new, table))
    s["len_out"].copy_(torch.where(ok, to, n))
    s["ref_out"].copy_(torch.where(ok, after, ref))
    s["stat"].copy_(torch.stack([torch.where(ok, 0, torch.where(long, -1, total - left)), torch.where(ok, left - total, (ref == 0).sum())]))
    move = tail.any(-1) & ok
    at = (lp // PAGE).clamp(max=ld - 1).long()[:, None]
    src = torch.where(move, row.gather(1, at)[:, 0], pages).long()
    dst = torch.where(move, new.gather(1, at)[:, 0], pages).long()
    s["pool"][dst] = s["pool"][src]


def _plain_compact(s):
    table, ref, pages = s["table"], s["ref"], s["case"]["pages"]
    live, ids = ref > 0, torch.arange(pages, device=DEV)
    L = live.sum()
    movers, holes = live & (ids >= L), ~live & (ids < L)
    hole = torch.sort(holes.int(), descending=True, stable=True).indices
    new = torch.where(movers, hole[(movers.long().cumsum(0) - 1).clamp(min=0)], ids)
    held = (table >= 0) & (table < pages)
    s["table_out"].copy_(torch.where(held, new[torch.where(held, table, 0).long()].int(), table))
    s["ref_out"].zero_()
    s["ref_out"].index_add_(0, new, torch.where(live, ref, 0))
    s["stat"].copy_(torch.stack([L, movers.sum()]))
    src = movers.nonzero()[:, 0]
    s["pool"][new[src]] = s["pool"][src]


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(c, seed):
    global own
    if c["op"] in ("step", "compact"):
        return None                                                  # whole numbers only
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["op"] == "beam":
        x = s["logits"].double().log_softmax(-1) + s["score"].double()[:, None]
        done = s["fin"] != 0
        x[done] = -math.inf
        x[done, 1] = s["score"].double()[done]
        top = x.view(c["groups"], -1).sort(-1, descending=True).values[:, :c["beams"]]
        return {"parent": None, "token": None, "score": top.flatten(), "fin": None}
    if c["op"] == "put":
        got = {}
        for name in ("k", "v"):
            x = s[name].double().clamp(-HOLD, HOLD).view(s["n"], c["nkv"], -1, 32)
            lo = x.min(-1, keepdim=True).values.half().double()
            sc = ((x.max(-1, keepdim=True).values - lo) / 15.0).half().double()
            sc[sc == 0] = 1.0
            got[name] = (((x - lo) / sc).round().clamp(0, 15) * sc + lo).half().double().view(s["n"], c["nkv"], c["D"])
        return got
    out, at = torch.zeros(s["n"], c["nh"], c["D"], dtype=torch.float64, device=DEV), 0
    for b, (n, T) in enumerate(_lens(c)):
        if n:
            ids = s["table"][b, :-(-n // PAGE)].long()
            pos = torch.arange(n - T, n, device=DEV)[:, None]
            key = torch.arange(n, device=DEV)[None]
            hide = key > pos
            if c["window"]:
                hide |= (key <= pos - c["window"]) & (key >= c["sinks"])
            for h in range(c["nh"]):
                r = s["pool"][ids, h * c["nkv"] // c["nh"]]
                k, v = (_values(r[:, i], torch.float64).reshape(-1, c["D"])[:n] for i in (0, 1))
                x = s["q"][at:at + T, h].double() @ k.T
                out[at:at + T, h] = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v
        at += T
    return {"out": out}
