"""Measured cases of the 8-bit operators: packF8 (values to e4m3 codes with a scale for each block of 128), normF8 (the
residual's addition and a root-mean-square norm, with such codes as its output) and gemmF8 (the product of two such
matrices, its results as f32 or f16, or gated and as codes again).

Where `own` is false `run` computes an operator in elementary torch operations in 32 bits; where it is true it makes the
framework's calls.

A matrix in 8 bits is codes u8 [rows][ld] (e4m3) and f32 scales; a code c of the block with scale s stands for c * s. Of
activations each row's 128 columns are a block, scales [K / 128][ld] (a column per row); of weights each 128 x 128 tile,
scales [N / 128][K / 128]. s = a / 448 with a the block's largest magnitude, code = e4m3(x * (448 / a)).
"""
import math
import weakref

import torch

own = False

DEV = "cuda"
B = 128                # rows and columns of a block
TOP = 448.0            # the largest e4m3 value
LEAST = 2.0 ** -100    # a block's largest magnitude counts as no less: zeros get a scale all the same
F8 = torch.float8_e4m3fn


def listed():
    return [
        # an attention output of a few drafted tokens before its projection: the call's latency
        _pack("pack_rows_few", "f32", 5, 2048, "row"),
        # a DiT's activations of 4096 image tokens before the down projection
        _pack("pack_rows_image", "f16", 4096, 12288, "row"),
        # a video DiT's weights, once at loading; K ends inside a block
        _pack("pack_weights", "f32", 8960, 2240, "tile"),
        # a decode token between attention and MLP: two partial sums, the norm behind the sublayer and the next one's
        _norm("norm_token", "f32", "f32", 1, 2560, parts=2, post=True),
        # a prompt's residual stream in f32, the sublayer's output in f16
        _norm("norm_prompt", "f32", "f16", 2051, 1536, parts=1, post=True),
        # a video's tokens in f16 throughout; D ends inside a block
        _norm("norm_video", "f16", "f16", 32760, 2240, parts=1),
        # one decode token's projection; eight tokens to verify through the gated half of an MLP
        _gemm("gemm_token", 1, 2048, 2048, "f32"),
        _gemm("gemm_verify_gated", 8, 8192, 2048, "geglu"),
        # a chunk of a prompt; more of one through the gated MLP
        _gemm("gemm_chunk", 100, 6720, 2240, "f16"),
        _gemm("gemm_prompt_gated", 1031, 8960, 2240, "swiglu"),
        # a picture's tokens; a video's (K ends inside a block, M and N inside tiles)
        _gemm("gemm_image", 4096, 12288, 4096, "f16", bias=True),
        _gemm("gemm_video", 32760, 6720, 2240, "f16"),
    ]


def _pack(name, kind, M, K, block):
    return {"name": name, "op": "pack", "type": kind, "M": M, "K": K, "block": block}


def _norm(name, kind, t, M, D, parts=0, post=False):
    """parts: partial sums that the sublayer left (0: the residual stream is normed as it is)"""
    return {"name": name, "op": "norm", "type": kind, "t": t, "M": M, "D": D, "parts": parts, "post": post}


def _gemm(name, M, N, K, epi, bias=False):
    return {"name": name, "op": "gemm", "M": M, "N": N, "K": K, "epi": epi, "bias": bias}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        top = {k: max(top.get(k, 0), w[k]) for k in w}
    while True:
        op = rng.choice(["pack", "norm", "gemm", "gemm", "gemm"])
        odd = lambda v: v if rng.random() < 0.3 else max(8, v // 8 * 8)
        M = _log(rng, 1, 32768)
        if op == "pack":
            c = _pack("", rng.choice(["f32", "f16"]), M, odd(_log(rng, 16, 16384)), rng.choice(["row", "row", "tile"]))
        elif op == "norm":
            kind, parts = rng.choice(["f32", "f16"]), rng.choice([0, 1, 1, 1, 2, 3])
            t = kind if not parts else rng.choice(["f32", "f16"]) if parts == 1 else "f32"
            c = _norm("", kind, t, M, odd(_log(rng, 64, 12288)), parts, parts > 0 and rng.random() < 0.5)
        else:
            epi = rng.choice(["f32", "f16", "f16", "swiglu", "geglu"])
            c = _gemm("", M, odd(_log(rng, 16, 16384)), odd(_log(rng, 32, 16384)), epi, epi in ("f32", "f16") and rng.random() < 0.3)
        del c["name"]
        w = work(c)
        if all(w[k] <= top[k] for k in w):
            return c


def _size(kind):
    return 4 if kind == "f32" else 2


def _up(n, m):
    return -(-n // m) * m


def _blocks(n):
    return -(-n // B)


def work(c):
    if c["op"] == "pack":
        n = c["M"] * c["K"]
        scales = (c["M"] if c["block"] == "row" else _blocks(c["M"])) * _blocks(c["K"])
        return {"bytes": n * (_size(c["type"]) + 1) + 4 * scales, "flops": 3 * n}
    if c["op"] == "norm":
        n = c["M"] * c["D"]
        stream = _size(c["type"]) * (2 if c["parts"] else 1)
        return {"bytes": n * (stream + c["parts"] * _size(c["t"]) + 1) + 4 * c["M"] * (_blocks(c["D"]) + 1) + 4 * c["D"] * (2 if c["post"] else 1),
                "flops": n * (7 + c["parts"] + (4 if c["post"] else 0))}
    M, N, K, gated = c["M"], c["N"], c["K"], c["epi"] in ("swiglu", "geglu")
    size = M * K + 4 * M * _blocks(K) + (2 if gated else 1) * (N * K + 4 * _blocks(N) * _blocks(K)) + (4 * N if c["bias"] else 0)
    size += M * N + 4 * M * _blocks(N) if gated else M * N * _size(c["epi"])
    return {"bytes": size, "flops": 2 * M * N * K * (2 if gated else 1)}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _type(kind):
    return torch.float32 if kind == "f32" else torch.float16


def _activations(g, M, K):
    """bell-shaped, rows of different sizes, a few columns far larger than the others, as a decoder's"""
    x = torch.randn(M, K, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(M, 1, generator=g, device=DEV))
    loud = torch.randint(0, K, (max(1, K // 256),), generator=g, device=DEV)
    x[:, loud] *= 20.0
    return x


def _f8(M, K, block):
    """an empty matrix in 8 bits: codes [M][K up to 16], scales"""
    s = (_blocks(K), _up(M, 4)) if block == "row" else (_blocks(M), _blocks(K))
    return torch.zeros(M, _up(K, 16), dtype=torch.uint8, device=DEV), torch.zeros(s, dtype=torch.float32, device=DEV)


def _weights(g, N, K):
    q, s = _f8(N, K, "tile")
    _pack_plain(torch.randn(N, K, generator=g, device=DEV) / math.sqrt(K), q, s, "tile")
    return q, s


class State(dict):
    """what a user's program has in hand; with the framework's own calls, its buffer registrations go when it goes"""


def prepare(c, seed):
    s, g = State(case=c), _gen(seed)
    if c["op"] == "pack":
        x = _activations(g, c["M"], c["K"]) if c["block"] == "row" else torch.randn(c["M"], c["K"], generator=g, device=DEV) / math.sqrt(c["K"])
        s["x"] = x.to(_type(c["type"]))
        s["y"], s["ys"] = _f8(c["M"], c["K"], c["block"])
    elif c["op"] == "norm":
        M, D = c["M"], c["D"]
        s["x"] = _activations(g, M, D).to(_type(c["type"]))
        if c["parts"]:
            s["t"] = torch.randn(c["parts"], M, D, generator=g, device=DEV).to(_type(c["t"]))
            s["h"] = torch.zeros(M, D, dtype=_type(c["type"]), device=DEV)
        if c["post"]:
            s["pw"] = 1.0 + 0.2 * torch.randn(D, generator=g, device=DEV)
        s["w"] = 1.0 + 0.2 * torch.randn(D, generator=g, device=DEV)
        s["y"], s["ys"] = _f8(M, D, "row")
        s["st"] = torch.zeros(M, device=DEV)
    else:
        M, N, K = c["M"], c["N"], c["K"]
        s["x"], s["xs"] = _f8(M, K, "row")
        _pack_plain(_activations(g, M, K), s["x"], s["xs"], "row")
        s["w"], s["ws"] = _weights(g, N, K)
        if c["epi"] in ("swiglu", "geglu"):
            s["u"], s["us"] = _weights(g, N, K)
            s["y"], s["ys"] = _f8(M, N, "row")
        else:
            s["y"] = torch.zeros(M, N, dtype=_type(c["epi"]), device=DEV)
        if c["bias"]:
            s["bv"] = 0.1 * torch.randn(N, generator=g, device=DEV)
    if own:
        _bind(s)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
_GPU = []


def _bind(s):
    """registers the tensors with the framework's context and keeps the call's checked arguments, as a serving loop does"""
    import p0pc0rn_b200 as p0
    if not _GPU:
        _GPU.append(p0.Gpu(0))
        _GPU[0].set_stream(1)                                        # the stream that torch's work is on
    g, c = _GPU[0], s["case"]
    bufs = {k: g.wrap(v.data_ptr(), v.numel() * v.element_size(), k) for k, v in s.items() if isinstance(v, torch.Tensor)}
    weakref.finalize(s, lambda: [g.free(b) for b in bufs.values()])
    b = lambda k: {"buf": bufs[k]}
    f8 = lambda k: {"buf": bufs[k], "ld": s[k].shape[1], "s": {"buf": bufs[k + "s"], "ld": s[k + "s"].shape[1]}}
    if c["op"] == "pack":
        call = (p0.packF8, {"x": b("x"), "type": c["type"], "M": c["M"], "K": c["K"], "block": c["block"], "y": f8("y")})
    elif c["op"] == "norm":
        a = {"x": b("x"), "type": c["type"], "w": b("w"), "y": f8("y"), "st": b("st"), "M": c["M"], "D": c["D"]}
        if c["parts"]:
            a.update(t={"buf": bufs["t"], "type": c["t"], "n": c["parts"]}, h=b("h"))
        if c["post"]:
            a["pw"] = b("pw")
        call = (p0.normF8, a)
    else:
        a = {"x": f8("x"), "w": f8("w"), "M": c["M"], "N": c["N"], "K": c["K"], "epi": c["epi"]}
        if "u" in s:
            a.update(u=f8("u"), y=f8("y"))
        else:
            a["y"] = b("y")
        if c["bias"]:
            a["bv"] = b("bv")
        call = (p0.gemmF8, a)
    s["call"] = p0.bound(call[0], g, call[1])


def run(s):
    c = s["case"]
    if own:
        s["call"]()
    else:
        {"pack": _plain_pack, "norm": _plain_norm, "gemm": _plain_gemm}[c["op"]](s)
    if c["op"] == "gemm" and "ys" not in s:
        return {"y": s["y"]}
    n = {"pack": c.get("K"), "norm": c.get("D"), "gemm": c.get("N")}[c["op"]]
    got = {"y": s["y"].view(F8)[:, :n], "s": s["ys"] if c.get("block") == "tile" else s["ys"][:, :c["M"]]}
    if c["op"] == "norm":
        got["st"] = s["st"]
        if c["parts"]:
            got["h"] = s["h"]
    return got


# ------------------------------------------------------------------------------------------------ the plain forms
def _pack_plain(x, q, s, block):
    """x f32 [M][K] -> codes into q, scales into s, each step in f32"""
    M, K = x.shape
    rows = 1 if block == "row" else B
    v = torch.nn.functional.pad(x, (0, _up(K, B) - K, 0, _up(M, rows) - M)).view(-1, rows, _blocks(K), B)
    a = v.abs().amax((1, 3), keepdim=True).clamp(min=LEAST)
    y = (v * (torch.full_like(a, TOP) / a)).to(F8).view(-1, _blocks(K) * B)
    q[:, :K].copy_(y[:M, :K].view(torch.uint8))
    a = a.view(a.shape[0], -1) / TOP
    s[:, :M].copy_(a.T) if block == "row" else s.copy_(a)


def _plain_pack(s):
    _pack_plain(s["x"].float(), s["y"], s["ys"], s["case"]["block"])


def _plain_norm(s):
    h = s["x"].float()
    if "t" in s:
        t = s["t"].float().sum(0)
        if "pw" in s:
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * s["pw"]
        s["h"].copy_(h + t)
        h = s["h"].float()
    r = torch.rsqrt(h.square().mean(-1) + 1e-6)
    s["st"].copy_(r)
    _pack_plain(h * r[:, None] * s["w"], s["y"], s["ys"], "row")


def _values(q, s, K, block, dt=torch.float32):
    """what codes stand for, [M][K]"""
    x = q.view(F8)[:, :K].to(dt)
    if block == "row":
        return x * s[:, :q.shape[0]].T.to(dt).repeat_interleave(B, 1)[:, :K]
    return x * s.to(dt).repeat_interleave(B, 0)[:q.shape[0]].repeat_interleave(B, 1)[:, :K]


def _plain_gemm(s):
    c = s["case"]
    x = _values(s["x"], s["xs"], c["K"], "row")
    y = x @ _values(s["w"], s["ws"], c["K"], "tile").T
    if "u" in s:
        u = x @ _values(s["u"], s["us"], c["K"], "tile").T
        if c["epi"] == "swiglu":
            y = y / (1.0 + torch.exp(-y))
        else:
            y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
        _pack_plain(y * u, s["y"], s["ys"], "row")
    else:
        s["y"].copy_(y + s["bv"] if "bv" in s else y)


# ------------------------------------------------------------------------------------------------ 64 bits
def _e4m3(v):
    """f64 values rounded to the nearest e4m3 value, halves to even"""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _coded(v, block):
    """f64 [M][K] -> the values of the codes, and the scales as they are laid out"""
    M, K = v.shape
    y, cols = torch.empty_like(v), []
    for k in range(0, K, B):
        a = v[:, k:k + B].abs().amax(1)
        if block == "tile":
            a = torch.stack([t.max() for t in a.split(B)])
        a = a.clamp(min=LEAST)
        cols.append(a / TOP)
        y[:, k:k + B] = _e4m3(v[:, k:k + B] / (cols[-1] if block == "row" else cols[-1].repeat_interleave(B)[:M])[:, None])
    return {"y": y, "s": torch.stack(cols) if block == "row" else torch.stack(cols, 1)}


def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.dtype != torch.uint8}
    if c["op"] == "pack":
        return _coded(d["x"], c["block"])
    if c["op"] == "norm":
        got, h = {}, d["x"]
        if c["parts"]:
            t = d["t"].sum(0)
            if c["post"]:
                t = t / (t.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * d["pw"]
            got["h"] = h + t
            h = got["h"].to(s["h"].dtype).double()
        got["st"] = 1.0 / (h.pow(2).mean(1) + 1e-6).sqrt()
        return {**got, **_coded(h * got["st"][:, None] * d["w"], "row")}
    side = lambda k, block: _values(s[k], s[k + "s"], c["K"], block, torch.float64)
    x = side("x", "row")
    y = x @ side("w", "tile").T
    if c["epi"] in ("swiglu", "geglu"):
        u = x @ side("u", "tile").T
        gate = torch.sigmoid(y) if c["epi"] == "swiglu" else torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
        return _coded(y * gate * u, "row")
    return {"y": y + d["bv"] if c["bias"] else y}
