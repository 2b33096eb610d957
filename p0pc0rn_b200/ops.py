"""The operators with the reference's own argument objects, over the C ABI.

  gemv(g, a)   -> nsplit   engine/llm/lops.js:108-141       (a = {w, x: {buf, rowB}, N, K, kPer, pro, epi, y: {buf},
                                                            ldy, stat: {buf, off}, norm: {buf, off}, ev: {buf, off},
                                                            src: {n, ld}, mx: {buf}, cap})
  gemvM(g, a)  -> nsplit   engine/llm/lops_spec.js:159-191  (adds M, x.ldx, y.ldm / y.ldy, stat.ld, ev.ld)
  gemm(gpu, a) -> flops    engine/ops/gemm.js:255-322       (a = {w, x: {buf, off, ld, k0, mode}, M, N, K, wr0, wr1, wk0,
                                                            epi, act, acc, y: {buf, off, ld, n0}, ev: {buf, off},
                                                            bv: {buf, off, up}, res, store, stats: {buf, off},
                                                            pv: {buf, off, stride}} + post_gelu)
w = {buf, off (bytes), bytes, enc, rows, cols} as WeightStore.t() returns it (core/store.js:249-253).
Every call enqueues one kernel on the context's stream; results are read with g.read() after it. Errors raise
P0Error with the reference's messages. There is no CPU path: these always run the CUDA kernels in libp0mm.so.
"""
import ctypes

from . import _lib as L
from .gpu import P0Error, handle


def _wview(w, op="gemv"):
    enc = w.get("enc")
    if enc not in L.ENC:
        # gemm.js:267 and lops.js:115 / lops_spec.js:166 word it differently
        raise P0Error(L.P0_EINVAL, (op + ": unsupported weight encoding " if op == "gemm" else op + ": encoding ") + str(enc))
    return L.p0_wview(handle(w["buf"]), int(w.get("off") or 0), int(w.get("bytes") or 0), L.ENC[enc], int(w["rows"]),
                      int(w["cols"]), int(w.get("ld") or 0))


def _b(o):
    return handle(o.get("buf")) if o else L.p0_buf(0)


def gemv(g, a):
    """gemv(g, a) -> nsplit (lops.js:111-141)"""
    x, y = a["x"], a["y"]
    stat, norm, ev, src, mx = a.get("stat"), a.get("norm"), a.get("ev"), a.get("src"), a.get("mx")
    pro, epi = a.get("pro") or "raw", a.get("epi") or "store"
    if pro not in L.PRO:
        raise P0Error(L.P0_EINVAL, "gemv: prologue " + str(pro))
    if epi not in L.EPI:
        raise P0Error(L.P0_EINVAL, "gemv: epilogue " + str(epi))
    args = L.p0_gemv_args(
        _wview(a["w"]), handle(x["buf"]), int(x.get("rowB") or 0), int(a["N"]), int(a["K"]), int(a.get("kPer") or 0), L.PRO[pro],
        L.EPI[epi], handle(y["buf"]), int(a.get("ldy") or 0), _b(stat), int((stat or {}).get("off") or 0), _b(norm),
        int((norm or {}).get("off") or 0), _b(ev), int((ev or {}).get("off") or 0), int((src or {}).get("n") or 0),
        int((src or {}).get("ld") or 0), _b(mx), float(a.get("cap") or 0.0))
    ns = ctypes.c_uint32()
    g._check(g._lib.p0_gemv(g.ctx, ctypes.byref(args), ctypes.byref(ns)))
    return ns.value


def gemvM(g, a):
    """gemvM(g, a) -> nsplit (lops_spec.js:163-191)"""
    return _gemvM(g, a, g._lib.p0_gemvM)


def gemvM_noalloc(g, a):
    """gemvM(g, a) -> nsplit without any device allocation during the call (no counterpart in the reference): for
    callers that must not allocate mid-call, e.g. a latency-bound decode loop that cannot afford the device-wide wait
    of a workspace re-allocation, or a process whose device memory belongs to another allocator. Its scratch is a
    fixed 16 MiB device array shared by every call on the device, so calls that overlap on the GPU race; calls that
    need more scratch raise P0Error (include/p0mm.h has the limits)."""
    return _gemvM(g, a, g._lib.p0_gemvM_noalloc)


def _gemvM(g, a, entry):
    x, y = a["x"], a["y"]
    stat, norm, ev, src, mx = a.get("stat"), a.get("norm"), a.get("ev"), a.get("src"), a.get("mx")
    pro, epi = a.get("pro") or "raw", a.get("epi") or "store"
    if pro not in L.PRO:
        raise P0Error(L.P0_EINVAL, "gemvM: prologue " + str(pro))
    if epi not in L.EPI:
        raise P0Error(L.P0_EINVAL, "gemvM: epilogue " + str(epi))
    args = L.p0_gemvM_args(
        _wview(a["w"], "gemvM"), handle(x["buf"]), int(x.get("rowB") or 0), int(x.get("ldx") or 0), int(a["M"]), int(a["N"]), int(a["K"]),
        int(a.get("kPer") or 0), L.PRO[pro], L.EPI[epi], handle(y["buf"]), int(y.get("ldy") or 0), int(y.get("ldm") or 0),
        _b(stat), int((stat or {}).get("off") or 0), int((stat or {}).get("ld") or 0), _b(norm), int((norm or {}).get("off") or 0),
        _b(ev), int((ev or {}).get("off") or 0), int((ev or {}).get("ld") or 0), int((src or {}).get("n") or 0),
        int((src or {}).get("ld") or 0), _b(mx), float(a.get("cap") or 0.0))
    ns = ctypes.c_uint32()
    g._check(entry(g.ctx, ctypes.byref(args), ctypes.byref(ns)))
    return ns.value


def gemm(gpu, a):
    """gemm(gpu, a) -> flops (gemm.js:264-322). x prologues 'f16', 'lnmod', 'rms'; acc 'f32' or 'f16' (both
    accumulate in f32 on the tensor cores); every epilogue of
    gemm.js:187-250 ('f16', 'f32', 'bias', 'resadd', 'swiglu', 'heads', 'onormgate')."""
    x, y = a["x"], a["y"]
    ev, bv = a.get("ev"), a.get("bv")
    epi = a.get("epi") or "f16"
    if epi not in L.GEPI:
        raise P0Error(L.P0_EINVAL, "gemm: epilogue %s is not built in this library yet" % epi)
    xmode = x.get("mode") or "f16"
    if xmode not in L.XPRO or a.get("conv"):
        raise P0Error(L.P0_EINVAL, "gemm: x prologue %s is not built in this library yet" % ("conv" if a.get("conv") else xmode))
    stats, pv = a.get("stats"), a.get("pv")
    acc = a.get("acc") or "f32"
    args = L.p0_gemm_args(
        _wview(a["w"], "gemm"), handle(x["buf"]), int(x.get("off") or 0), int(x.get("ld") or 0), int(x.get("k0") or 0), int(a["M"]),
        int(a["N"]), int(a["K"]), int(a.get("wr0") or 0), int(a.get("wr1") or 0), int(a.get("wk0") or 0), L.GEPI[epi],
        L.ACT[a.get("act") or "silu"], 1 if acc == "f16" else 0, handle(y["buf"]), int(y.get("off") or 0), int(y.get("ld") or 0),
        int(y.get("n0") or 0), _b(ev), int((ev or {}).get("off") or 0), _b(bv), int((bv or {}).get("off") or 0),
        int((bv or {}).get("up") or 0), int(bool(a.get("res"))), int(bool(a.get("store"))), int(bool(a.get("post_gelu"))),
        L.XPRO[xmode], _b(stats), int((stats or {}).get("off") or 0), _b(pv), int((pv or {}).get("off") or 0),
        int((pv or {}).get("stride") or 0))
    h = a.get("heads") or {}
    args.h_Ltot, args.h_Hq, args.h_Hkv, args.h_rowOff = (int(h.get(k) or 0) for k in ("Ltot", "Hq", "Hkv", "rowOff"))
    args.h_eps = float(h.get("eps") or 0.0)
    args.h_rope_mode = L.P0_ROPE_HALF if h.get("ropeMode") == "half" else L.P0_ROPE_INTER
    args.rope, args.gt = _b(h.get("rope")), _b(a.get("gt"))   # bound from the buffer start, as gemm.js:304 binds them
    fl = ctypes.c_double()
    gpu._check(gpu._lib.p0_gemm(gpu.ctx, ctypes.byref(args), ctypes.byref(fl)))
    return fl.value


def dequant_f16(g, w, out):
    """the GEMM's in-kernel dequantisation of a q4 view written to out (rows*cols fp16), for bit-exact checks"""
    wv = _wview(w, "dequant")
    g._check(g._lib.p0_dequant_f16(g.ctx, ctypes.byref(wv), handle(out)))


def pack_q4(g, w_f32, N, K, out=None, w_off=0, ldw=0, out_off=0):
    """packQ4 (engine/kcheck.js:22-38) on the device: a W f32 [N][K] buffer -> q4g32a.t64 records; returns the out buffer"""
    if out is None:
        out = g.buffer(N * K // 32 * 20, "q4")
    g._check(g._lib.p0_pack_q4(g.ctx, handle(w_f32), int(w_off), int(ldw), int(N), int(K), handle(out), int(out_off)))
    return out


def pack_q8(g, w_f32, N, K, out=None, w_off=0, ldw=0, out_off=0):
    """packQ8 (engine/kcheck.js:39-52) on the device: a W f32 [N][K] buffer -> q8g64s.t64 records; returns the out buffer"""
    if out is None:
        out = g.buffer(N * K // 64 * 66, "q8")
    g._check(g._lib.p0_pack_q8(g.ctx, handle(w_f32), int(w_off), int(ldw), int(N), int(K), handle(out), int(out_off)))
    return out


# ---------------------------------------------------------------- decode-path operators (lops.js, lops_spec.js)
def argmax(g, a):
    """argmax(g, a) (lops.js:434-436): a = {mx: {buf}, n, out: {buf}}; out[0] = the index of the largest of the n
    (max, bitcast index) pairs (ties: the lowest index), out[1] = the bits of that max"""
    g._check(g._lib.p0_argmaxM(g.ctx, handle(a["mx"]["buf"]), int(a["n"]), 1, handle(a["out"]["buf"])))


def argmaxM(g, a):
    """argmaxM(g, a) (lops_spec.js:346-348): a = {mx: {buf}, n, M, out: {buf}}; per row m of mx [M][n][2], out[2m] /
    out[2m + 1] as argmax"""
    g._check(g._lib.p0_argmaxM(g.ctx, handle(a["mx"]["buf"]), int(a["n"]), int(a["M"]), handle(a["out"]["buf"])))


def embed(g, a):
    """embed(g, a) (lops.js:352-365): a = {w (q4 / q8 table view), ids: {buf}, x: {buf}, st: {buf, off}, K, n, scale,
    rowOut, eps}; x[(rowOut + m) * K + k] = dequant(w[ids[m]]) * scale, st[off + m] = the row's rstd"""
    w = a["w"]
    enc = w.get("enc") or "q4g32a.t64"
    if enc not in ("q4g32a.t64", "q8g64s.t64"):
        raise P0Error(L.P0_EINVAL, "embed: encoding " + str(enc))
    st = a["st"]
    args = L.p0_embed_args(_wview(w, "embed"), handle(a["ids"]["buf"]), handle(a["x"]["buf"]), handle(st["buf"]),
                           int(st.get("off") or 0), int(a["K"]), int(a["n"]), int(a.get("rowOut") or 0), float(a["scale"]),
                           float(a.get("eps") or 0.0))
    g._check(g._lib.p0_embed(g.ctx, ctypes.byref(args)))


def normadd(g, a):
    """normadd(g, a) (lops.js:174-180): a = {t: {buf, n, ld}, w: {buf, off} (mode 0), x: {buf}, st: {buf, off}, D, M,
    eps, scale (default 1), mode (0: x = (x + rms(t) * w) * scale, 1: x = t)}"""
    t, w, st = a["t"], a.get("w"), a["st"]
    scale = a.get("scale")
    args = L.p0_normadd_args(handle(t["buf"]), int(t.get("n") or 1), int(t.get("ld") or 0), _b(w), int((w or {}).get("off") or 0),
                             handle(a["x"]["buf"]), handle(st["buf"]), int(st.get("off") or 0), int(a["D"]), int(a.get("M") or 1),
                             int(a.get("mode") or 0), float(a.get("eps") or 0.0), 1.0 if scale is None else float(scale))
    g._check(g._lib.p0_normadd(g.ctx, ctypes.byref(args)))


def dhead(g, a):
    """dhead(g, a) (lops_spec.js:475-482): a = {w (q4 / q8 head view), x: {buf}, stat: {buf, off}, norm: {buf, off},
    sel: {buf}, mx: {buf}, K (<= 512), tPer, nsel}; per selected tile its largest row dot and that row's index"""
    w = a["w"]
    enc = w.get("enc") or "q4g32a.t64"
    if enc not in ("q4g32a.t64", "q8g64s.t64"):
        raise P0Error(L.P0_EINVAL, "dhead: encoding " + str(enc))
    if int(a["K"]) > 512:
        raise P0Error(L.P0_EINVAL, "dhead: K > 512")
    stat, norm = a["stat"], a["norm"]
    args = L.p0_dhead_args(_wview(w, "dhead"), handle(a["x"]["buf"]), handle(stat["buf"]), int(stat.get("off") or 0),
                           handle(norm["buf"]), int(norm.get("off") or 0), handle(a["sel"]["buf"]), handle(a["mx"]["buf"]),
                           int(a["K"]), int(a["tPer"]), int(a["nsel"]))
    g._check(g._lib.p0_dhead(g.ctx, ctypes.byref(args)))


def qkrope(g, a):
    """qkrope(g, a) (lops.js:226-233): a = {s: {buf, n, ld}, norm: {buf}, rope: {buf, off}, q: {buf}, kc: {buf}, vc: {buf},
    D, nq, hasKV, pos, eps, qw, kw, npairs, kvRow, nkv, kvLen}; q f32 out, k / v into the fp16 caches at kvRow"""
    s, rope = a["s"], a["rope"]
    kc, vc = a.get("kc"), a.get("vc")
    args = L.p0_qkrope_args(handle(s["buf"]), int(s.get("n") or 1), int(s.get("ld") or 0), handle(a["norm"]["buf"]), int(a.get("qw") or 0),
                            int(a.get("kw") or 0), handle(rope["buf"]), int(rope.get("off") or 0), int(a["npairs"]), int(a.get("pos") or 0),
                            handle(a["q"]["buf"]), _b(kc), _b(vc), int(a["D"]), int(a["nq"]), int(a.get("nkv") or 1),
                            int(bool(a.get("hasKV"))), int(a.get("kvRow") or 0), int(a.get("kvLen") or 0), float(a.get("eps") or 0.0))
    g._check(g._lib.p0_qkrope(g.ctx, ctypes.byref(args)))


def attnDec(g, a):
    """attnDec(g, a) (lops.js:306-321): a = {q: {buf}, kc: {buf}, vc: {buf}, part: {buf}, out: {buf}, D, nh, kStart, kEnd,
    ring, nkv, kvLen}; out f32 [nh][D] = softmax(q . k) . v over the keys (a tuner's `ad` choice is not used)"""
    args = L.p0_attn_dec_args(handle(a["q"]["buf"]), handle(a["kc"]["buf"]), handle(a["vc"]["buf"]), handle(a["part"]["buf"]),
                              handle(a["out"]["buf"]), int(a["D"]), int(a["nh"]), int(a.get("nkv") or 1), int(a.get("kvLen") or 0),
                              int(a["kStart"]), int(a["kEnd"]), int(a.get("ring") or 0))
    g._check(g._lib.p0_attn_dec(g.ctx, ctypes.byref(args)))


# ---------------------------------------------------------------- paged 4-bit cache and beam search
# Each operator's arguments become a C struct once per call; a loop that repeats a call keeps it with bound().
def _kv(kv):
    pool, table, ln = kv["pool"], kv["table"], kv["len"]
    return L.p0_kv(handle(pool["buf"]), int(pool.get("off") or 0), int(pool.get("stride") or 0), handle(table["buf"]), int(table.get("off") or 0),
                   int(table["ld"]), handle(ln["buf"]), int(ln.get("off") or 0), int(kv["pages"]), int(kv["rows"]), int(kv.get("D") or 0),
                   int(kv.get("nkv") or 0))


def _rows(r):
    return L.p0_rows(handle(r["buf"]), int(r.get("off") or 0), int(r.get("ld") or 0), int(r.get("ldh") or 0))


def _type(a, op):
    t = a.get("type") or "f32"
    if t not in L.TYPE:
        raise P0Error(L.P0_EINVAL, "%s: type %s" % (op, t))
    return L.TYPE[t]


def _kv4_rows_args(a, op):
    cu = a.get("cu")
    return L.p0_kv4_rows_args(_kv(a["kv"]), _rows(a["k"]), _rows(a["v"]), _type(a, op), int(a["n"]), int(a.get("T") or 0), _b(cu),
                              int((cu or {}).get("off") or 0))


def _kv4_attn_args(a):
    cu = a.get("cu")
    return L.p0_kv4_attn_args(_kv(a["kv"]), _rows(a["q"]), _rows(a["out"]), _type(a, "kv4Attn"), int(a["nh"]), int(a["n"]), int(a.get("T") or 0),
                              _b(cu), int((cu or {}).get("off") or 0), int(a.get("window") or 0), int(a.get("sinks") or 0),
                              float(a.get("scale") or 0.0))


def _kv_step_args(a):
    to, add = a["to"], a.get("add")
    num = not isinstance(add, dict)
    return L.p0_kv_step_args(_kv(a["kv"]), handle(a["ref"]["buf"]), handle(to["table"]["buf"]), handle(to["len"]["buf"]), handle(to["ref"]["buf"]),
                             _b(a.get("parent")), _b(None if num else add), int(add or 0) if num else 0, int(a.get("window") or 0),
                             int(a.get("sinks") or 0), handle(a["stat"]["buf"]))


def _kv_compact_args(a):
    to = a["to"]
    return L.p0_kv_compact_args(_kv(a["kv"]), handle(a["ref"]["buf"]), handle(to["table"]["buf"]), handle(to["ref"]["buf"]), handle(a["stat"]["buf"]))


def _beam_args(a):
    lg, eos = a["logits"], a.get("eos")
    return L.p0_beam_args(handle(lg["buf"]), int(lg.get("off") or 0), int(lg.get("ld") or 0), handle(a["score"]["buf"]), _b(a.get("fin")),
                          int(a["groups"]), int(a["beams"]), int(a["V"]), L.P0_KV_NONE if eos is None else int(eos), handle(a["parent"]["buf"]),
                          handle(a["token"]["buf"]), handle(a["scoreOut"]["buf"]), _b(a.get("finOut")))


def kv4Put(g, a):
    """a = {kv, k, v: {buf, off, ld, ldh}, type ('f32' | 'f16'), n, T or cu: {buf, off}}: the n newest tokens' K and V rows
    quantised into their pages. kv = {pool: {buf, off, stride}, pages, table: {buf, off, ld}, len: {buf, off}, rows, D,
    nkv} is one layer's view of the cache (p0_kv in include/p0mm.h)."""
    bound(kv4Put, g, a)()


def kv4Get(g, a):
    """a as kv4Put's, with k and v the rows to write: the values the newest tokens' codes stand for"""
    bound(kv4Get, g, a)()


def kv4Attn(g, a):
    """a = {kv, q, out: {buf, off, ld, ldh}, type, nh, n, T or cu, window, sinks, scale}: attention of each sequence's
    newest tokens over its pages (causal; window 0 = the whole context, else the last `window` keys and the first
    `sinks`)"""
    bound(kv4Attn, g, a)()


def kvStep(g, a):
    """a = {kv, ref, to: {table, len, ref}, parent (optional), add ({buf} or a number), window, sinks, stat}: forks,
    reorders, frees, trims and extends the sequences' pages; the new state goes to `to`, stat = {pages missing, free}"""
    bound(kvStep, g, a)()


def kvCompact(g, a):
    """a = {kv, ref, to: {table, ref}, stat}: the pages in use moved into the lowest ones; stat = {in use, moved}"""
    bound(kvCompact, g, a)()


def beamSelect(g, a):
    """a = {logits: {buf, off, ld}, score, fin (optional), groups, beams, V, eos, parent, token, scoreOut, finOut
    (optional)}: the best `beams` continuations of each group's beams; parent is what kvStep takes"""
    bound(beamSelect, g, a)()


# ---------------------------------------------------------------- matrices in 8 bits
def _f8(m):
    sc = (m or {}).get("s") or {}
    m = m or {}
    return L.p0_f8(_b(m), int(m.get("off") or 0), int(m.get("ld") or 0), _b(sc), int(sc.get("off") or 0), int(sc.get("ld") or 0))


def _o(o, k="off"):
    return int((o or {}).get(k) or 0)


def _pack_f8_args(a):
    x, block = a["x"], a.get("block") or "row"
    if block not in L.F8BLOCK:
        raise P0Error(L.P0_EINVAL, "packF8: block %s" % block)
    return L.p0_pack_f8_args(handle(x["buf"]), _o(x), _o(x, "ld"), _type(a, "packF8"), int(a["M"]), int(a["K"]), L.F8BLOCK[block], _f8(a["y"]))


def _norm_f8_args(a):
    x, t, pw, h, w, st, scale = a["x"], a.get("t"), a.get("pw"), a.get("h"), a["w"], a.get("st"), a.get("scale")
    return L.p0_norm_f8_args(handle(x["buf"]), _o(x), _o(x, "ld"), _type(a, "normF8"), _b(t), _o(t), _o(t, "ld"), _o(t, "ldm"), _type(t or {}, "normF8"),
                             _o(t, "n"), _b(pw), _o(pw), _b(h), _o(h), _o(h, "ld"), handle(w["buf"]), _o(w), _f8(a["y"]), _b(st), _o(st), int(a["M"]),
                             int(a["D"]), float(a.get("eps") or 0.0), 1.0 if scale is None else float(scale))


def _gemm_f8_args(a):
    epi, bv = a.get("epi") or "f16", a.get("bv")
    if epi not in L.F8EPI:
        raise P0Error(L.P0_EINVAL, "gemmF8: epilogue %s" % epi)
    return L.p0_gemm_f8_args(_f8(a["x"]), _f8(a["w"]), _f8(a.get("u")), int(a["M"]), int(a["N"]), int(a["K"]), L.F8EPI[epi], _b(bv), _o(bv), _f8(a["y"]))


def packF8(g, a):
    """a = {x: {buf, off, ld}, type ('f32' | 'f16'), M, K, block ('row' | 'tile'), y}: values as e4m3 codes with a scale for
    each 128 columns of a row (activations) or each 128 x 128 tile (weights). y = {buf, off, ld, s: {buf, off, ld}} is a matrix
    in 8 bits (p0_f8 in include/p0mm.h)."""
    bound(packF8, g, a)()


def normF8(g, a):
    """a = {x: {buf, off, ld}, type, t: {buf, off, type, n, ld, ldm} (optional), pw: {buf, off} (optional), h: {buf, off, ld}
    (default: x itself), w: {buf, off}, y, st: {buf, off} (optional), M, D, eps, scale (default 1)}: h = (x + t) * scale, t
    summed over n partial rows and with pw normed first; y = the codes of rms(h) * w, st = the rows' rstd"""
    bound(normF8, g, a)()


def gemmF8(g, a):
    """a = {x, w, u (gated only), M, N, K, epi, bv: {buf, off} (optional), y}: x [M][K] in blocks of rows times w [N][K] in
    tiles, all matrices in 8 bits. epi 'f16' (default) | 'f32': y = {buf, off, ld} of that type; 'swiglu' | 'geglu': y = the
    codes of act(x w^T) * (x u^T)"""
    bound(gemmF8, g, a)()


_BOUND = {
    packF8: ("p0_pack_f8", _pack_f8_args),
    normF8: ("p0_norm_f8", _norm_f8_args),
    gemmF8: ("p0_gemm_f8", _gemm_f8_args),
    kv4Put: ("p0_kv4_put", lambda a: _kv4_rows_args(a, "kv4Put")),
    kv4Get: ("p0_kv4_get", lambda a: _kv4_rows_args(a, "kv4Get")),
    kv4Attn: ("p0_kv4_attn", _kv4_attn_args),
    kvStep: ("p0_kv_step", _kv_step_args),
    kvCompact: ("p0_kv_compact", _kv_compact_args),
    beamSelect: ("p0_beam_select", _beam_args),
}


def bound(op, g, a):
    """the call op(g, a) with its arguments converted once: a function without arguments that makes it (and checks it)
    again each time. For loops whose buffers stay and whose lengths live on the device; a's later changes are not seen."""
    name, make = _BOUND[op]
    entry, args = getattr(g._lib, name), make(a)
    ref = ctypes.byref(args)

    def call():
        st = entry(g.ctx, ref)
        if st:
            g._check(st)
    return call
