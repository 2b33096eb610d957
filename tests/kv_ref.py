"""Plain statements of the paged 4-bit cache and beam search operators on the host, for the tests: quantisation in f32 as
the operator defines it, everything else in 64 bits or whole numbers, with loops."""
import numpy as np

PAGE, NONE, HOLD = 64, 0xffffffff, np.float32(60000.0)


def quantise(x):
    """[..., 32] f32 -> (codes u8 [..., 32], s f16, mn f16), every step in f32"""
    x = np.where(np.isnan(x), np.float32(0), np.clip(x.astype(np.float32), -HOLD, HOLD))
    mn = (x.min(-1) + np.float32(0)).astype(np.float16)              # -0 as +0
    s = ((x.max(-1) - mn.astype(np.float32)) / np.float32(15)).astype(np.float16)
    s = np.where(s == 0, np.float16(1), s)
    q = np.rint((x - mn.astype(np.float32)[..., None]) / s.astype(np.float32)[..., None])
    return np.clip(q, 0, 15).astype(np.uint8), s, mn


def stands_for(q, s, mn):
    """f16(q * s + mn) as f64 (the f64 sum is exact; one rounding)"""
    v = q.astype(np.float64) * s.astype(np.float64)[..., None] + mn.astype(np.float64)[..., None]
    with np.errstate(over="ignore"):
        return v.astype(np.float16).astype(np.float64)


class Cache:
    """one layer of a cache on the host: pool u8 [pages][stride], table, len, ref"""

    def __init__(self, rng, lens, nkv, D, ld=None, spare=3, stride=0, off=0):
        self.nkv, self.D, self.lens = nkv, D, np.array(lens, np.uint32)
        self.part = D // 32 * 1280
        self.stride, self.off = stride or nkv * 2 * self.part, off
        need = [-(-int(n) // PAGE) for n in lens]
        self.pages, self.ld = sum(need) + spare, ld or max(need + [1]) + 1
        ids = rng.permutation(self.pages).astype(np.uint32)
        self.table = np.full((len(lens), self.ld), NONE, np.uint32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = ids[at:at + k]
            at += k
        self.pool = np.zeros((self.pages, self.stride), np.uint8)

    def write(self, b, pos, kv, head, x):
        """row x [D] as sequence b's K (kv = 0) or V (1) at pos"""
        page = self.table[b, pos // PAGE]
        if page >= self.pages:
            return
        q, s, mn = quantise(np.asarray(x, np.float32).reshape(-1, 32))
        at = self.off + (head * 2 + kv) * self.part
        r = pos % PAGE
        for g in range(self.D // 32):
            rec = self.pool[page, at + g * 1280:at + (g + 1) * 1280]
            rec[r * 16:(r + 1) * 16] = q[g, 0::2] | (q[g, 1::2] << 4)
            rec[1024 + 4 * r:1028 + 4 * r] = np.array([s[g], mn[g]], np.float16).view(np.uint8)

    def fill(self, rng, scale=1.0):
        """every mapped slot below its sequence's length gets random rows"""
        for b, n in enumerate(self.lens):
            for pos in range(int(n)):
                for h in range(self.nkv):
                    for kv in (0, 1):
                        self.write(b, pos, kv, h, rng.standard_normal(self.D).astype(np.float32) * scale)

    def fill_fast(self, rng):
        """random codes, scales and minima in every slot of the layer"""
        G = self.D // 32
        rec = np.zeros((self.pages, self.nkv, 2, G, 1280), np.uint8)
        rec[..., :1024] = rng.integers(0, 256, (self.pages, self.nkv, 2, G, 1024), dtype=np.uint8)
        s = rng.uniform(0.12, 0.25, (self.pages, self.nkv, 2, G, 64)).astype(np.float16)
        mn = (-7.5 * s.astype(np.float32) + 0.1 * rng.standard_normal(s.shape)).astype(np.float16)
        rec[..., 1024:] = np.stack([s, mn], -1).reshape(self.pages, self.nkv, 2, G, 128).view(np.uint8)
        self.pool[:, self.off:self.off + self.nkv * 2 * self.part] = rec.reshape(self.pages, -1)

    def poison_unseen(self, b, seen):
        """slots of sequence b whose position is not in `seen`: NaN scale and infinite minimum"""
        bad = np.array([np.nan, np.inf], np.float16).view(np.uint8)
        for j in range(self.ld):
            page = self.table[b, j]
            if page >= self.pages:
                continue
            for r in range(PAGE):
                if j * PAGE + r not in seen:
                    for rec in range(self.nkv * 2 * self.D // 32):
                        at = self.off + rec * 1280 + 1024 + 4 * r
                        self.pool[page, at:at + 4] = bad

    def values(self, b, kv, head, n):
        """rows 0 .. n - 1 in f64 (zeros where there is no page), and which have one"""
        out, there = np.zeros((n, self.D)), np.zeros(n, bool)
        at, G = self.off + (head * 2 + kv) * self.part, self.D // 32
        for j in range(-(-n // PAGE)):
            page = self.table[b, j] if j < self.ld else NONE
            if page >= self.pages:
                continue
            rec = self.pool[page, at:at + self.part].reshape(G, 1280)
            c = rec[:, :1024].reshape(G, 64, 16)
            q = np.stack([c & 15, c >> 4], -1).reshape(G, 64, 32)
            sm = np.ascontiguousarray(rec[:, 1024:]).view(np.float16).reshape(G, 64, 2)
            v = stands_for(q, sm[..., 0], sm[..., 1]).transpose(1, 0, 2).reshape(64, self.D)
            m = min(PAGE, n - j * PAGE)
            out[j * PAGE:j * PAGE + m] = v[:m]
            there[j * PAGE:j * PAGE + m] = True
        return out, there


def visible(p, n, window, sinks):
    j = np.arange(n)
    see = j <= p
    if window:
        see &= (j > p - window) | (j < sinks)
    return see


def attention(c, q, counts, nh, window=0, sinks=0, scale=1.0):
    """(out, sum p |v|, max over seen keys of scale * sum |q k|) in f64, [n][nh][D] twice and [n][nh]"""
    n, D = q.shape[0], c.D
    out, spread, size = np.zeros((n, nh, D)), np.zeros((n, nh, D)), np.zeros((n, nh))
    at = 0
    for b, T in enumerate(counts):
        ln = min(int(c.lens[b]), c.ld * PAGE)
        for h in range(c.nkv):
            (k, there), (v, _) = c.values(b, 0, h, ln), c.values(b, 1, h, ln)
            k, v = np.nan_to_num(k, posinf=0, neginf=0), np.nan_to_num(v, posinf=0, neginf=0)
            for i in range(T):
                see = visible(ln - T + i, ln, window, sinks) & there
                if not see.any():
                    continue
                for hq in range(h * nh // c.nkv, (h + 1) * nh // c.nkv):
                    x = q[at + i, hq].astype(np.float64)
                    s = scale * (k[see] @ x)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[at + i, hq] = p @ v[see]
                    spread[at + i, hq] = p @ np.abs(v[see])
                    size[at + i, hq] = abs(scale) * (np.abs(k[see]) @ np.abs(x)).max()
        at += T
    return out, spread, size


def attention_prompt(c, q, counts, nh, window=0, sinks=0, scale=1.0):
    """attention(), a head's rows at a time"""
    n, D = q.shape[0], c.D
    out, spread, size = np.zeros((n, nh, D)), np.zeros((n, nh, D)), np.zeros((n, nh))
    at = 0
    for b, T in enumerate(counts):
        ln = min(int(c.lens[b]), c.ld * PAGE)
        see = np.stack([visible(ln - T + i, ln, window, sinks) for i in range(T)])
        for h in range(c.nkv):
            (k, there), (v, _) = c.values(b, 0, h, ln), c.values(b, 1, h, ln)
            mask = see & there
            any_ = mask.any(-1)
            for hq in range(h * nh // c.nkv, (h + 1) * nh // c.nkv):
                x = q[at:at + T, hq].astype(np.float64)
                s = np.where(mask, scale * (x @ k.T), -np.inf)
                p = np.exp(s - np.where(any_, s.max(-1, initial=-np.inf), 0.0)[:, None])
                p /= np.maximum(p.sum(-1, keepdims=True), 1e-300)
                out[at:at + T, hq], spread[at:at + T, hq] = p @ v, p @ np.abs(v)
                size[at:at + T, hq] = abs(scale) * np.where(mask, np.abs(x) @ np.abs(k).T, 0.0).max(-1, initial=0.0)
        at += T
    return out, spread, size


def attention_bound(spread, size, out, D, pages, f16):
    """How far a right kernel's output may be from 64 bits, element by element. f32: q split into two f16 parts leaves
    2^-22 |q|, at most D / 16 + D / 32 sums of f32 in a score, P split leaves 2^-22 p, exp within 2^-21, one f32 sum a
    page and eight inside it. A score's error e changes each p, and the sum of p, by a factor of at most exp(e). f16: P and
    the output are rounded to f16 (2^-11 each; a P below 2^-14 to a multiple of 2^-24), f32 sums otherwise."""
    e = (D / 16 + D / 32 + 4) * 2.0 ** -23 * size[..., None]
    rel = 2 * e + 2.0 ** -20 + (pages + 8) * 2.0 ** -23
    if not f16:
        return rel * spread + 1e-30
    return (rel + 2.0 ** -11) * spread + 2.0 ** -11 * np.abs(out) + pages * PAGE * 2.0 ** -25 * 3.0 + 2.0 ** -24


def step(table, lens, ref, pages, parent=None, add=0, window=0, sinks=0):
    """kvStep: (table, len, ref, stat, [(source, destination)]) or the old state with what is missing"""
    R, ld = table.shape
    add = np.full(R, add, np.int64) if np.isscalar(add) else np.asarray(add, np.int64)
    parent = np.arange(R) if parent is None else parent
    n_of = lambda b: min(int(lens[b]), ld * PAGE)
    old_free = int((ref == 0).sum())
    r = ref.astype(np.int64).copy()
    for b in range(R):
        for j in range(-(-n_of(b) // PAGE)):
            if table[b, j] < pages:
                r[table[b, j]] -= 1
    new, ln = np.full((R, ld), NONE, np.uint32), np.zeros(R, np.uint32)
    seen, wants = set(), []
    for i in range(R):
        p = int(parent[i])
        if p >= R or p < 0:
            continue
        n = n_of(p)
        if n + add[i] > ld * PAGE:
            return table.copy(), lens.copy(), ref.copy(), (NONE, old_free), []
        for j in range(-(-n // PAGE)):
            page = table[p, j]
            if page >= pages or (window and j * PAGE + 63 <= n - window and j * PAGE >= sinks):
                continue
            if n % PAGE and j == n // PAGE and p in seen:
                wants.append((i, j, int(page)))
                continue
            new[i, j] = page
            r[page] += 1
        for j in range(-(-n // PAGE), -(-(n + int(add[i])) // PAGE)):
            wants.append((i, j, None))
        ln[i] = n + add[i]
        seen.add(p)
    free = np.nonzero(r == 0)[0]
    if len(wants) > len(free):
        return table.copy(), lens.copy(), ref.copy(), (len(wants) - len(free), old_free), []
    copies = []
    for (i, j, src), page in zip(wants, free):
        new[i, j] = page
        r[page] = 1
        if src is not None:
            copies.append((src, int(page)))
    return new, ln, r.astype(np.uint32), (0, len(free) - len(wants)), copies


def compact(table, ref, pages):
    live = np.nonzero(ref)[0]
    L = len(live)
    movers = [p for p in live if p >= L]
    holes = [p for p in range(L) if ref[p] == 0]
    to = dict(zip(movers, holes))
    t = np.array([[to.get(p, p) if p < pages else p for p in row] for row in table.tolist()], np.uint32).reshape(table.shape)
    r = np.zeros_like(ref)
    for p in live:
        r[to.get(p, p)] = ref[p]
    return t, r, (L, len(movers)), list(to.items())


def beam(logits, score, groups, k, eos, fin=None):
    """candidates' c in f32 from an lse rounded once; the k largest, ties to the lowest b * V + v"""
    V = logits.shape[1]
    parent, token = np.full(groups * k, NONE, np.uint32), np.full(groups * k, NONE, np.uint32)
    out, fo = np.full(groups * k, -np.inf, np.float32), np.zeros(groups * k, np.uint32)
    with np.errstate(all="ignore"):
        for g in range(groups):
            c = np.full((k, V), -np.inf, np.float32)
            for b in range(k):
                r = g * k + b
                if fin is not None and fin[r]:
                    c[b, eos] = score[r]
                    continue
                x = logits[r].astype(np.float64)
                m = x.max()
                lse = np.float32(m + np.log(np.exp(x - m).sum())) if np.isfinite(m) else np.float32(np.nan)
                c[b] = score[r] + (logits[r] - lse)
            c[np.isnan(c)] = -np.inf
            c = c.reshape(-1) + np.float32(0)
            order = np.argsort(-c, kind="stable")[:k]
            for i, at in enumerate(order):
                if c[at] > -np.inf:
                    b, v = divmod(int(at), V)
                    s = g * k + i
                    parent[s], token[s], out[s] = g * k + b, v, c[at]
                    fo[s] = v == eos or (fin is not None and fin[g * k + b] != 0)
    return parent, token, out, fo
