// kv.cu -- the paged 4-bit cache around its attention: the host checks of a cache view, kv4Put / kv4Get (rows quantised
// into pages and read back) and kvStep / kvCompact (fork, reorder, extend, trim, free and compact the pages of a batch
// of sequences). No counterpart in the reference, whose caches are contiguous fp16 arrays of one stream each
// (engine/llm/gemma4.js:97-116).
#include "kv.cuh"
#include "launch.cuh"
#include "tc.cuh"

// ---------------------------------------------------------------- host checks
p0_status kv_view(p0_ctx *c, const p0_kv &kv, bool layer, const char *op, KvView *v) {
  if (!kv.rows || kv.rows > kKvMaxRows) return p0_fail(c, P0_EINVAL, "%s: %u sequences (1 to %u)", op, kv.rows, kKvMaxRows);
  if (!kv.pages || kv.pages > 0x7fffffffu) return p0_fail(c, P0_EINVAL, "%s: %u pages", op, kv.pages);
  if (!kv.table_ld || kv.table_ld > (1u << 23)) return p0_fail(c, P0_EINVAL, "%s: table rows of %u pages (1 to 2^23)", op, kv.table_ld);
  uint64_t part = 0, need = kv.page_stride;
  if (layer) {
    if (kv.D != 64 && kv.D != 128 && kv.D != 256 && kv.D != 512) return p0_fail(c, P0_EINVAL, "%s: D %u must be 64, 128, 256 or 512", op, kv.D);
    if (!kv.nkv || kv.nkv > 1024) return p0_fail(c, P0_EINVAL, "%s: %u KV heads (1 to 1024)", op, kv.nkv);
    part = (uint64_t)kv.D / 32 * 1280;
    need = kv.nkv * 2 * part;
  }
  const uint64_t stride = kv.page_stride ? kv.page_stride : need;
  if (!stride) return p0_fail(c, P0_EINVAL, "%s: the page stride is missing", op);
  if (stride < need) return p0_fail(c, P0_EINVAL, "%s: page stride %llu below the layer's %llu bytes", op, (unsigned long long)stride, (unsigned long long)need);
  if (stride > (1ull << 40)) return p0_fail(c, P0_EINVAL, "%s: page stride %llu", op, (unsigned long long)stride);
  if (kv.pages - 1 > (~0ull - need) / stride) return p0_fail(c, P0_EINVAL, "%s: %u pages of %llu bytes pass 64 bits", op, kv.pages, (unsigned long long)stride);
  P0Range rp, rt, rl;
  p0_status st;
  if ((st = p0_range(c, kv.pool, kv.pool_off, (uint64_t)(kv.pages - 1) * stride + need, op, "pool", &rp))) return st;
  if ((uintptr_t)rp.base % 16 || stride % 16) return p0_fail(c, P0_EALIGN, "%s: the pool's offset and page stride must be 16-byte aligned", op);
  if ((st = p0_range(c, kv.table, (uint64_t)kv.table_off * 4, (uint64_t)kv.rows * kv.table_ld * 4, op, "table", &rt))) return st;
  if ((st = p0_range(c, kv.len, (uint64_t)kv.len_off * 4, (uint64_t)kv.rows * 4, op, "len", &rl))) return st;
  if ((uintptr_t)rt.base % 4 || (uintptr_t)rl.base % 4) return p0_fail(c, P0_EALIGN, "%s: table and len must be 4-byte aligned", op);
  *v = KvView{rp.base, stride, (const uint32_t *)rt.base, (const uint32_t *)rl.base, nullptr, kv.table_ld, kv.pages, kv.rows, kv.nkv, kv.D, 0, 0};
  return P0_OK;
}

p0_status kv_new_tokens(p0_ctx *c, uint32_t n, uint32_t T, p0_buf cu, uint32_t cu_off, const char *op, KvView *v) {
  if (n > (1u << 28)) return p0_fail(c, P0_EINVAL, "%s: %u tokens in one call (at most 2^28)", op, n);   // positions stay well inside 32 bits
  v->n = n;
  v->T = T;
  if (cu.id) {
    P0Range r;
    p0_status st = p0_range(c, cu, (uint64_t)cu_off * 4, ((uint64_t)v->rows + 1) * 4, op, "cu", &r);
    if (st) return st;
    if ((uintptr_t)r.base % 4) return p0_fail(c, P0_EALIGN, "%s: cu must be 4-byte aligned", op);
    v->cu = (const uint32_t *)r.base;
    return P0_OK;
  }
  if (!T) return p0_fail(c, P0_EINVAL, "%s: T (new tokens per sequence) or cu is missing", op);
  if ((uint64_t)T * v->rows != n) return p0_fail(c, P0_EINVAL, "%s: n %u is not T %u x %u sequences", op, n, T, v->rows);
  return P0_OK;
}

p0_status kv_rows(p0_ctx *c, const p0_rows &r, uint32_t n, uint32_t heads, uint32_t D, uint32_t type, const char *op, const char *name, KvRows *out) {
  const uint64_t e = type == P0_F16 ? 2 : 4, ldh = r.ldh ? r.ldh : D, ld = r.ld ? r.ld : (uint64_t)heads * D;
  if (r.off > (1ull << 60)) return p0_fail(c, P0_EINVAL, "%s: %s offset", op, name);
  P0Range rr;
  p0_status st = p0_range(c, r.buf, r.off * e, ((uint64_t)(n - 1) * ld + (uint64_t)(heads - 1) * ldh + D) * e, op, name, &rr);
  if (st) return st;
  if ((uintptr_t)rr.base % e) return p0_fail(c, P0_EALIGN, "%s: %s must be aligned to its type", op, name);
  out->base = (uint8_t *)rr.base;
  out->ld = ld;
  out->ldh = ldh;
  out->wide = (uintptr_t)rr.base % 16 == 0 && ld * e % 16 == 0 && ldh * e % 16 == 0;
  return P0_OK;
}

namespace {

constexpr int kT = 256;

// ---------------------------------------------------------------- kv4Put / kv4Get
// A warp takes 8 consecutive tokens of one head's K or V and a run of its groups of 32 dims (a lane: one token's code word, 8
// dims), so that it finds the tokens' places once, reads or writes whole runs of 32 values and, where the tokens are
// neighbours in a page, 128 contiguous bytes of codes. 8192 tokens of 2 heads of 256: kv4Put of f32 13.6 us, 2.9 TB/s (f16, half the
// bytes read: 11.8), kv4Get to f16 6.7 us, 3.3 TB/s. kv4Put has 5 warps a scheduler (72 registers) and uses 53 % of the issue slots; of
// the cycles between a warp's instructions 36 % are waits for its loads, 20 % for the instruction before (places, extent, rounded
// division, codes: a chain). kv4Get: 51 % and 10 warps, half the cycles waits for loads. 8 tokens: 4.5 us each, the launch.
constexpr float kHold = 60000.0f;   // 15 * f16(range / 15) + f16(-60000) stays finite in f16
constexpr uint32_t kGroups = 4;     // groups whose values a lane holds at a time

struct RowsJob {
  KvView v;
  uint8_t *rec;         // the pool again, writable for kv4Put
  KvRows k, vv;
  uint32_t runs;        // of groups: warps per 8 tokens, head and K or V
  uint32_t warps;       // of the whole call
};

struct Place { uint32_t g0, g1, vsel, head, tok, word; bool in; };
__device__ __forceinline__ Place place_of(const RowsJob &j, uint32_t w) {
  const uint32_t lane = threadIdx.x & 31u, G = j.v.D / 32u;
  Place p;
  const uint32_t run = w % j.runs;
  p.g0 = G * run / j.runs;
  p.g1 = G * (run + 1) / j.runs;
  w /= j.runs;
  p.vsel = w & 1u;
  w >>= 1;
  p.head = w % j.v.nkv;
  w /= j.v.nkv;
  p.tok = w * 8u + (lane >> 2);
  p.word = lane & 3u;
  p.in = p.tok < j.v.n;
  return p;
}
// the first record of a place's token row, or null where the token has no page
__device__ __forceinline__ uint8_t *record_of(const RowsJob &j, const Place &p, uint32_t &slot) {
  uint32_t b, pos;
  if (!p.in || !kv_place(j.v, p.tok, b, pos)) return nullptr;
  const uint32_t page = j.v.table[(uint64_t)b * j.v.ld + pos / kPage];
  if (page >= j.v.pages) return nullptr;
  slot = pos % kPage;
  return j.rec + page * j.v.stride + (uint64_t)(p.head * 2u + p.vsel) * (j.v.D / 32u * 1280u);
}

template <bool F16, bool WIDE>
__device__ __forceinline__ void load8(const uint8_t *base, uint64_t at, float (&x)[8]) {
  if (F16) {
    const __half *h = reinterpret_cast<const __half *>(base) + at;
    if (WIDE) {
      const uint4 u = *reinterpret_cast<const uint4 *>(h);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = __half2float(h[i]);
    }
  } else {
    const float *f = reinterpret_cast<const float *>(base) + at;
    if (WIDE) {
      const float4 a = *reinterpret_cast<const float4 *>(f), b = *reinterpret_cast<const float4 *>(f + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = f[i];
    }
  }
}

// The codes clamp(rint(fl(d / s)), 0, 15) of 8 values d = fl(x - mn) as a word, with r = fl(1 / s). d * r is within three units in
// the last place of the quotient, so it rounds to the same whole number unless it lies next to a half, and then the divisions
// decide. d * r + 1.5 * 2^23 rounds it to a whole number, half to even, and holds that in its low bits; what the upper bits add up
// to, shifted, is taken off at the end.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float mn, float s, float r) {
  constexpr float kRound = 12582912.0f;
  constexpr uint32_t kBits = 0x4b400000u;   // of kRound
  uint32_t word = 0;
  float off = 0.0f;
#pragma unroll
  for (int e = 7; e >= 0; e--) {
    const float d = __fsub_rn(x[e], mn), t = __fmaf_rn(d, r, kRound);
    off = fmaxf(off, fabsf(__fmaf_rn(d, r, -__fsub_rn(t, kRound))));
    word = (word << 4) + __float_as_uint(fminf(fmaxf(t, kRound), kRound + 15.0f));
  }
  word -= kBits + (kBits << 4) + (kBits << 8);
  if (!(off <= 0.4999f)) {
    word = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) word |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e], mn), s)), 0.0f), 15.0f) << (4 * e);
  }
  return word;
}
// the smaller, the larger; NaN where one of them is
__device__ __forceinline__ float min_nan(float a, float b) {
  float c;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// per 32 dims: mn = f16(min), s = f16((max - mn) / 15) (0 -> 1), q = clamp(rhe((x - mn) / s), 0, 15), every step rounded
// in f32 as written (pack_q4 takes f64 for the division: a value on the border of two codes may land on the other)
template <bool F16, bool WIDE>
__global__ void __launch_bounds__(kT) kv4_put_kernel(RowsJob j) {
  dep_enter();
  const uint32_t w = blockIdx.x * (kT / 32) + threadIdx.x / 32u;
  if (w >= j.warps) return;
  const Place p = place_of(j, w);
  const KvRows &r = p.vsel ? j.vv : j.k;
  const uint64_t at = p.tok * r.ld + p.head * r.ldh + p.word * 8u;
  uint32_t slot = 0;
  uint8_t *rec = nullptr;
  for (uint32_t g0 = p.g0; g0 < p.g1; g0 += kGroups) {
    float x[kGroups][8] = {};
#pragma unroll
    for (uint32_t i = 0; i < kGroups; i++)   // on their way while the place is looked up
      if (p.in && g0 + i < p.g1) load8<F16, WIDE>(r.base, at + (g0 + i) * 32u, x[i]);
    if (g0 == p.g0) rec = record_of(j, p, slot);
#pragma unroll
    for (uint32_t i = 0; i < kGroups; i++) {
      if (g0 + i >= p.g1) break;
      float lo = x[i][0], hi = lo;
#pragma unroll
      for (int e = 1; e < 8; e++) {
        lo = min_nan(lo, x[i][e]);
        hi = max_nan(hi, x[i][e]);
      }
      if (!(lo >= -kHold && hi <= kHold)) {   // held at +-60000, NaN as 0
        lo = kHold;
        hi = -kHold;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x[i][e] = x[i][e] != x[i][e] ? 0.0f : fminf(fmaxf(x[i][e], -kHold), kHold);
          lo = fminf(lo, x[i][e]);
          hi = fmaxf(hi, x[i][e]);
        }
      }
      __syncwarp();
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {   // the four lanes of a token
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const __half mnh = __float2half_rn(lo + 0.0f);   // a minimum of -0 is stored as +0, whichever zero the reduction kept
      const float mn = __half2float(mnh);
      __half sh = __float2half_rn(__fdiv_rn(__fsub_rn(hi, mn), 15.0f));
      if (__half2float(sh) == 0.0f) sh = __float2half_rn(1.0f);
      const float s = __half2float(sh), inv = __frcp_rn(s);
      const uint32_t word = codes_of(x[i], mn, s, inv);
      if (rec) {
        uint8_t *to = rec + (g0 + i) * 1280u;
        *reinterpret_cast<uint32_t *>(to + slot * 16u + p.word * 4u) = word;
        if (p.word == 0)
          *reinterpret_cast<uint32_t *>(to + 1024u + slot * 4u) = (uint32_t)__half_as_ushort(sh) | ((uint32_t)__half_as_ushort(mnh) << 16);
      }
    }
  }
}

// the values of the same rows; a row without a page reads as zeros
template <bool F16, bool WIDE>
__global__ void __launch_bounds__(kT) kv4_get_kernel(RowsJob j) {
  dep_enter();
  const uint32_t w = blockIdx.x * (kT / 32) + threadIdx.x / 32u;
  if (w >= j.warps) return;
  const Place p = place_of(j, w);
  if (!p.in) return;
  const KvRows &r = p.vsel ? j.vv : j.k;
  uint32_t slot = 0;
  const uint8_t *rec = record_of(j, p, slot);
  for (uint32_t g0 = p.g0; g0 < p.g1; g0 += kGroups) {
    uint32_t word[kGroups] = {}, sm[kGroups] = {};
#pragma unroll
    for (uint32_t i = 0; i < kGroups; i++) {
      if (!rec || g0 + i >= p.g1) break;
      word[i] = *reinterpret_cast<const uint32_t *>(rec + (g0 + i) * 1280u + slot * 16u + p.word * 4u);
      sm[i] = *reinterpret_cast<const uint32_t *>(rec + (g0 + i) * 1280u + 1024u + slot * 4u);
    }
#pragma unroll
    for (uint32_t i = 0; i < kGroups; i++) {
      if (g0 + i >= p.g1) break;
      const uint32_t s2 = __byte_perm(sm[i], 0, 0x1010), mn2 = __byte_perm(sm[i], 0, 0x3232), y = word[i] >> 4;
      const uint32_t v[4] = {kv_deq2(__byte_perm(word[i], y, 0x4400), s2, mn2), kv_deq2(__byte_perm(word[i], y, 0x5511), s2, mn2),   // byte i: 2i, 2i + 1
                             kv_deq2(__byte_perm(word[i], y, 0x6622), s2, mn2), kv_deq2(__byte_perm(word[i], y, 0x7733), s2, mn2)};
      const uint64_t at = p.tok * r.ld + p.head * r.ldh + (g0 + i) * 32u + p.word * 8u;
      if (F16) {
        __half *h = reinterpret_cast<__half *>(r.base) + at;
        if (WIDE) *reinterpret_cast<uint4 *>(h) = make_uint4(v[0], v[1], v[2], v[3]);
        else
#pragma unroll
          for (int e = 0; e < 8; e++) h[e] = __ushort_as_half((unsigned short)(v[e / 2] >> (16 * (e & 1))));
      } else {
        float *f = reinterpret_cast<float *>(r.base) + at;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __half2float(__ushort_as_half((unsigned short)(v[e / 2] >> (16 * (e & 1)))));
        if (WIDE) {
          *reinterpret_cast<float4 *>(f) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4 *>(f + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else
#pragma unroll
          for (int e = 0; e < 8; e++) f[e] = x[e];
      }
    }
  }
}

// ---------------------------------------------------------------- kvStep / kvCompact: the plans
// One cluster of kPC CTAs plans a call in phases with cluster barriers between them; the page copies follow in a second
// kernel from the list that the plan leaves in the workspace. Counts are integer sums, so their order does not matter.
// 64 sequences of 9000 tokens, 26 layers (16 MB of tails): 12.9 us; 8 small ones: 6.2 us, of which two
// launches are most. Compacting 160 MB of pages: 59 us, 51 of them the copies at the copy rate.
constexpr uint32_t kPC = 8, kPT = 1024;
constexpr uint32_t kNone = P0_KV_NONE;
// One CTA plans a step, the counts in shared memory, where no thread has more than a few entries: 8 sequences of 3011 tokens, 200
// pages: 6.3 us, by a cluster 9.2; 16 of 20000, 3000 pages: 10.4 and 10.2; 64 of 9000, 2300 pages: 15.4 and 13.6
constexpr uint32_t kOnePages = 4096, kOneEntries = 4096;

__device__ __forceinline__ uint32_t plan_tid() { return blockIdx.x * kPT + threadIdx.x; }

// inclusive sum over the CTA's threads; every thread gets the total too
__device__ __forceinline__ uint32_t cta_scan(uint32_t v, uint32_t *red, uint32_t &total) {
  const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= (uint32_t)o) v += u;
  }
  __syncthreads();
  if (lane == 31u) red[w] = v;
  __syncthreads();
  if (w == 0) {
    uint32_t t = red[lane];   // kPT / 32 = 32 warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= (uint32_t)o) t += u;
    }
    red[lane] = t;
  }
  __syncthreads();
  total = red[31];
  return v + (w ? red[w - 1] : 0u);
}

struct StepJob {
  KvView v;
  const uint32_t *ref, *parent, *add;
  uint32_t addn, window, sinks;
  uint32_t *to_table, *to_len, *to_ref, *stat;
  uint32_t *cnt;        // [kPC] free pages of each CTA's share
  uint2 *list;          // [rows] (source, destination) page of each row's tail copy, or (none, none)
};

// page j of a row of length n lies wholly outside the window of every later token and behind the sinks
__device__ __forceinline__ bool page_dead(uint32_t j, uint32_t n, uint32_t window, uint32_t sinks) {
  const uint64_t first = (uint64_t)j * kPage;
  return window && first + kPage - 1 + window <= n && first >= sinks;
}

// NC CTAs: one, which keeps the counts in shared memory, where the state is small, or a cluster
template <uint32_t NC>
__device__ __forceinline__ void step_plan(const StepJob &j) {
  dep_enter();
  // per row: the parent (kNone: an empty row), its length, the new length, and (first needed page rank << 1 | copies
  // its tail)
  extern __shared__ uint32_t sm[];
  const uint32_t R = j.v.rows, ld = j.v.ld, P = j.v.pages;
  uint32_t *par = sm, *lp = sm + R, *to = sm + 2 * R, *want = sm + 3 * R, *first = sm + 4 * R;
  uint32_t *rc = NC == 1 ? sm + 5 * R : j.to_ref;   // the counts as they become
  __shared__ uint32_t red[32], too_long;
  const uint32_t tid = plan_tid(), all = NC * kPT;
  const auto meet = [] {
    if (NC == 1) __syncthreads();
    else tc::cluster_sync();
  };
  const auto count = [&](uint32_t p) { return NC == 1 ? rc[p] : __ldcg(&rc[p]); };
  for (uint32_t p = tid; p < P; p += all) rc[p] = j.ref[p];
  if (threadIdx.x == 0) too_long = 0u;
  for (uint32_t i = threadIdx.x; i < R; i += kPT) first[i] = kNone;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < R; i += kPT) {
    const uint32_t p = j.parent ? j.parent[i] : i;
    const bool ok = p < R;
    const uint32_t n = ok ? kv_len(j.v, p) : 0u, a = ok ? (j.add ? j.add[i] : j.addn) : 0u;
    if ((uint64_t)n + a > (uint64_t)ld * kPage) atomicOr(&too_long, 1u);
    par[i] = ok ? p : kNone;
    lp[i] = n;
    to[i] = n + a;
    if (ok) atomicMin(&first[p], i);
  }
  __syncthreads();
  uint32_t total = 0;
  {
    uint32_t w = 0, copies = 0;
    const uint32_t i = threadIdx.x;   // R <= kPT: a thread per row
    if (i < R && par[i] != kNone && !too_long) {
      const uint32_t t = lp[i] / kPage;
      if (lp[i] % kPage && first[par[i]] != i && !page_dead(t, lp[i], j.window, j.sinks)) copies = j.v.table[(uint64_t)par[i] * ld + t] < P;
      w = copies + (to[i] + kPage - 1) / kPage - (lp[i] + kPage - 1) / kPage;
    }
    const uint32_t incl = cta_scan(w, red, total);
    if (i < R) want[i] = (incl - w) << 1 | copies;
  }
  meet();   // rc holds the old counts
  // the table without the new pages, and the counts that follow from it: an entry that a row keeps in place changes
  // nothing. Old entries beyond a length (it may have been lowered) are references as well, and end here
  for (uint64_t e = tid; e < (uint64_t)R * ld; e += all) {
    const uint32_t i = (uint32_t)e / ld, p = (uint32_t)e - i * ld;
    uint32_t a = j.v.table[e], b = kNone;
    if (a >= P) a = kNone;
    if (par[i] != kNone && p < (lp[i] + kPage - 1) / kPage) {
      b = j.v.table[(uint64_t)par[i] * ld + p];
      if (b >= P || page_dead(p, lp[i], j.window, j.sinks) || ((want[i] & 1u) && p == lp[i] / kPage)) b = kNone;
    }
    if (a != b) {
      if (a != kNone) atomicSub(&rc[a], 1u);
      if (b != kNone) atomicAdd(&rc[b], 1u);
    }
    j.to_table[e] = b;
  }
  meet();
  // free pages: each CTA counts its share, then gives out the lowest ones in the order of the rows' needs
  const uint32_t per = (P + NC - 1) / NC, lo = min(P, blockIdx.x * per), hi = min(P, lo + per);
  uint32_t mine = 0;
  for (uint32_t p = lo + threadIdx.x; p < hi; p += kPT) mine += count(p) == 0u;
  uint32_t share;
  cta_scan(mine, red, share);
  uint32_t before = 0, left = share;
  if (NC > 1) {
    if (threadIdx.x == 0) j.cnt[blockIdx.x] = share;
    meet();
    left = 0;
    for (uint32_t k = 0; k < NC; k++) {
      const uint32_t s = __ldcg(&j.cnt[k]);
      if (k < blockIdx.x) before += s;
      left += s;
    }
  }
  const bool ok = !too_long && total <= left;
  if (!ok) {   // all or nothing: the state as it was
    for (uint64_t e = tid; e < (uint64_t)R * ld; e += all) j.to_table[e] = j.v.table[e];
    uint32_t was = 0;
    for (uint32_t p = tid; p < P; p += all) j.to_ref[p] = j.ref[p];
    for (uint32_t i = tid; i < R; i += all) {
      j.to_len[i] = j.v.len[i];
      j.list[i] = make_uint2(kNone, kNone);
    }
    if (blockIdx.x == 0) {
      for (uint32_t p = threadIdx.x; p < P; p += kPT) was += j.ref[p] == 0u;
      uint32_t sum;
      cta_scan(was, red, sum);
      if (threadIdx.x == 0) {
        j.stat[0] = too_long ? kNone : total - left;
        j.stat[1] = sum;
      }
    }
    return;
  }
  for (uint32_t i = tid; i < R; i += all) {
    j.to_len[i] = to[i];
    if (!(want[i] & 1u)) j.list[i] = make_uint2(kNone, kNone);
  }
  if (tid == 0) {
    j.stat[0] = 0u;
    j.stat[1] = left - total;
  }
  for (uint32_t p0 = lo; p0 < hi && before < total; p0 += kPT) {
    const uint32_t p = p0 + threadIdx.x;
    const bool fr = p < hi && count(p) == 0u;
    uint32_t here;
    const uint32_t k = before + cta_scan(fr ? 1u : 0u, red, here) - 1u;
    if (fr && k < total) {
      uint32_t a = 0, b = R;   // the last row whose first rank is <= k: ranks of rows without needs repeat the next one's
      while (b - a > 1) {
        const uint32_t m = (a + b) >> 1;
        if ((want[m] >> 1) <= k) a = m; else b = m;
      }
      uint32_t at = k - (want[a] >> 1);
      if (want[a] & 1u) {
        if (at == 0) j.list[a] = make_uint2(j.v.table[(uint64_t)par[a] * ld + lp[a] / kPage], p);
        at = at == 0 ? lp[a] / kPage : (lp[a] + kPage - 1) / kPage + at - 1;
      } else {
        at += (lp[a] + kPage - 1) / kPage;
      }
      j.to_table[(uint64_t)a * ld + at] = p;
      rc[p] = 1u;
    }
    before += here;
  }
  if (NC == 1) {
    __syncthreads();
    for (uint32_t p = tid; p < P; p += all) j.to_ref[p] = rc[p];
  }
}

__global__ void __launch_bounds__(kPT) kv_step_plan_one(StepJob j) { step_plan<1>(j); }
__global__ void __cluster_dims__(kPC, 1, 1) __launch_bounds__(kPT) kv_step_plan(StepJob j) { step_plan<kPC>(j); }

struct CompactJob {
  KvView v;
  const uint32_t *ref;
  uint32_t *to_table, *to_ref, *stat;
  uint32_t *cnt;        // [kPC] live pages of each CTA's share, then the live pages below L
  uint32_t *live, *hole, *rank;   // [pages] each: the k-th live page, the k-th free page below L; of a page, the live pages before it
};

// L live pages: the k-th live page at L or beyond moves to the k-th free page below L. With f(p) = the live pages before p,
// a free page p < L is the (p - f(p))-th hole, and a live page p >= L the (f(p) - f(L))-th to move: one scan gives both.
// A CTA takes a run of the pages, a thread a run of those
__global__ void __cluster_dims__(kPC, 1, 1) __launch_bounds__(kPT) kv_compact_plan(CompactJob j) {
  dep_enter();
  __shared__ uint32_t red[32];
  const uint32_t P = j.v.pages, tid = plan_tid(), all = kPC * kPT;
  const uint32_t per = (P + all - 1) / all, lo = min((uint64_t)P, (uint64_t)tid * per), hi = min(P, lo + per);
  uint32_t n = 0, sum;
  for (uint32_t p = lo; p < hi; p++) n += j.ref[p] != 0u;
  uint32_t f = cta_scan(n, red, sum) - n;
  if (threadIdx.x == 0) j.cnt[blockIdx.x] = sum;
  tc::cluster_sync();
  uint32_t L = 0;
  for (uint32_t k = 0; k < kPC; k++) {
    const uint32_t c = __ldcg(&j.cnt[k]);
    if (k < blockIdx.x) f += c;
    L += c;
  }
  for (uint32_t p = lo; p < hi; p++) {
    if (p == L) j.cnt[kPC] = f;
    j.rank[p] = f;
    if (j.ref[p]) j.live[f++] = p;
    else if (p < L) j.hole[p - f] = p;
  }
  if (tid == 0 && L == P) j.cnt[kPC] = L;
  tc::cluster_sync();
  const uint32_t fL = __ldcg(&j.cnt[kPC]);
  for (uint64_t e = tid; e < (uint64_t)j.v.rows * j.v.ld; e += all) {
    uint32_t p = j.v.table[e];
    if (p < P && p >= L && j.ref[p]) p = __ldcg(&j.hole[__ldcg(&j.rank[p]) - fL]);
    j.to_table[e] = p;
  }
  for (uint32_t p = tid; p < P; p += all) {
    uint32_t r = 0;
    if (p < L) r = j.ref[p] ? j.ref[p] : j.ref[__ldcg(&j.live[fL + p - __ldcg(&j.rank[p])])];
    j.to_ref[p] = r;
  }
  if (tid == 0) {
    j.stat[0] = L;
    j.stat[1] = L - fL;
  }
}

// ---------------------------------------------------------------- page copies
// kvStep: CTA (x, i) copies its 16-byte words of row i's tail page
constexpr uint32_t kCopyT = 256, kCopyU = 4;   // 16 KB per CTA and pass
__device__ __forceinline__ void copy_run(const uint4 *__restrict__ s, uint4 *__restrict__ d, uint64_t n) {
  uint4 u[kCopyU];
#pragma unroll
  for (uint32_t k = 0; k < kCopyU; k++)
    if (threadIdx.x + k * kCopyT < n) u[k] = __ldcs(s + threadIdx.x + k * kCopyT);
#pragma unroll
  for (uint32_t k = 0; k < kCopyU; k++)
    if (threadIdx.x + k * kCopyT < n) __stcs(d + threadIdx.x + k * kCopyT, u[k]);
}
__global__ void __launch_bounds__(kCopyT) kv_copy_tails(uint8_t *pool, uint64_t stride, const uint2 *__restrict__ list) {
  dep_enter();
  const uint2 m = list[blockIdx.y];
  if (m.x == kNone) return;
  const uint64_t n = stride / 16, at = (uint64_t)blockIdx.x * kCopyT * kCopyU;
  copy_run(reinterpret_cast<const uint4 *>(pool + m.x * stride) + at, reinterpret_cast<uint4 *>(pool + m.y * stride) + at, n - at);
}
// kvCompact: the moves' runs of 16 KB dealt to a grid of fixed size (the host does not know the number of moves)
__global__ void __launch_bounds__(kCopyT) kv_copy_moves(uint8_t *pool, uint64_t stride, const uint32_t *__restrict__ cnt,
                                                        const uint32_t *__restrict__ live, const uint32_t *__restrict__ hole) {
  dep_enter();
  uint32_t L = 0;
  for (uint32_t k = 0; k < kPC; k++) L += cnt[k];
  const uint32_t *mover = live + cnt[kPC];
  const uint64_t n = stride / 16, runs = (n + kCopyT * kCopyU - 1) / (kCopyT * kCopyU), all = runs * (L - cnt[kPC]);
  for (uint64_t r = blockIdx.x; r < all; r += gridDim.x) {
    const uint64_t k = r / runs, at = r % runs * (kCopyT * kCopyU);
    copy_run(reinterpret_cast<const uint4 *>(pool + mover[k] * stride) + at, reinterpret_cast<uint4 *>(pool + hole[k] * stride) + at, n - at);
  }
}

p0_status rows_call(p0_ctx *c, const p0_kv4_rows_args *a, bool put) {
  if (!c || !a) return P0_EINVAL;
  const char *op = put ? "kv4Put" : "kv4Get";
  if (a->type > P0_F16) return p0_fail(c, P0_EINVAL, "%s: type %u", op, a->type);
  if (!a->n) return P0_OK;
  RowsJob j;
  p0_status st;
  if ((st = kv_view(c, a->kv, true, op, &j.v))) return st;
  if ((st = kv_new_tokens(c, a->n, a->T, a->cu, a->cu_off, op, &j.v))) return st;
  if ((st = kv_rows(c, a->k, a->n, a->kv.nkv, a->kv.D, a->type, op, "k", &j.k))) return st;
  if ((st = kv_rows(c, a->v, a->n, a->kv.nkv, a->kv.D, a->type, op, "v", &j.vv))) return st;
  j.rec = const_cast<uint8_t *>(j.v.pool);
  // a warp takes four groups; where there are few tokens, one
  const uint64_t eights = (uint64_t)((a->n + 7) / 8) * a->kv.nkv * 2, G = a->kv.D / 32;
  j.runs = (uint32_t)(eights < 8u * (uint32_t)c->sm_count ? G : (G + kGroups - 1) / kGroups);
  const uint64_t warps = eights * j.runs, grid = (warps + kT / 32 - 1) / (kT / 32);
  j.warps = (uint32_t)warps;
  if (warps > 0xffffff00u) return p0_fail(c, P0_EINVAL, "%s: %u tokens in one call", op, a->n);
  const bool f16 = a->type == P0_F16, wide = j.k.wide && j.vv.wide;
  cudaSetDevice(c->device);
  auto go = [&](auto kern) { launch_dep(kern, dim3((unsigned)grid), dim3(kT), 0, c->stream, j); };
  if (put) f16 ? (wide ? go(kv4_put_kernel<true, true>) : go(kv4_put_kernel<true, false>))
               : (wide ? go(kv4_put_kernel<false, true>) : go(kv4_put_kernel<false, false>));
  else f16 ? (wide ? go(kv4_get_kernel<true, true>) : go(kv4_get_kernel<true, false>))
           : (wide ? go(kv4_get_kernel<false, true>) : go(kv4_get_kernel<false, false>));
  return p0_launched(c, op);
}

// a bound range of u32, 4-byte aligned
p0_status words(p0_ctx *c, p0_buf b, uint64_t n, const char *op, const char *name, uint32_t **out, bool optional = false) {
  P0Range r;
  p0_status st = p0_range(c, b, 0, n * 4, op, name, &r, optional);
  if (st) return st;
  if ((uintptr_t)r.base % 4) return p0_fail(c, P0_EALIGN, "%s: %s must be 4-byte aligned", op, name);
  *out = (uint32_t *)r.base;
  return P0_OK;
}
bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + nb * 4 && y < x + na * 4;
}

}  // namespace

extern "C" {

p0_status p0_kv4_put(p0_ctx *c, const p0_kv4_rows_args *a) { return rows_call(c, a, true); }
p0_status p0_kv4_get(p0_ctx *c, const p0_kv4_rows_args *a) { return rows_call(c, a, false); }

p0_status p0_kv_step(p0_ctx *c, const p0_kv_step_args *a) {
  if (!c || !a) return P0_EINVAL;
  const char *op = "kvStep";
  StepJob j;
  p0_status st;
  if ((st = kv_view(c, a->kv, false, op, &j.v))) return st;
  const uint64_t R = a->kv.rows, E = R * a->kv.table_ld, P = a->kv.pages;
  if (E > 0xffffffffull) return p0_fail(c, P0_EINVAL, "%s: a table of %llu entries", op, (unsigned long long)E);
  uint32_t *ref, *parent, *add;
  if ((st = words(c, a->ref, P, op, "ref", &ref))) return st;
  if ((st = words(c, a->parent, R, op, "parent", &parent, true))) return st;
  if ((st = words(c, a->add, R, op, "add", &add, true))) return st;
  if ((st = words(c, a->to_table, E, op, "to.table", &j.to_table))) return st;
  if ((st = words(c, a->to_len, R, op, "to.len", &j.to_len))) return st;
  if ((st = words(c, a->to_ref, P, op, "to.ref", &j.to_ref))) return st;
  if ((st = words(c, a->stat, 2, op, "stat", &j.stat))) return st;
  if (overlap(j.to_table, E, j.v.table, E) || overlap(j.to_len, R, j.v.len, R) || overlap(j.to_ref, P, ref, P))
    return p0_fail(c, P0_EINVAL, "%s: the new state must not lie over the old one", op);
  j.ref = ref;
  j.parent = parent;
  j.add = add;
  j.addn = a->addn;
  j.window = a->window;
  j.sinks = a->sinks;
  uint32_t *cnt;
  void *ws;
  cudaSetDevice(c->device);
  if ((st = p0_workspace(c, 0, 256 + R * sizeof(uint2), &cnt, &ws))) return st;
  j.cnt = (uint32_t *)ws;
  j.list = (uint2 *)((uint8_t *)ws + 256);
  if (P <= kOnePages && E <= kOneEntries) launch_dep(kv_step_plan_one, dim3(1), dim3(kPT), (size_t)(R * 5 + P) * 4, c->stream, j);
  else launch_dep(kv_step_plan, dim3(kPC), dim3(kPT), (size_t)R * 5 * 4, c->stream, j);
  if ((st = p0_launched(c, op))) return st;
  if (!parent) return P0_OK;   // without parents no row has a second child: there is nothing to copy
  const uint64_t runs = (j.v.stride / 16 + kCopyT * kCopyU - 1) / (kCopyT * kCopyU);
  if (runs > 0x7fffffffu) return p0_fail(c, P0_EINVAL, "%s: page stride %llu", op, (unsigned long long)j.v.stride);
  launch_dep(kv_copy_tails, dim3((unsigned)runs, (unsigned)R), dim3(kCopyT), 0, c->stream, const_cast<uint8_t *>(j.v.pool), j.v.stride, (const uint2 *)j.list);
  return p0_launched(c, "kvStep copy");
}

p0_status p0_kv_compact(p0_ctx *c, const p0_kv_compact_args *a) {
  if (!c || !a) return P0_EINVAL;
  const char *op = "kvCompact";
  CompactJob j;
  p0_status st;
  if ((st = kv_view(c, a->kv, false, op, &j.v))) return st;
  const uint64_t E = (uint64_t)a->kv.rows * a->kv.table_ld, P = a->kv.pages;
  if (E > 0xffffffffull) return p0_fail(c, P0_EINVAL, "%s: a table of %llu entries", op, (unsigned long long)E);
  uint32_t *ref;
  if ((st = words(c, a->ref, P, op, "ref", &ref))) return st;
  if ((st = words(c, a->to_table, E, op, "to.table", &j.to_table))) return st;
  if ((st = words(c, a->to_ref, P, op, "to.ref", &j.to_ref))) return st;
  if ((st = words(c, a->stat, 2, op, "stat", &j.stat))) return st;
  if (overlap(j.to_table, E, j.v.table, E) || overlap(j.to_ref, P, ref, P))
    return p0_fail(c, P0_EINVAL, "%s: the new state must not lie over the old one", op);
  j.ref = ref;
  uint32_t *cnt;
  void *ws;
  cudaSetDevice(c->device);
  if ((st = p0_workspace(c, 0, 256 + P * 12, &cnt, &ws))) return st;
  j.cnt = (uint32_t *)ws;
  j.live = (uint32_t *)((uint8_t *)ws + 256);
  j.hole = j.live + P;
  j.rank = j.hole + P;
  launch_dep(kv_compact_plan, dim3(kPC), dim3(kPT), 0, c->stream, j);
  if ((st = p0_launched(c, op))) return st;
  launch_dep(kv_copy_moves, dim3((unsigned)c->sm_count * 8u), dim3(kCopyT), 0, c->stream, const_cast<uint8_t *>(j.v.pool), j.v.stride,
             (const uint32_t *)j.cnt, (const uint32_t *)j.live, (const uint32_t *)j.hole);
  return p0_launched(c, "kvCompact copy");
}

}  // extern "C"
