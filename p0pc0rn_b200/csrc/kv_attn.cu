// kv_attn.cu -- kv4Attn: attention of each sequence's newest tokens over its paged 4-bit cache (causal; whole context, or
// a sliding window with the first `sinks` tokens kept visible). No counterpart in the reference, whose attnDec takes one
// token over a contiguous fp16 cache (engine/llm/lops.js:236-321).
//
//   o_i = sum_j p_ij v_j,  p_i = softmax over the visible j of scale * (q_i . k_j),  k, v = f16(q * s + mn)
//   visible: j <= pos_i and (window = 0 or j > pos_i - window or j < sinks);  nothing visible: o_i = 0
//
// Work is cut as kv_attn.cuh says: the pages that row blocks see, in order, in equal runs, one per CTA, from the lengths on
// the device: long and short sequences, windows and empty slots fill the GPU alike. A unit that lies in one run is
// finished there; otherwise each run leaves (m, l, acc) in the workspace and the join kernel adds them in run order, so
// results do not depend on timing.
//
// An item, one or two pages: bulk copies bring a head's K and V records to shared memory, a ring of stages hides them. K records
// lie 1312 bytes apart there, so that a quarter warp's 16-byte reads of four records fall in different banks. The codes
// become f16 pairs in registers (kv_deq8) and go straight into mma.sync fragments without moves: any order of the dims
// serves a dot product, so a lane takes 32 dims of one group of a key (q is staged in that order): one 16-byte read and
// one (s, mn) for 32 codes; two keys' V words give 8 (key, key + 1) pairs by two byte permutes.
//   S = Q K^T   a warp takes 8 or 16 of the item's keys
//   P = exp(S - m) through shared memory, m over all warps
//   O += P V    a warp takes 64 (or 32) dims and a share of the keys; the shares meet when the unit ends
// A batch of long contexts is bound by the instructions per code, about 2 for each of K and V (3500 warp instructions a page of 256
// dims, 2.2 a cycle), and by what 16 warps an SM, as many as their registers allow, leave of the issue slots: the two barriers an
// item are a quarter of the cycles between a warp's instructions. 32 contexts up to 65500 keys, 8 f32 heads on one of 256: 114 us,
// 3.1 TB/s of records, 56 % of the issue slots. Small calls are two launches, with grids for the whole GPU, and their latencies: 8
// contexts in a window of 512, 11.7 us. 4 x 8 tokens, 8190 keys, 8 f32 heads on 2 of 512: 55 us.
//
// Precision. f32 queries and outputs: q and P are split into f16 high and low parts (about 22 bits) in rows r and r + 8
// of the fragments; a row of q is brought to [2^14, 2^15) by a power of two first, which its scores give back, so that
// neither part leaves f16's range for any f32 q; P is held as 2^15 P, as its sum l is, for the same reason: parts that f16
// does not hold lie below 2^-40 (P <= 1), and a long tail of small P counts in the output as it does in l; each item's P V is summed from zero and added in f32. f16: q as it is, P rounded to f16 once (as any
// f16 matrix operand; as 2^15 P, too), 16 rows per fragment.
#include <cstdlib>

#include "kv_attn.cuh"

namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same from zero
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t lds_u32(const uint8_t *p) { return *reinterpret_cast<const uint32_t *>(p); }

// The power of two that brings a row whose largest |q| has these bits to [2^14, 2^15), and its inverse; rows below 2^-112
// as if they reached it, so that both are normal numbers
__device__ __forceinline__ float row_up(uint32_t bits) { return __uint_as_float((268u - max(bits >> 23, 15u)) << 23); }
__device__ __forceinline__ float row_down(uint32_t bits) { return __uint_as_float((max(bits >> 23, 15u) - 14u) << 23); }

constexpr float kPUp = 32768.0f;   // P in [0, 1] uses f16's whole range
constexpr uint32_t kRec = 1312;   // a K record's place in shared memory

template <int D, bool F32, int NPL, int RT, int KP, int NW>
struct Cfg {
  static constexpr int kThreads = NW * 32;
  static constexpr int kRowsPer = F32 ? 8 : 16;          // query rows per fragment
  static constexpr int kRows = kRowsPer * RT;            // of a block
  static constexpr int kNt = 8 * KP / NW;               // 8-key tiles per warp in Q K^T
  static constexpr int kDs = D / (8 * NPL);              // warps over the dims in P V (NPL dims a lane and key),
  static constexpr int kKs = NW / kDs;                  // and over the keys
  static constexpr int kSteps = KP * 4 / kKs;            // 16-key steps per warp
  static constexpr uint32_t kRecs = D / 32, kPart = kRecs * 1280, kK = kRecs * kRec, kPage2 = kK + kPart;   // K and V of a page
  static constexpr uint32_t kStage = KP * kPage2;
  static constexpr int kStages = D >= 256 ? 2 : 3;
  static constexpr uint32_t kQ = RT * D / 16 * 512;      // q fragments
  static constexpr uint32_t kPRow = 64 * KP * 2 + 16;    // a row of P, padded against bank conflicts
  static constexpr uint32_t kP = RT * 16 * kPRow;
  static constexpr uint32_t kSmem = kStages * kStage + kQ + kP;
  static_assert(kKs == 1 || (uint32_t)(RT * D * 64) <= kStages * kStage, "the key shares meet in the ring");
};

template <int D, bool F32, int NPL, int RT, int KP, int NW>
__global__ void __launch_bounds__(NW * 32, RT > 1 ? 1 : 16 / NW) kv4_attn_kernel(AttnJob j, uint32_t polls) {
  dep_enter();
  using C = Cfg<D, F32, NPL, RT, KP, NW>;
  constexpr int NT = C::kNt, RR = C::kRowsPer, RB = C::kRows, NS = C::kStages;
  constexpr int KW = D >= 128 ? 4 : 2;   // a lane's K words at a time: of one group (D = 64: half of one)
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t *ring = smem;
  uint4 *qf = reinterpret_cast<uint4 *>(smem + NS * C::kStage);
  uint8_t *ps = smem + NS * C::kStage + C::kQ;
  uint32_t *pre = reinterpret_cast<uint32_t *>(smem + C::kSmem);   // [rows + 1] items before each sequence
  __shared__ __align__(8) uint64_t full[NS];
  __shared__ uint32_t abort_flag, page_ok[NS][KP];
  __shared__ __align__(16) float wmax[RB][NW], wsum[RB][NW];
  __shared__ int32_t rpos[RB];
  __shared__ uint32_t qmax[RB];   // f32: the largest |q| of a row, as bits
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g4 = lane >> 2, t4 = lane & 3u;
  const uint32_t hpg = j.hpg, R = j.v.rows, W = j.window, S = j.sinks;
  if (tid == 0) {
    for (int i = 0; i < NS; i++) tc::mbar_init(&full[i], 1);
    abort_flag = 0u;
    tc::fence_mbar_init();
  }
  if (F32 && tid < (uint32_t)RB) qmax[tid] = 0u;
  plan_items<RB, KP, 0>(j, pre);
  const uint32_t total = pre[R], G = min(gridDim.x, max(total, 1u));   // no run is empty
  if (tid == 0) j.desc[blockIdx.x] = make_uint4(0u, 0u, 0u, 0u);
  if (blockIdx.x >= G) return;
  const uint32_t lo = (uint32_t)((uint64_t)total * blockIdx.x / G), hi = (uint32_t)((uint64_t)total * (blockIdx.x + 1) / G);
  uint32_t b = find_sequence(pre, R, lo);
  const float log2_scale = j.scale * 1.44269504088896340736f;   // f16: scores and maxima in powers of two
  const auto ex = [](float x) { return exp2_fast(F32 ? x * 1.44269504088896340736f : x); };
  uint32_t at = lo, it = 0, started = 0;   // item; items through the ring so far; items whose copies were started (warp 0's)
  while (at < hi) {
    while (pre[b + 1] <= at) b++;
    const Unit u = find_unit<RB, KP, 0>(j, pre, b, at);
    const Span &s = u.s;
    const uint32_t first = u.first, T = u.T, len = u.len, rows = u.rows, r0 = u.r0, head = u.head, begin = u.begin, n = u.n;
    const uint32_t from = at - begin, to = min(hi - begin, n);
    const uint32_t nrow = min((uint32_t)RB, rows - r0);
    const uint32_t steps = s.n ? to - from : 0u;
    const uint8_t *heads = j.v.pool + (uint64_t)head * 2u * C::kPart;
    // warp 0 brings an item's records, a K record or a page's V a lane; it looks an item's pages up one item ahead
    constexpr uint32_t PR = C::kRecs + 1;
    static_assert(KP * PR <= 32, "a lane per copy");
    const uint32_t ck = lane / PR, cr = lane % PR;
    const auto look_up = [&](uint32_t i) {   // the page that this lane copies from for item from + i of the unit
      const uint32_t pi = (from + i) * KP + ck;
      return ck < (uint32_t)KP && i < steps && pi < s.n ? j.v.table[(uint64_t)b * j.v.ld + page_at(s, pi)] : P0_KV_NONE;
    };
    uint32_t ahead = P0_KV_NONE;
    const auto issue = [&](uint32_t i) {
      if (__any_sync(0xffffffffu, *(volatile uint32_t *)&abort_flag)) return;   // the slot's last copies may still be on their way
      started = it + i + 1u;
      const uint32_t st = (it + i) % NS, p = ahead;
      const bool have = p < j.v.pages;
      const uint32_t n_k = __popc(__ballot_sync(0xffffffffu, have && cr < C::kRecs)), n_v = __popc(__ballot_sync(0xffffffffu, have && cr == C::kRecs));
      if (cr == 0 && ck < (uint32_t)KP) page_ok[st][ck] = have;
      __syncwarp();
      if (lane == 0) {
        if (n_k) tc::mbar_expect_tx(&full[st], n_k * 1280u + n_v * C::kPart);
        else tc::mbar_arrive(&full[st]);   // no such pages: their keys are not there
      }
      __syncwarp();
      if (have)
        bulk_load(ring + st * C::kStage + ck * C::kPage2 + cr * kRec, heads + p * j.v.stride + cr * 1280u, cr < C::kRecs ? 1280u : C::kPart, &full[st]);
      ahead = look_up(i + 1);
    };
    if (warp == 0) {
      ahead = look_up(0);
      for (uint32_t i = 0; i < (uint32_t)NS && i < steps; i++) issue(i);
    }
    // the rows' positions and q fragments
    if (tid < (uint32_t)RB) rpos[tid] = tid < nrow ? (int32_t)(len - T + (r0 + tid) / hpg) : -1;
    {
      constexpr uint32_t all = RT * (D / 16) * 32, E = (all + C::kThreads - 1) / C::kThreads, H = F32 ? 1 : 2;   // a thread's, all on their way before one is used
      const bool wide = j.q.wide;
      uint2 x[E][H][2];   // dims d0, + 1 and + 4, + 5 (f16: the low words)
#pragma unroll
      for (uint32_t i = 0; i < E; i++) {
        const uint32_t e = i * C::kThreads + tid, ln = e & 31u, step = (e >> 5) % (D / 16), rt = (e >> 5) / (D / 16);
        const uint32_t wi = step >> 1, l4 = ln & 3u;   // the lane's K word wi; its codes d0, +4, +1, +5
        const uint32_t d0 = (D >= 128 ? ((wi >> 2) * 4u + l4) * 32u + (wi & 3u) * 8u : l4 * 16u + wi * 8u) + (step & 1u) * 2u;
#pragma unroll
        for (uint32_t half = 0; half < H; half++) {
          const uint32_t r = rt * RR + (ln >> 2) + 8u * half, tok = (r0 + r) / hpg;
          x[i][half][0] = x[i][half][1] = make_uint2(0u, 0u);
          if (r >= nrow || e >= all) continue;
          const uint64_t o = (uint64_t)(first + tok) * j.q.ld + (uint64_t)(head * hpg + r0 + r - tok * hpg) * j.q.ldh + d0;
#pragma unroll
          for (uint32_t k = 0; k < 2; k++) {
            if (F32) {
              const uint32_t *q = reinterpret_cast<const uint32_t *>(j.q.base) + o + 4u * k;
              x[i][half][k] = wide ? *reinterpret_cast<const uint2 *>(q) : make_uint2(q[0], q[1]);
            } else {
              const uint16_t *q = reinterpret_cast<const uint16_t *>(j.q.base) + o + 4u * k;
              x[i][half][k].x = wide ? *reinterpret_cast<const uint32_t *>(q) : q[0] | ((uint32_t)q[1] << 16);
            }
          }
        }
      }
      if (F32) {   // a thread's rows are g4 of its fragments
#pragma unroll
        for (uint32_t i = 0; i < E; i++) {
          float mx = 0.0f;   // of the numbers
#pragma unroll
          for (uint32_t k = 0; k < 2; k++) mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(x[i][0][k].x)), fabsf(__uint_as_float(x[i][0][k].y))));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const uint32_t rt = (i * C::kThreads + tid) / (32u * (D / 16));
          if (t4 == 0 && rt < (uint32_t)RT) atomicMax(&qmax[rt * RR + g4], __float_as_uint(mx));
        }
        __syncthreads();
      }
#pragma unroll
      for (uint32_t i = 0; i < E; i++) {
        uint4 f;
        if (F32) {   // rows + 8: what f16 leaves of the same rows
          const uint32_t rt = min((i * C::kThreads + tid) / (32u * (D / 16)), (uint32_t)RT - 1u);
          const float up = row_up(qmax[rt * RR + g4]);
          const float2 a = make_float2(__uint_as_float(x[i][0][0].x) * up, __uint_as_float(x[i][0][1].x) * up), c = make_float2(__uint_as_float(x[i][0][0].y) * up, __uint_as_float(x[i][0][1].y) * up);
          f.x = pack2(a.x, a.y);
          f.z = pack2(c.x, c.y);
          const float2 h0 = __half22float2(*reinterpret_cast<const __half2 *>(&f.x)), h1 = __half22float2(*reinterpret_cast<const __half2 *>(&f.z));
          f.y = pack2(a.x - h0.x, a.y - h0.y);
          f.w = pack2(c.x - h1.x, c.y - h1.y);
        } else {
          f.x = __byte_perm(x[i][0][0].x, x[i][0][1].x, 0x5410);
          f.z = __byte_perm(x[i][0][0].x, x[i][0][1].x, 0x7632);
          f.y = __byte_perm(x[i][H - 1][0].x, x[i][H - 1][1].x, 0x5410);
          f.w = __byte_perm(x[i][H - 1][0].x, x[i][H - 1][1].x, 0x7632);
        }
        if (all % C::kThreads == 0 || i * C::kThreads + tid < all) qf[i * C::kThreads + tid] = f;
      }
    }
    __syncthreads();
    // this warp's dims and keys in P V
    const uint32_t ds = warp % C::kDs, kshare = warp / C::kDs;
    const uint32_t d0 = ds * (8 * NPL) + g4 * NPL;                 // the lane's first dim
    const uint32_t swap = NPL == 8 ? (g4 >> 2) & 1u : 0u;          // the second group of 32 dims starts with the odd key: other banks
    const uint32_t step0 = kshare * C::kSteps;                     // the warp's first 16-key step of an item (kSteps divides 4, or is the item)
    const uint32_t voff = (step0 / 4u) * C::kPage2 + C::kK + d0 / 32u * 1280u, word = (d0 % 32u) / 8u * 4u;
    constexpr int RH = F32 ? 1 : 2;   // rows of a lane per fragment: g4 (and g4 + 8)
    float o[RT][NPL][4], m[RT][RH], l[RT][RH];
    int32_t pos[RT][RH];
    float scale[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      scale[rt] = F32 ? j.scale * row_down(qmax[rt * RR + g4]) : log2_scale;
#pragma unroll
      for (int i = 0; i < NPL; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[rt][i][e] = 0.0f;
#pragma unroll
      for (int h = 0; h < RH; h++) {
        m[rt][h] = -INFINITY;
        l[rt][h] = 0.0f;
        pos[rt][h] = rpos[rt * RR + g4 + 8 * h];
      }
    }
    const int32_t pos0 = (int32_t)(len - T + r0 / hpg), pos1 = (int32_t)s.end - 1;   // of the block's rows
    bool lost = false;
    for (uint32_t i = 0; i < steps; i++) {
      const uint32_t st = (it + i) % NS, pi = (from + i) * KP;
      if (!tc::mbar_wait(&full[st], ((it + i) / NS) & 1u, &abort_flag, j.err, 0x4a1u, polls)) lost = true;
      const uint8_t *stage = ring + st * C::kStage;
      uint32_t key0[KP], ok[KP];
#pragma unroll
      for (int k = 0; k < KP; k++) {
        key0[k] = page_at(s, pi + k) * kPage;
        ok[k] = page_ok[st][k];
      }
      // ---- S = Q K^T: this warp's 8-key tiles, all of one page
      const int kpw = KP == 1 ? 0 : (int)(warp / (NW / KP));
      const uint32_t wk = (warp % (NW / KP)) * NT;                     // its first tile in the page
      const uint8_t *kp = stage + kpw * C::kPage2 + (D >= 128 ? t4 * kRec : (t4 >> 1) * kRec);
      float sc[RT][NT][4];
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[rt][nt][e] = 0.0f;
#pragma unroll
      for (int g = 0; g < (D >= 128 ? D / 128 : 1); g++) {
        uint32_t w[NT][KW], s2[NT], mn2[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint32_t key = (wk + nt) * 8u + g4;
          const uint8_t *rec = kp + g * 4 * kRec;
          if constexpr (KW == 4) {
            const uint4 u4 = *reinterpret_cast<const uint4 *>(rec + key * 16u);
            w[nt][0] = u4.x; w[nt][1] = u4.y; w[nt][2] = u4.z; w[nt][3] = u4.w;
          } else {
            const uint2 u2 = *reinterpret_cast<const uint2 *>(rec + key * 16u + (t4 & 1u) * 8u);
            w[nt][0] = u2.x; w[nt][1] = u2.y;
          }
          const uint32_t sm = lds_u32(rec + 1024 + key * 4u);
          s2[nt] = __byte_perm(sm, 0, 0x1010);
          mn2[nt] = __byte_perm(sm, 0, 0x3232);
        }
#pragma unroll
        for (int wi = 0; wi < KW; wi++) {
          uint32_t kb[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; nt++) kv_deq8(w[nt][wi], s2[nt], mn2[nt], kb[nt]);   // dims (e, e + 4)
#pragma unroll
          for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
              const uint4 f = qf[(rt * (D / 16) + 2 * (g * KW + wi) + half) * 32 + lane];
              const uint32_t a[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
              for (int nt = 0; nt < NT; nt++) mma_f16(sc[rt][nt], a, kb[nt][2 * half], kb[nt][2 * half + 1]);
            }
        }
      }
      // ---- mask (a page that the whole block sees needs none), the row maxima
      const int32_t k0 = (int32_t)(KP == 1 ? key0[0] : key0[kpw]);
      const bool here = (KP == 1 ? ok[0] : ok[kpw]) != 0u;
      const bool plain = here && k0 + 63 <= pos0 && (!W || k0 > pos1 - (int32_t)W || (uint32_t)k0 + 63u < S);
      float x[RT][NT][RH][2];
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int h = 0; h < RH; h++) {
          float mx = -INFINITY;
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) x[rt][nt][h][e] = (F32 ? sc[rt][nt][e] + sc[rt][nt][e + 2] : sc[rt][nt][2 * h + e]) * scale[rt];
          if (!plain) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const int32_t key = k0 + (int32_t)((wk + nt) * 8u + 2u * t4) + e;
                if (!(here && key <= pos[rt][h] && (!W || key > pos[rt][h] - (int32_t)W || (uint32_t)key < S))) x[rt][nt][h][e] = -INFINITY;
              }
          }
#pragma unroll
          for (int nt = 0; nt < NT; nt++) mx = fmaxf(mx, fmaxf(x[rt][nt][h][0], x[rt][nt][h][1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if (t4 == 0) wmax[rt * RR + g4 + 8 * h][warp] = mx;
        }
      __syncthreads();   // the previous item's P V is done: its ring slot is free
      if (warp == 0 && i > 0 && i - 1 + NS < steps) issue(i - 1 + NS);
      // slots that no row of the unit sees hold zeros, whatever the memory holds: their (s, mn) of V
#pragma unroll
      for (int k = 0; k < KP; k++) {
        const uint32_t ky = key0[k];
        if (!ok[k] || ky + kPage > s.end || (ky < s.first_pos && ky + kPage > S)) {
          uint8_t *vs = ring + st * C::kStage + k * C::kPage2 + C::kK + 1024u;
          for (uint32_t e = tid; e < 64u * C::kRecs; e += C::kThreads) {
            const uint32_t key = ky + (e & 63u);
            if (!ok[k] || key >= s.end || (key < s.first_pos && key >= S)) *reinterpret_cast<uint32_t *>(vs + (e >> 6) * 1280u + (e & 63u) * 4u) = 0u;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy into this slot
        }
      }
      // ---- P = 2^15 exp(x - m), into shared memory as f16 (f32: high and low parts)
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        float keep[RH];
#pragma unroll
        for (int h = 0; h < RH; h++) {
          const uint32_t r = rt * RR + g4 + 8 * h;
          float mn = m[rt][h];
#pragma unroll
          for (int w = 0; w < NW; w += 4) {
            const float4 x4 = *reinterpret_cast<const float4 *>(&wmax[r][w]);
            mn = fmaxf(mn, fmaxf(fmaxf(x4.x, x4.y), fmaxf(x4.z, x4.w)));
          }
          const float ref = mn == -INFINITY ? 0.0f : mn;
          keep[h] = mn == m[rt][h] ? 1.0f : ex(m[rt][h] - ref);   // 0 while nothing has been seen
          m[rt][h] = mn;
          l[rt][h] *= keep[h];
          uint8_t *row = ps + (rt * 16 + g4 + 8 * h) * C::kPRow;
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            const float p0 = ex(x[rt][nt][h][0] - ref) * kPUp, p1 = ex(x[rt][nt][h][1] - ref) * kPUp;
            l[rt][h] += p0 + p1;
            const uint32_t hi2 = pack2(p0, p1), col = ((warp * NT + nt) * 8u + 2u * t4) * 2u;
            *reinterpret_cast<uint32_t *>(row + col) = hi2;
            if (F32) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi2));
              *reinterpret_cast<uint32_t *>(row + 8 * C::kPRow + col) = pack2(p0 - f.x, p1 - f.y);
            }
          }
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[RH - 1] != 1.0f)) {
#pragma unroll
          for (int nt = 0; nt < NPL; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[rt][nt][e] *= keep[F32 ? 0 : e >> 1];
        }
      }
      __syncthreads();
      // ---- O += P V: this warp's dims and keys
      float c[RT][NPL][4];
#pragma unroll
      for (int ks = 0; ks < C::kSteps; ks++) {
        const uint8_t *vg = stage + voff + (C::kSteps > 4 ? (ks / 4) * C::kPage2 : 0u), *vw = vg + word;
        const uint32_t row16 = (C::kSteps >= 4 ? ks % 4 : step0 % 4u + ks) * 16u;   // in the page
        uint32_t vb[2][NPL];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t key = row16 + h * 8 + 2 * t4;
          const uint32_t w0 = lds_u32(vw + (key + swap) * 16u), w1 = lds_u32(vw + (key + 1u - swap) * 16u);
          const uint2 sm = *reinterpret_cast<const uint2 *>(vg + 1024u + key * 4u);
          const uint32_t s2 = __byte_perm(sm.x, sm.y, 0x5410), mn2 = __byte_perm(sm.x, sm.y, 0x7632);   // (key, key + 1)
          uint32_t q[4];
          if constexpr (NPL == 8) {
            kv_deq8(__byte_perm(w0, w1, swap ? 0x1054u : 0x5410u), s2, mn2, q);
#pragma unroll
            for (int e = 0; e < 4; e++) vb[h][e] = q[e];
            kv_deq8(__byte_perm(w0, w1, swap ? 0x3276u : 0x7632u), s2, mn2, q);
#pragma unroll
            for (int e = 0; e < 4; e++) vb[h][e + 4] = q[e];
          } else {
            kv_deq8(__byte_perm(w0, w1, (d0 & 4u) ? 0x7632u : 0x5410u), s2, mn2, vb[h]);
          }
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
          uint32_t a[4];
          ldsm_x4(tc::smem_u32(ps + (rt * 16 + (lane & 15u)) * C::kPRow + (step0 + ks) * 32u + (lane >> 4) * 16u), a);
#pragma unroll
          for (int nt = 0; nt < NPL; nt++) {
            if (!F32) mma_f16(o[rt][nt], a, vb[0][nt], vb[1][nt]);
            else if (ks == 0) mma_f16_zero(c[rt][nt], a, vb[0][nt], vb[1][nt]);
            else mma_f16(c[rt][nt], a, vb[0][nt], vb[1][nt]);
          }
        }
      }
      if (F32) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
          for (int nt = 0; nt < NPL; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[rt][nt][e] += c[rt][nt][e];
      }
    }
    if (__syncthreads_or(lost)) {   // a copy did not arrive in time: j.err says so. The copies in flight, each slot's last, land before
      if (warp == 0)                // the CTA leaves: a slot's wait is bounded, too
        for (uint32_t i = started > (uint32_t)NS ? started - NS : 0u; i < started; i++)
          for (uint32_t k = 0; k < (1u << 16) && !tc::mbar_try(&full[i % NS], (i / NS) & 1u); k++) {}
      return;
    }
    it += steps;
    // ---- the rows' sums over the warps, then out or into the workspace
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int h = 0; h < RH; h++) {
        float t = l[rt][h];
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        if (t4 == 0) wsum[rt * RR + g4 + 8 * h][warp] = t;
      }
    __syncthreads();
    if (F32 && tid < (uint32_t)RB) qmax[tid] = 0u;   // every thread has its rows' scales; before the next unit's barriers
    // ---- the key shares of O meet in the first one, through the ring (no copy is in flight)
#pragma unroll 1
    for (int k = 1; k < C::kKs; k++) {
      float *x = reinterpret_cast<float *>(ring) + (size_t)ds * (RT * NPL * 4 * 32) + lane;
      if (kshare == (uint32_t)k) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
          for (int nt = 0; nt < NPL; nt++)
#pragma unroll
            for (int e = 0; e < (F32 ? 2 : 4); e++) x[((rt * NPL + nt) * 4 + e) * 32] = F32 ? o[rt][nt][e] + o[rt][nt][e + 2] : o[rt][nt][e];
      }
      __syncthreads();
      if (kshare == 0) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
          for (int nt = 0; nt < NPL; nt++)
#pragma unroll
            for (int e = 0; e < (F32 ? 2 : 4); e++) o[rt][nt][e] += x[((rt * NPL + nt) * 4 + e) * 32];
      }
      __syncthreads();
    }
    const bool whole = from == 0 && to == n;
    // a run has at most one part of a unit that began earlier (slot 0) and one of a unit that goes on after it (slot 1)
    float *part = j.part + ((uint64_t)blockIdx.x * 2u + (from ? 0u : 1u)) * RB * (D + 2);
    if (!whole && from == 0 && tid == 0) {
      j.desc[blockIdx.x] = make_uint4(1u + run_of(begin + n - 1u, total, G), b, r0, head);
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int h = 0; h < RH; h++) {
        const uint32_t r = rt * RR + g4 + 8 * h;
        if (r >= nrow || kshare) continue;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) sum += wsum[r][w];
        const float inv = whole ? (sum > 0.0f ? 1.0f / sum : 0.0f) : 1.0f;
        float y[2][NPL];   // dims 2 t4 * NPL .. and (2 t4 + 1) * NPL ..: contiguous
#pragma unroll
        for (int nt = 0; nt < NPL; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) y[e][nt] = (F32 ? o[rt][nt][e] + o[rt][nt][e + 2] : o[rt][nt][2 * h + e]) * inv;
        const uint32_t d = ds * (8 * NPL) + 2 * t4 * NPL;
        if (whole) {
          const uint64_t q = (uint64_t)(first + (r0 + r) / hpg) * j.out.ld + (uint64_t)(head * hpg + (r0 + r) % hpg) * j.out.ldh + d;
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int nt = 0; nt < NPL; nt++) {
              if (F32) reinterpret_cast<float *>(j.out.base)[q + e * NPL + nt] = y[e][nt];
              else reinterpret_cast<__half *>(j.out.base)[q + e * NPL + nt] = __float2half_rn(y[e][nt]);
            }
        } else {
          float *p = part + (uint64_t)r * (D + 2);
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int nt = 0; nt < NPL; nt += 2) *reinterpret_cast<float2 *>(p + d + e * NPL + nt) = make_float2(y[e][nt], y[e][nt + 1]);
          if (warp == 0 && t4 == 0) {
            p[D] = m[rt][h];
            p[D + 1] = sum;
          }
        }
      }
    at = begin + to;
    if (C::kKs > 1) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the ring was written: before the next unit's copies
    __syncthreads();   // q fragments, wsum and rpos are free
  }
}

// joins the parts of the units that several runs share: CTA (c, r) takes row r of the unit that run c begins.
// M = max m, o = sum exp(m - M) acc / sum exp(m - M) l, in run order
template <int D, bool F32, int RB>
__global__ void __launch_bounds__(256) kv4_attn_join_kernel(AttnJob j) {
  dep_enter();
  constexpr int L = D / 4, K = 256 / L > 0 ? 256 / L : 1;   // lanes per row (4 dims each), parts at a time
  __shared__ float4 acc[K][L];
  __shared__ float sums[K];
  const uint4 u = j.desc[blockIdx.x];
  const uint32_t r = blockIdx.y;
  if (!u.x) return;
  const uint32_t b = u.y, r0 = u.z, head = u.w, hpg = j.hpg;
  uint32_t first;
  const uint32_t T = kv_tokens(j.v, b, first);
  if (r0 + r >= T * hpg) return;
  const uint32_t n = u.x - blockIdx.x;   // parts: this run's slot 1, then slot 0 of the following runs
  const auto part = [&](uint32_t i) {
    return j.part + ((uint64_t)(blockIdx.x + i) * 2u + (i ? 0u : 1u)) * RB * (D + 2) + (uint64_t)r * (D + 2);
  };
  float M = -INFINITY;   // each warp for itself
#pragma unroll 4
  for (uint32_t i = threadIdx.x & 31u; i < n; i += 32) M = fmaxf(M, part(i)[D]);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
  const float ref = M == -INFINITY ? 0.0f : M;
  const uint32_t k = threadIdx.x / L, e = threadIdx.x % L;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
#pragma unroll 4
  for (uint32_t i = k; i < n; i += K) {
    const float *p = part(i);
    const float w = F32 ? expf(p[D] - ref) : exp2f(p[D] - ref);
    const float2 a = *reinterpret_cast<const float2 *>(p + 4 * e), c = *reinterpret_cast<const float2 *>(p + 4 * e + 2);
    o.x = fmaf(w, a.x, o.x);
    o.y = fmaf(w, a.y, o.y);
    o.z = fmaf(w, c.x, o.z);
    o.w = fmaf(w, c.y, o.w);
    sum = fmaf(w, p[D + 1], sum);
  }
  acc[k][e] = o;
  if (e == 0) sums[k] = sum;
  __syncthreads();
  if (k) return;
  for (int i = 1; i < K; i++) {
    const float4 a = acc[i][e];
    o.x += a.x;
    o.y += a.y;
    o.z += a.z;
    o.w += a.w;
    sum += sums[i];
  }
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  const uint64_t q = (uint64_t)(first + (r0 + r) / hpg) * j.out.ld + (uint64_t)(head * hpg + (r0 + r) % hpg) * j.out.ldh + 4 * e;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (F32) reinterpret_cast<float *>(j.out.base)[q + i] = y[i];
    else reinterpret_cast<__half *>(j.out.base)[q + i] = __float2half_rn(y[i]);
  }
}

template <int D, bool F32, int NPL, int RT, int KP, int NW>
p0_status attn_launch(p0_ctx *c, AttnJob &j) {
  using C = Cfg<D, F32, NPL, RT, KP, NW>;
  const size_t smem = C::kSmem + ((size_t)j.v.rows + 1) * 4;
  const auto kern = kv4_attn_kernel<D, F32, NPL, RT, KP, NW>;
  int per = 0;
  cudaError_t e = p0_smem_limit((const void *)kern);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, C::kThreads, smem);
  if (e != cudaSuccess || per < 1) { cudaGetLastError(); return p0_fail(c, P0_EDEVICE, "kv4Attn: the kernel does not fit this device"); }
  const uint32_t G = (uint32_t)(per * c->sm_count);
  uint32_t *cnt;
  void *ws;
  const size_t parts = (size_t)G * 2 * C::kRows * (D + 2) * 4;
  p0_status st = p0_workspace(c, 0, (size_t)G * sizeof(uint4) + parts, &cnt, &ws);
  if (st) return st;
  j.desc = (uint4 *)ws;
  j.part = (float *)(j.desc + G);
  const char *limit = getenv("P0MM_KV4_POLLS");   // for tests of what follows a wait that gives up
  const uint32_t polls = limit ? (uint32_t)strtoul(limit, nullptr, 10) : P0_SPIN_LIMIT;
  launch_dep(kern, dim3(G), dim3(C::kThreads), smem, c->stream, j, polls);
  if ((st = p0_launched(c, "kv4Attn"))) return st;
  launch_dep(kv4_attn_join_kernel<D, F32, C::kRows>, dim3(G, C::kRows), dim3(256), 0, c->stream, j);
  return p0_launched(c, "kv4Attn join");
}

// fragments per block: one, two or four, so that a page is dequantised for as many rows at once as there are. Four of f32 take 32
// dims a warp instead of 64. At D = 512 one: with two, a warp's sums leave one CTA an SM, and dequantising twice on two is as fast
// or faster (4 sequences of 8000 keys, 32 rows a KV head: f32 58 us with two, 57 with one; f16 53 and 47)
template <int D, bool F32, int KP>
p0_status pick(p0_ctx *c, AttnJob &j, uint32_t frags) {
  // One fragment and room for many pages (the lengths are on the device: what the table and the window allow decides): four
  // warps and a page an item, four CTAs to an SM that do not wait for one another at the barriers. 32 contexts up to 65500
  // keys: 117 us, with eight warps and two pages 123 (114 since); 8 contexts of 10 pages: 14.1 and 12.2, which is what short
  // contexts in wide tables lose
  const uint64_t most = j.window ? min((uint64_t)j.v.ld, (uint64_t)j.window / kPage + 2 + (j.sinks + kPage - 1) / kPage) : j.v.ld;
  if constexpr (D < 512)
    if (frags <= 1 && most * j.v.rows * j.v.nkv >= 16ull * c->sm_count) return attn_launch<D, F32, 8, 1, 1, 4>(c, j);
  if constexpr (D < 512) {
    if (frags == 2) return attn_launch<D, F32, 8, 2, KP, 8>(c, j);
    if (frags > 2) return attn_launch<D, F32, F32 ? 4 : 8, 4, KP, 8>(c, j);
  }
  return attn_launch<D, F32, 8, 1, KP, 8>(c, j);
}

}  // namespace

extern "C" p0_status p0_kv4_attn(p0_ctx *c, const p0_kv4_attn_args *a) {
  if (!c || !a) return P0_EINVAL;
  const char *op = "kv4Attn";
  if (a->type > P0_F16) return p0_fail(c, P0_EINVAL, "%s: type %u", op, a->type);
  if (!a->n) return P0_OK;
  AttnJob j = {};
  p0_status st;
  if ((st = kv_view(c, a->kv, true, op, &j.v))) return st;
  if (!a->nh || a->nh % a->kv.nkv) return p0_fail(c, P0_EINVAL, "%s: %u query heads over %u KV heads", op, a->nh, a->kv.nkv);
  if ((st = kv_new_tokens(c, a->n, a->T, a->cu, a->cu_off, op, &j.v))) return st;
  if ((st = kv_rows(c, a->q, a->n, a->nh, a->kv.D, a->type, op, "q", &j.q))) return st;
  if ((st = kv_rows(c, a->out, a->n, a->nh, a->kv.D, a->type, op, "out", &j.out))) return st;
  j.hpg = a->nh / a->kv.nkv;
  j.units = a->kv.nkv;
  const uint32_t most = a->kv.table_ld * kPage;          // no position is that large, so positions and bounds fit 31 bits
  j.window = a->window < most ? a->window : 0u;          // a longer window hides nothing
  j.sinks = a->sinks < most ? a->sinks : most;
  j.scale = a->scale != 0.0f ? a->scale : 1.0f;
  j.err = c->d_err;
  // the kernels count query rows and items (pages of row blocks) in 32 bits
  const uint64_t rows = (uint64_t)a->n * j.hpg;
  if (rows > 0x7fffffffu || (rows / 8 + a->kv.rows + 1) * a->kv.nkv * a->kv.table_ld > 0xffffffffull)
    return p0_fail(c, P0_EINVAL, "%s: %u tokens x %u heads over %u pages pass 32 bits", op, a->n, a->nh, a->kv.table_ld);
  cudaSetDevice(c->device);
  const bool f32 = a->type == P0_F32;
  if (!f32) {
    bool taken = false;
    if ((st = kv4_attn_prompt(c, j, &taken)) || taken) return st;
  }
  const uint32_t per = a->T && !a->cu.id ? a->T * j.hpg : (uint32_t)((rows + a->kv.rows - 1) / a->kv.rows), frags = (per + (f32 ? 7u : 15u)) / (f32 ? 8u : 16u);
  switch (a->kv.D) {
    case 64: return f32 ? pick<64, true, 2>(c, j, frags) : pick<64, false, 2>(c, j, frags);
    case 128: return f32 ? pick<128, true, 2>(c, j, frags) : pick<128, false, 2>(c, j, frags);
    case 256: return f32 ? pick<256, true, 2>(c, j, frags) : pick<256, false, 2>(c, j, frags);
    default: return f32 ? pick<512, true, 1>(c, j, frags) : pick<512, false, 1>(c, j, frags);
  }
}
