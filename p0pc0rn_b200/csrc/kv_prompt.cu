// kv_prompt.cu -- kv4Attn for prompts: f16 queries with many rows per KV head, on the tensor cores.
//
// Two kernels. The first turns the pages that the call sees into f16 once (each serves every row block of its sequence),
// as the tiles that the matrix instructions read: K as [64 keys][64 dims] blocks, V transposed as [D dims][64 keys], both
// rows of 128 bytes in the 128-byte swizzle, so that plain bulk copies bring them to shared memory. Slots that no row of
// the call sees become zeros.
// The second is attention over tiles of 128 keys (two pages) for 256 query rows (of one KV head: tokens x its query heads)
// by a pair of CTAs, each with 128 of the rows. The pair's MMAs (cta_group::2) read half of K and V from either CTA's
// shared memory: a CTA loads one of the two pages of K and half of V's dims, half the bytes out of L2 that a CTA on its
// own would need for the same rows, and the rings hold two tiles of D = 256. In each CTA one warp issues the copies of K and
// V, one those of q, two the pair's MMAs (the odd CTA's tell the even one's what has landed), eight hold half a row (64
// keys) per thread:
//   S_j = Q K_j^T     tcgen05.mma, 256 x 128 x D, f32 in tensor memory: S_j+1 runs while softmax_j computes, as soon as it has
//                     read S_j (256 dims and more: one buffer) or S_j-1 (two)
//   P_j = 2^(S_j c - m)   the row's maximum by its two threads through shared memory; f16 in tensor memory (an operand's type:
//                     a rounding of 2^-11 of each P, as the output's own), two buffers
//   O  += P_j V_j     tcgen05.mma with P from tensor memory
// Nothing in tensor memory is written while an MMA that was not waited for may read it (MMAs of different shapes or
// accumulators have no order among themselves).
// m is 7 less than the row's maximum as of the last time O was rescaled: P starts at 2^7 and may grow to 2^15 (f16 ends at
// 2^16) before O, in tensor memory, is read and written again, which then happens in few tiles. P that f16 does not hold lies
// below 2^-32 of the maximum's, so that a long tail of small P counts in O as it does in l.
// At 512 dims O does not fit: a unit is a row block and half of the output's dims, S is computed for each half, 1.5 times
// the products of a whole.
// Work is cut into equal runs of key tiles as in kv_attn.cuh, one per pair; a unit's parts meet in the join kernel.
//
// What bounds it: an MMA of 128 columns occupies the issuing thread for 84 cycles (64 of them at the tensor core's rate), one of 256
// columns 128, and what a thread issues after a wait that is already over comes 150 cycles late: S and P V by one thread took
// 4100 cycles a tile of 256 dims, by a thread each 2800, the softmax's chain (load 64 scores, maximum, barrier, exponentials, store P)
// with one S buffer. A unit's end (the last P V, output through shared memory) costs another 6000 to 8000 cycles, under which the
// next unit's K, q and first S run; the widening takes 7 us, the join of parts 8 to 10. 3 sequences with 2048 new of up to
// 5003 tokens, 8 heads of 256 dims: 119 us, 0.91 PFLOP/s (132 in long runs at the power limit); 4 with 1500 of 6001, 16 heads of 128 on 4, window 1024: 131 us,
// 0.34 PFLOP/s (units of 9 tiles); 2048 of 6000, 8 heads of 512: 246 us, 0.68 PFLOP/s. Where the compiler places the code decides 5 % of these.
#include "kv_attn.cuh"

namespace {

constexpr uint32_t kDrain = 1u << 16;                // polls for what is in flight when a wait has given up: copies and MMAs end in microseconds
constexpr uint32_t kRB = 256, kCR = 128, kPP = 2;   // query rows of a block and of a CTA, pages of a key tile
constexpr uint32_t kE = 4;                   // a unit's beginning and end cost about as much as four key tiles
constexpr int kSoft = 256, kThreads = kSoft + 128;   // warps 0-7: softmax (0-3 the tile's first page, 4-7 its second); 8: copies; 9: S; 10: P V; 11: q

template <int D>
struct Cfg {
  static constexpr uint32_t kKB = D / 64;                      // 64-dim blocks of K
  static constexpr uint32_t kParts = D == 512 ? 2 : 1, kDV = D / kParts;   // parts of an output row; dims of one
  static constexpr uint32_t kNK = D == 512 ? 4 : 1, kNV = D == 512 ? 2 : 1;   // stages of a K and of a V tile
  static constexpr uint32_t kStage = D * 128 / kNK;            // of the ring: (a quarter of the dims of) a page of K; half of V's dims of two pages (one)
  static constexpr uint32_t kQ = kKB * 16384;
  static constexpr int kSK = D == 512 ? 3 : D == 256 ? 2 : 4, kSV = D >= 256 ? 2 : 4, kStages = kSK + kSV;   // stages of the rings of K and V
  static constexpr uint32_t kSlot = D * 256;                   // a page of one head in f16: K blocks, then V
  static constexpr uint32_t kOut = 32 * 80;                    // a warp's 32 x 32 f16 of the output, rows padded to 80 bytes
  // tensor memory: O at 0, then P and S, 64 and 128 columns a buffer
  static constexpr uint32_t kSB = kDV == 256 ? 1 : 2, kColS = 256, kColP = kDV == 256 ? 384 : 128;
  static constexpr uint32_t kStg = D == 512 ? 0 : kQ + kStages * kStage;   // the output on its way; D = 512: in q's place
  static constexpr uint32_t kSmem = 1024 + kQ + kStages * kStage + (kStg ? 8 * kOut : 0);
};

// The pages of sequence b that the call sees, in order: those of the span over all its tokens. exo[b] = pages before it.
__device__ __forceinline__ Span whole_span(const AttnJob &j, uint32_t b) {
  uint32_t lo;
  const uint32_t T = kv_tokens(j.v, b, lo);
  return T ? span_of(kv_len(j.v, b), T, 0, T - 1, j.window, j.sinks) : span_of(0, 1, 0, 0, 0, 0);
}
__device__ __forceinline__ void plan_pages(const AttnJob &j, uint32_t *exo) {
  for (uint32_t b = threadIdx.x; b < j.v.rows; b += blockDim.x) exo[b + 1] = whole_span(j, b).n;
  if (threadIdx.x == 0) exo[0] = 0u;
  __syncthreads();
  if (threadIdx.x < 32) warp_sums(exo + 1, j.v.rows);
  __syncthreads();
}

// ---------------------------------------------------------------- pages to f16 tiles
constexpr int kET = 256;
template <int D>
__global__ void __launch_bounds__(kET) kv4_widen_kernel(AttnJob j) {
  dep_enter();
  extern __shared__ uint32_t exo[];
  plan_pages(j, exo);
  const uint32_t total = claims_fit(j.v) ? exo[j.v.rows] : 0u, nkv = j.v.nkv;
  constexpr uint32_t part = D / 32 * 1280;
  uint32_t b = 0;
  for (uint64_t w2 = blockIdx.x; w2 < (uint64_t)total * nkv * 2u; w2 += gridDim.x) {   // K, or V, of a page and head
    const uint64_t w = w2 >> 1;
    const uint32_t i = (uint32_t)(w / nkv), head = (uint32_t)(w % nkv);
    while (exo[b + 1] <= i) b++;
    const Span s = whole_span(j, b);
    const uint32_t jp = page_at(s, i - exo[b]), page = j.v.table[(uint64_t)b * j.v.ld + jp], key0 = jp * kPage;
    const bool ok = page < j.v.pages;
    const uint8_t *rec = j.v.pool + (ok ? page : 0u) * j.v.stride + (uint64_t)head * 2u * part + (w2 & 1u) * part;
    uint8_t *to = j.wide + w * Cfg<D>::kSlot + (w2 & 1u) * (D * 128);
    const auto there = [&](uint32_t k) { return ok && key0 + k < s.end && (key0 + k >= s.first_pos || key0 + k < j.sinks); };
    if (!(w2 & 1u)) {
      // K: a thread turns one word (8 dims of a key) into 16 bytes; 8 lanes make a key's 128-byte row of a block
      constexpr uint32_t N = 64u * (D / 8) / kET, U = N < 8 ? N : 8;
#pragma unroll 1
      for (uint32_t n0 = 0; n0 < N; n0 += U) {
        uint32_t x[U], sm[U];
#pragma unroll
        for (uint32_t n = 0; n < U; n++) {
          const uint32_t e = (n0 + n) * kET + threadIdx.x, c = e & 7u, key = (e >> 3) & 63u, g = (e >> 9) * 2u + (c >> 2);
          x[n] = *reinterpret_cast<const uint32_t *>(rec + g * 1280u + key * 16u + (c & 3u) * 4u);
          sm[n] = *reinterpret_cast<const uint32_t *>(rec + g * 1280u + 1024u + key * 4u);
        }
#pragma unroll
        for (uint32_t n = 0; n < U; n++) {
          const uint32_t e = (n0 + n) * kET + threadIdx.x, c = e & 7u, key = (e >> 3) & 63u, blk = e >> 9;
          uint4 o = make_uint4(0u, 0u, 0u, 0u);
          if (there(key)) {
            const uint32_t s2 = __byte_perm(sm[n], 0, 0x1010), mn2 = __byte_perm(sm[n], 0, 0x3232), y = x[n] >> 4;
            o.x = kv_deq2(__byte_perm(x[n], y, 0x4400), s2, mn2);   // byte i: dims 2i, 2i + 1
            o.y = kv_deq2(__byte_perm(x[n], y, 0x5511), s2, mn2);
            o.z = kv_deq2(__byte_perm(x[n], y, 0x6622), s2, mn2);
            o.w = kv_deq2(__byte_perm(x[n], y, 0x7733), s2, mn2);
          }
          *reinterpret_cast<uint4 *>(to + blk * 8192u + key * 128u + ((c ^ (key & 7u)) * 16u)) = o;
        }
      }
    } else {
      // V: a thread turns the words of 8 keys (the same 8 dims) into 8 dims' 16-byte runs of 8 keys
      for (uint32_t e = threadIdx.x; e < 8u * (D / 8); e += kET) {
        const uint32_t kc = e & 7u, dw = e >> 3;
        const uint8_t *g = rec + (dw >> 2) * 1280u;
        uint32_t x[8], o[8][4];
        uint2 sm[4];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) x[k] = *reinterpret_cast<const uint32_t *>(g + (kc * 8u + k) * 16u + (dw & 3u) * 4u);
#pragma unroll
        for (uint32_t p = 0; p < 4; p++) sm[p] = *reinterpret_cast<const uint2 *>(g + 1024u + (kc * 8u + 2u * p) * 4u);
#pragma unroll
        for (uint32_t p = 0; p < 4; p++) {
          const uint32_t key = kc * 8u + 2u * p;
          if (!there(key)) sm[p].x = 0u;
          if (!there(key + 1)) sm[p].y = 0u;
          const uint32_t s2 = __byte_perm(sm[p].x, sm[p].y, 0x5410), mn2 = __byte_perm(sm[p].x, sm[p].y, 0x7632);
          const uint32_t lo = __byte_perm(x[2 * p], x[2 * p + 1], 0x5410), hi = __byte_perm(x[2 * p], x[2 * p + 1], 0x7632);
#pragma unroll
          for (uint32_t d = 0; d < 4; d++) {
            o[d][p] = kv_deq2((lo >> (4 * d)), s2, mn2);
            o[d + 4][p] = kv_deq2((hi >> (4 * d)), s2, mn2);
          }
        }
#pragma unroll
        for (uint32_t d = 0; d < 8; d++)
          *reinterpret_cast<uint4 *>(to + (dw * 8u + d) * 128u + ((kc ^ d) * 16u)) = make_uint4(o[d][0], o[d][1], o[d][2], o[d][3]);
      }
    }
  }
}

// ---------------------------------------------------------------- attention
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const void *tmap, uint64_t *bar, int32_t c0, int32_t c1, int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"(tmap), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// bits 0 .. n - 1
__device__ __forceinline__ uint64_t first_bits(int32_t n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// the same, held at 65504: scores of 2^24 and more may come out a few units above their maximum
__device__ __forceinline__ uint32_t pack2_finite(float a, float b) {
  uint32_t d;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
#pragma unroll
  for (int h = 0; h < 2; h++) {
    uint32_t t[16];
#pragma unroll
    for (int i = 0; i < 16; i++) t[i] = r[16 * h + i];
    tc::tmem_st16(taddr + 16u * h, t);
  }
}

template <int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) kv4_prompt_kernel(AttnJob j, const __grid_constant__ CUtensorMap qm) {
  using C = Cfg<D>;
  constexpr int NS = C::kStages, SK = C::kSK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *qs = smem, *ring = smem + C::kQ, *stg = smem + C::kStg;
  uint32_t *pre = reinterpret_cast<uint32_t *>(smem_raw + C::kSmem), *exo = pre + j.v.rows + 1;
  // full / empty: the stages, K's before V's (the even CTA's is full when the odd one's is, too); sfull: S of a tile is there, sread: both CTAs have read it;
  // pfull: both CTAs' P is there; odone: P V of a tile is done (each by buffer); qfull: both CTAs' q of a unit is there; qdone:
  // its last S is; ofree: this CTA's output of a unit has left q's place
  __shared__ __align__(8) uint64_t full[NS], empty[NS], sfull[2], sread[2], pfull[2], odone[2], qfull, qland, qdone, ofree, mdone[2];
  __shared__ uint32_t tmem_slot, abort_word;
  __shared__ Unit units[kThreads / 32];
  __shared__ float mx2[2][2][kCR], l2[2][2][kCR];   // [tile, unit parity][half of the tile][row]
  volatile uint32_t *abort_flag = &abort_word;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = tc::cluster_rank(), run = blockIdx.x >> 1;
  const uint32_t hpg = j.hpg, nkv = j.v.nkv, R = j.v.rows, W = j.window, S = j.sinks;
  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      tc::mbar_init(&full[i], rank ? 1 : 2);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&sfull[i], 1);
      tc::mbar_init(&sread[i], 2 * kSoft / 32);
      tc::mbar_init(&pfull[i], 2 * kSoft / 32);
      tc::mbar_init(&odone[i], 1);
    }
    tc::mbar_init(&qfull, 2);
    tc::mbar_init(&qland, 1);
    tc::mbar_init(&qdone, 1);
    tc::mbar_init(&ofree, kSoft / 32);
    tc::mbar_init(&mdone[0], 1);
    tc::mbar_init(&mdone[1], 1);
    abort_word = 0u;
    tc::fence_mbar_init();
  }
  if (warp == 8) {
    tc::tmem_alloc_pair(&tmem_slot, 512);
    tc::tmem_relinquish_pair();
  }
  plan_pages(j, exo);
  plan_items<kRB, kPP, kE>(j, pre);
  tc::fence_before();
  tc::cluster_sync();
  tc::fence_after();
  // This kernel starts when every CTA of the widening one has passed its own wait, so all that came before that one is done: lengths,
  // tables, q and the workspace are read and written while it still runs. Only the widened pages are waited for, by the warp that
  // copies them; every CTA has that warp, so this kernel does not end before the other
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 8) asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  const uint32_t total = pre[R], runs = gridDim.x >> 1, G = min(runs, max(total / 2u, 1u));   // two tiles at least: parts cost more
  if (tid == 0 && rank == 0) j.desc[run] = make_uint4(0u, 0u, 0u, 0u);
  const uint32_t lo = run < G ? (uint32_t)((uint64_t)total * run / G) : 0u, hi = run < G ? (uint32_t)((uint64_t)total * (run + 1) / G) : 0u;
  uint32_t b = lo < hi ? find_sequence(pre, R, lo) : 0u;
  uint32_t tile = 0, unit = 0;   // key tiles and units with tiles so far
  struct Ring {                  // the stage to use next, how often they came round (each role counts its own uses alike)
    uint32_t i = 0, round = 0;
    __device__ __forceinline__ void next(uint32_t n) {
      if (++i == n) i = 0u, round++;
    }
  } rk, rv;
  const float c = fabsf(j.scale) * 1.44269504088896340736f;
  const bool flip = j.scale < 0.0f;   // a negative scale turns S around, so that maxima stay maxima
  // A wait that gives up sets the CTA's abort word, after which all its waits give up at once; every warp still walks the
  // same units to the end. Nothing stops between units: the next one's K, q and first S run under this one's end
  Unit &u = units[warp];   // in shared memory: what a tile does not need stays out of the registers
  for (uint32_t at = lo; at < hi;) {
    Span s;
    {
      Unit w;
      if (at == lo || pre[b + 1] <= at) {
        while (pre[b + 1] <= at) b++;
        w = find_unit<kRB, kPP, kE>(j, pre, b, at);
      } else {   // the next one of this sequence
        w = u;
        w.begin += w.n;
        if (++w.head == j.units) {
          w.head = 0;
          w.r0 += kRB;
          w.n = unit_items<kRB, kPP, kE>(j, w.len, w.T, w.r0, w.s);
        }
      }
      s = w.s;
      __syncwarp();
      if (lane == 0) u = w;
      __syncwarp();
    }
    const uint32_t from = max(at - u.begin, kE) - kE, nt = u.n - kE, end = min(hi - u.begin, u.n), to = max(end, kE) - kE;
    at = u.begin + end;
    if (from == to) continue;   // this run holds none of the unit's tiles
    const uint32_t tiles = s.n ? to - from : 0u;
    const uint32_t head = u.head / C::kParts, oh = u.head % C::kParts;   // KV head, part of the output's dims
    const uint32_t rc = u.r0 + rank * kCR, nrow = rc < u.rows ? min(kCR, u.rows - rc) : 0u;   // this CTA's rows
    if (warp == 8) {
      // ------------------------------------------------------------ copies
      const Span all = whole_span(j, b);
      const uint8_t *base = j.wide + ((uint64_t)exo[b] * nkv + head) * C::kSlot;
      const auto slot = [&](uint32_t i) {   // page i of the unit's span (an odd last tile repeats its first page)
        const uint32_t jp = page_at(s, min(i, s.n - 1u)), k = jp < all.sink_pages ? jp : all.sink_pages + (jp - all.from);
        return base + (uint64_t)k * nkv * C::kSlot;
      };
      if (lane == 0 && tiles) {   // whichever ring has a free stage
        constexpr uint32_t half = C::kDV * 64, per = 2 / C::kNV;   // bytes of this CTA's dims of a page, pages of a stage
        const uint32_t nk = tiles * C::kNK, nv = tiles * C::kNV;
        for (uint32_t ik = 0, iv = 0, spins = 0; (ik < nk || iv < nv) && !*abort_flag;) {
          bool idle = true;
          if (ik < nk && tc::mbar_test(&empty[rk.i], (rk.round & 1u) ^ 1u)) {
            tc::mbar_expect_tx(&full[rk.i], C::kStage);
            bulk_load(ring + rk.i * C::kStage, slot(2u * (from + ik / C::kNK) + rank) + ik % C::kNK * C::kStage, C::kStage, &full[rk.i]);
            rk.next(SK);
            ik++;
            idle = false;
          }
          if (iv < nv && tc::mbar_test(&empty[SK + rv.i], (rv.round & 1u) ^ 1u)) {
            tc::mbar_expect_tx(&full[SK + rv.i], C::kStage);
            for (uint32_t k = 0; k < per; k++)
              bulk_load(ring + (SK + rv.i) * C::kStage + k * half, slot(2u * from + iv * per + k) + D * 128 + (oh * 2u + rank) * half, half, &full[SK + rv.i]);
            rv.next(C::kSV);
            iv++;
            idle = false;
          }
          spins = idle ? spins + 1u : 0u;
          if (spins == P0_SPIN_LIMIT) {
            *abort_flag = 1u;
            atomicOr(j.err, 0x4b1u);
          }
        }
      }
      __syncwarp();
    } else if (warp == 9 || warp == 10) {
      // ------------------------------------------------------------ the pair's MMAs (even CTA), word of what landed (odd CTA): S by one
      // warp, P V by another. What a thread issues after a wait comes a few hundred cycles late; with a thread each, S and P V hide that
      // for one another. The waits that are over come first
      const auto landed = [&](uint32_t i, uint32_t round) {   // the even CTA's barriers are completed by the odd one, too: acquire over the pair
        return rank ? tc::mbar_wait(&full[i], round & 1u, abort_flag, j.err, 0x4b3u, P0_SPIN_LIMIT)
                    : tc::mbar_wait_cluster(&full[i], round & 1u, abort_flag, j.err, 0x4b3u, P0_SPIN_LIMIT);
      };
      const auto part_of = [](uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); };   // within shared memory: no carry out of the address
      if (lane == 0 && rank == 1) {
        Ring &g = warp == 9 ? rk : rv;
        const uint32_t n = tiles * (warp == 9 ? C::kNK : C::kNV), size = warp == 9 ? SK : C::kSV, base = warp == 9 ? 0u : SK;
        for (uint32_t i = 0; i < n && landed(base + g.i, g.round); i++) {
          tc::mbar_arrive_rank(&full[base + g.i], 0);
          g.next(size);
        }
      } else if (lane == 0 && warp == 9 && tiles) {
        constexpr uint32_t is = tc::idesc_f16_f32(256, 128), per = C::kKB / C::kNK;   // 64-dim blocks of a stage
        bool ok = tc::mbar_wait_cluster(&qfull, unit & 1u, abort_flag, j.err, 0x4bcu, P0_SPIN_LIMIT);
        for (uint32_t t = tile; t < tile + tiles && ok; t++) {   // over S of tile t - kSB
          const uint32_t o = t - C::kSB, sb = t % C::kSB, dst = tmem + C::kColS + sb * 128u;
#pragma unroll 1
          for (uint32_t y = 0; y < C::kNK; y++) {
            if (!(ok = landed(rk.i, rk.round))) break;
            if (y == 0 && t >= C::kSB && !(ok = tc::mbar_wait(&sread[o % C::kSB], (o / C::kSB) & 1u, abort_flag, j.err, 0x4b9u, P0_SPIN_LIMIT))) break;
            tc::fence_after();
            const uint64_t kd = tc::desc_sw128(tc::smem_u32(ring + rk.i * C::kStage)), qd = tc::desc_sw128(tc::smem_u32(qs) + y * per * 16384u);
#pragma unroll
            for (uint32_t x = 0; x < per * 4u; x++)
              tc::mma_ss_f16_pair(dst, part_of(qd, (x >> 2) * 16384u + (x & 3u) * 32u), part_of(kd, (x >> 2) * 8192u + (x & 3u) * 32u), is, (y | x) != 0u);
            if (y + 1 == C::kNK) tc::mma_commit_pair(&sfull[sb]);
            tc::mma_commit_pair(&empty[rk.i]);
            rk.next(SK);
          }
        }
        if (ok) tc::mma_commit_pair(&qdone);
      } else if (lane == 0 && warp == 10 && tiles) {
        constexpr uint32_t iv = tc::idesc_f16_f32(256, C::kDV), steps = 8 / C::kNV;   // of 16 keys
        bool ok = true;
        for (uint32_t t = tile; t < tile + tiles && ok; t++) {
          const uint32_t pa = tmem + C::kColP + (t & 1u) * 64u;
#pragma unroll 1
          for (uint32_t y = 0; y < C::kNV; y++) {
            if (!(ok = landed(SK + rv.i, rv.round))) break;
            if (y == 0 && !(ok = tc::mbar_wait(&pfull[t & 1u], (t >> 1) & 1u, abort_flag, j.err, 0x4b4u, P0_SPIN_LIMIT))) break;
            tc::fence_after();
            const uint64_t vd = tc::desc_sw128(tc::smem_u32(ring + (SK + rv.i) * C::kStage));
#pragma unroll
            for (uint32_t x = 0; x < steps; x++)
              tc::mma_ts_f16_pair(tmem, pa + (y * steps + x) * 8u, part_of(vd, (x >> 2) * (C::kDV * 64u) + (x & 3u) * 32u), iv, (t != tile) | (y | x) != 0u);
            if (y + 1 == C::kNV) tc::mma_commit_pair(&odone[t & 1u]);
            tc::mma_commit_pair(&empty[SK + rv.i]);
            rv.next(C::kSV);
          }
        }
      }
      __syncwarp();
    } else if (warp == 11) {
      // ------------------------------------------------------------ q rows, as K's: blocks of 64 dims, swizzled rows of 128 bytes
      bool ok = true;
      if (unit && tiles) ok = tc::mbar_wait(&qdone, (unit - 1u) & 1u, abort_flag, j.err, 0x4bdu, P0_SPIN_LIMIT);
      if (!C::kStg && unit && tiles) ok = ok && tc::mbar_wait(&ofree, (unit - 1u) & 1u, abort_flag, j.err, 0x4beu, P0_SPIN_LIMIT);
      ok = __all_sync(0xffffffffu, ok && tiles);
      if (ok && j.qbox) {          // by tensor copies; rows of other sequences beyond this one's are not looked at
        if (lane == 0) {
          uint64_t *bar = rank ? &qland : &qfull;
          tc::mbar_expect_tx(bar, C::kQ);
          for (uint32_t k = 0; k < C::kKB; k++)
            tma_load_3d(qs + k * 16384u, &qm, bar, (int32_t)(k * 64u), (int32_t)(head * hpg + rc % hpg), (int32_t)(u.first + rc / hpg));
          if (rank && tc::mbar_wait(&qland, unit & 1u, abort_flag, j.err, 0x4bfu, P0_SPIN_LIMIT)) tc::mbar_arrive_rank(&qfull, 0);
        }
      } else if (ok) {             // RW rows at a time, 16 bytes a lane; each lane works out the places of four. Zeros beyond the rows
        constexpr uint32_t CH = D < 256 ? D / 8 : 32, RW = 32 / CH;
        uint64_t place[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
          const uint32_t row = rc + 32u * i + lane, tok = row / hpg;
          place[i] = (uint64_t)(u.first + tok) * j.q.ld + (uint64_t)(head * hpg + row - tok * hpg) * j.q.ldh;
        }
#pragma unroll
        for (uint32_t g = 0; g < 4; g++) {
#pragma unroll 4
          for (uint32_t r0 = 0; r0 < 32; r0 += RW) {
            const uint32_t row = 32u * g + r0 + lane / CH;
            const bool there = row < nrow;
            const uint64_t at = __shfl_sync(0xffffffffu, place[g], r0 + lane / CH);
            const __half *q = reinterpret_cast<const __half *>(j.q.base) + (there ? at : 0u);
#pragma unroll
            for (uint32_t d8 = lane % CH; d8 < D / 8; d8 += CH) {
              uint8_t *to = qs + (d8 >> 3) * 16384u + row * 128u + (((d8 & 7u) ^ (row & 7u)) * 16u);
              if (j.q.wide) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(to)), "l"(q + d8 * 8u), "r"(there ? 16u : 0u) : "memory");
              } else {
                uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int i = 0; i < 4; i++)
                  if (there) w[i] = (uint32_t)__half_as_ushort(q[d8 * 8u + 2 * i]) | ((uint32_t)__half_as_ushort(q[d8 * 8u + 2 * i + 1]) << 16);
                *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the generic writes before the MMAs' reads
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_rank(&qfull, 0);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------ softmax: half h of row r
      const bool whole = from == 0 && to == nt;
      if (!whole && from == 0 && tid == 0 && rank == 0) j.desc[run] = make_uint4(1u + run_of(u.begin + u.n - 1u, total, G), b, u.r0, u.head);
      const auto orow = [&](uint32_t r) {   // row r's place in out
        const uint32_t tok = (rc + r) / hpg;
        return (uint64_t)(u.first + tok) * j.out.ld + (uint64_t)(head * hpg + rc + r - tok * hpg) * j.out.ldh + oh * C::kDV;
      };
      if (!tiles) {   // nothing to see: zeros
        for (uint32_t e = tid; e < nrow * C::kDV; e += kSoft) reinterpret_cast<__half *>(j.out.base)[orow(e / C::kDV) + e % C::kDV] = __half();
        continue;
      }
      const uint32_t r = tid & 127u, h = tid >> 7, lanes = ((warp & 3u) * 32u) << 16;
      const int32_t pos = r < nrow ? (int32_t)(u.len - u.T + (rc + r) / hpg) : -1;
      const int32_t pos0 = (int32_t)(u.len - u.T + u.r0 / hpg), pos1 = (int32_t)s.end - 1;   // of the block
      float m = -INFINITY, l = 0.0f;
      const uint32_t *trow = j.v.table + (uint64_t)b * j.v.ld;
      const auto entry = [&](uint32_t i) { return 2u * i + h < s.n ? trow[page_at(s, 2u * i + h)] : P0_KV_NONE; };
      bool ok = true;
      uint32_t next = entry(from);
      for (uint32_t i = 0; i < tiles; i++) {   // a warp that gave up keeps meeting the others at the barrier
        const uint32_t t = tile + i, jp = page_at(s, min(2u * (from + i) + h, s.n - 1u));
        const bool here = next < j.v.pages;
        if (i + 1 < tiles) next = entry(from + i + 1);
        ok = __all_sync(0xffffffffu, ok && tc::mbar_wait(&sfull[t % C::kSB], (t / C::kSB) & 1u, abort_flag, j.err, 0x4b6u, P0_SPIN_LIMIT));
        const uint32_t sc = tmem + lanes + C::kColS + (t % C::kSB) * 128u, pc = tmem + lanes + C::kColP + (t & 1u) * 64u;
        uint32_t x[2][32];
        float mx = -INFINITY;
        if (ok) {
          tc::fence_after();
          tc::tmem_ld32(sc + 64u * h, x[0]);
          tc::tmem_ld32(sc + 64u * h + 32u, x[1]);
          // meanwhile: P of tile t - 2 has been used (before that it lies in a unit whose end was waited for)
          if (i > 1 && !tc::mbar_wait(&odone[t & 1u], ((t >> 1) - 1u) & 1u, abort_flag, j.err, 0x4bbu, P0_SPIN_LIMIT)) ok = false;
          tc::tmem_wait_ld();
          tc::fence_after();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_peer(&sread[t % C::kSB], 0);   // the even CTA's MMAs wait for both
          if (flip)
#pragma unroll
            for (int e = 0; e < 64; e++) x[e >> 5][e & 31] ^= 0x80000000u;
          // keys that this row does not see; a page that the whole block sees needs no look
          const int32_t k0 = (int32_t)(jp * kPage);
          if (!(here && k0 + 63 <= pos0 && (!W || k0 > pos1 - (int32_t)W || (uint32_t)k0 + 63u < S))) {
            // keys up to `gone` are behind the window, those below `sink` are kept all the same
            const int32_t last = here ? pos - k0 : -1, gone = W ? pos - (int32_t)W - k0 : -1;
            const int32_t sink = S > (uint32_t)k0 ? (int32_t)min(S - (uint32_t)k0, kPage) : 0;
            const uint64_t see = first_bits(last + 1) & (~first_bits(gone + 1) | first_bits(sink));
#pragma unroll
            for (int q = 0; q < 2; q++) {
              const uint32_t bits = (uint32_t)(see >> (32 * q));
#pragma unroll
              for (int e = 0; e < 32; e++)
                if (!(bits >> e & 1u)) x[q][e] = 0xff800000u;
            }
          }
          float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int q = 0; q < 2; q++)
#pragma unroll
            for (int e = 0; e < 32; e++) y[e & 3] = fmaxf(y[e & 3], __uint_as_float(x[q][e]));
          mx = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) * c;
          if (mx != mx) mx = -INFINITY;   // -inf times a scale of 0
        }
        mx2[t & 1u][h][r] = mx;
        asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory");
        if (!(ok = __all_sync(0xffffffffu, ok))) continue;
        mx = fmaxf(mx, mx2[t & 1u][h ^ 1u][r]);
        // O follows a maximum whose P would pass 2^15 (or that is a row's first)
        const bool grow = mx > m + 15.0f;
        if (__any_sync(0xffffffffu, grow)) {
          const float to_m = mx - 7.0f, f = grow ? exp2_fast(m - to_m) : 1.0f;
          if (grow) m = to_m;
          l *= f;
          if (i) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&odone[(t - 1u) & 1u], ((t - 1u) >> 1) & 1u, abort_flag, j.err, 0x4b7u, P0_SPIN_LIMIT));
            tc::fence_after();
#pragma unroll 1
            for (uint32_t d = h * (C::kDV / 2); ok && d < (h + 1u) * (C::kDV / 2); d += 32u) {
              uint32_t o[32];
              tc::tmem_ld32(tmem + lanes + d, o);
              tc::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(tmem + lanes + d, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < 2; q++) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float a = exp2_fast(fmaf(__uint_as_float(x[q][2 * e]), c, -ref)), d = exp2_fast(fmaf(__uint_as_float(x[q][2 * e + 1]), c, -ref));
            sum[2 * (e & 1)] += a;
            sum[2 * (e & 1) + 1] += d;
            p[e] = pack2_finite(a, d);
          }
          tc::tmem_st16(pc + 32u * h + 16u * q, p);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tc::tmem_wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_peer(&pfull[t & 1u], 0);
      }
      l2[unit & 1u][h][r] = l;
      asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory");
      l += l2[unit & 1u][h ^ 1u][r];
      if (ok) {
        const uint32_t t = tile + tiles - 1u;
        if (tiles > 1) ok = tc::mbar_wait(&odone[(t - 1u) & 1u], ((t - 1u) >> 1) & 1u, abort_flag, j.err, 0x4bau, P0_SPIN_LIMIT);
        ok = ok && tc::mbar_wait(&odone[t & 1u], (t >> 1) & 1u, abort_flag, j.err, 0x4b8u, P0_SPIN_LIMIT);
        tc::fence_after();
      }
      ok = __all_sync(0xffffffffu, ok);
      float *part = j.part + (((uint64_t)run * 2u + (from ? 0u : 1u)) * 2u + rank) * kCR * (C::kDV + 2);   // [dims][rows], then m and l
      if (ok) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        const uint64_t own = orow(r);
        uint8_t *so = stg + warp * C::kOut;
#pragma unroll 1
        for (uint32_t d = h * (C::kDV / 2); d < (h + 1u) * (C::kDV / 2); d += 32u) {
          uint32_t o[32];
          __syncwarp();
          tc::tmem_ld32(tmem + lanes + d, o);
          tc::tmem_wait_ld();
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 32; e++) part[(d + e) * kCR + r] = __uint_as_float(o[e]);
          } else {   // through shared memory: 8 rows' 64 bytes a store
            uint4 y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; i++) w[i] = pack2(__uint_as_float(o[8 * e + 2 * i]) * inv, __uint_as_float(o[8 * e + 2 * i + 1]) * inv);
              *reinterpret_cast<uint4 *>(so + lane * 80u + e * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) y[k] = *reinterpret_cast<const uint4 *>(so + (8u * k + (lane >> 2)) * 80u + (lane & 3u) * 16u);
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
              const uint32_t row = (warp & 3u) * 32u + 8u * k + (lane >> 2);
              const uint64_t place = __shfl_sync(0xffffffffu, own, 8u * k + (lane >> 2));
              if (row >= nrow) continue;
              __half *out = reinterpret_cast<__half *>(j.out.base) + place + d + 8u * (lane & 3u);
              if (j.out.wide) {
                *reinterpret_cast<uint4 *>(out) = y[k];
              } else {
                const uint32_t w[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
#pragma unroll
                for (int i = 0; i < 8; i++) out[i] = __ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i & 1))));
              }
            }
          }
        }
        if (!whole && h == 0) {
          part[C::kDV * kCR + r] = m;
          part[(C::kDV + 1) * kCR + r] = l;
        }
      }
      tc::fence_before();   // O is read before the next unit's MMAs write it: they wait for this warp's next P
      if (!C::kStg) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the output stood in q's place: before q's next copy
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ofree);
    }
    tile += tiles;
    unit += tiles != 0u;
  }
  __syncthreads();
  if (abort_word && lane == 0) {   // a wait gave up (j.err says which): nothing may be in flight when the CTA leaves. Bounded
    volatile uint32_t never = 0;
    if (warp == 8)
      for (uint32_t i = 0; i < (uint32_t)NS; i++) {
        const Ring &g = i < SK ? rk : rv;
        const uint32_t n = i < SK ? i : i - SK;
        never = 0;   // each one is waited for
        if (g.round || n < g.i) tc::mbar_wait(&full[i], (n < g.i ? g.round : g.round - 1u) & 1u, &never, j.err, 0x4b2u, kDrain);
      }
    if (warp == 11 && j.qbox && unit) tc::mbar_wait(rank ? &qland : &qfull, (unit - 1u) & 1u, &never, j.err, 0x4b2u, kDrain);
    if ((warp == 9 || warp == 10) && rank == 0) {
      tc::mma_commit_pair(&mdone[warp - 9]);
      tc::mbar_wait(&mdone[warp - 9], 0, &never, j.err, 0x4b5u, kDrain);
    }
  }
  __syncwarp();
  tc::fence_before();
  tc::cluster_sync();   // neither CTA frees its tensor memory or exits while the other may still use it
  if (warp == 8) {
    tc::fence_after();
    tc::tmem_dealloc_pair(tmem, 512);
  }
}

// joins the parts of a unit that several runs share: CTA (run, 8 dims, 128 of the rows), a thread per row and every kJoin-th part,
// then those in order. M = max m, o = sum 2^(m - M) acc / sum 2^(m - M) l
template <int D, uint32_t kJoin>
__global__ void __launch_bounds__(kCR *kJoin) kv4_prompt_join_kernel(AttnJob j) {
  dep_enter();
  const uint4 w = j.desc[blockIdx.x];
  if (!w.x) return;
  constexpr uint32_t DV = Cfg<D>::kDV;
  __shared__ float got[kJoin][10][kCR];
  const uint32_t r = threadIdx.x % kCR, g = threadIdx.x / kCR, d0 = blockIdx.y * 8u, rank = blockIdx.z, b = w.y, r0 = w.z + rank * kCR, hpg = j.hpg;
  const uint32_t head = w.w / Cfg<D>::kParts, oh = w.w % Cfg<D>::kParts, n = w.x - blockIdx.x;
  uint32_t first;
  const uint32_t T = kv_tokens(j.v, b, first);
  const bool here = r0 + r < T * hpg;
  const auto part = [&](uint32_t i) { return j.part + (((uint64_t)(blockIdx.x + i) * 2u + (i ? 0u : 1u)) * 2u + rank) * kCR * (DV + 2) + r; };
  float M = -INFINITY, acc[8], sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) acc[e] = 0.0f;
  if (here) {
#pragma unroll 8
    for (uint32_t i = g; i < n; i += kJoin) M = fmaxf(M, part(i)[DV * kCR]);
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll 4
    for (uint32_t i = g; i < n; i += kJoin) {
      const float *p = part(i);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = p[(d0 + e) * kCR];
      const float f = exp2f(p[DV * kCR] - ref);
      sum = fmaf(f, p[(DV + 1) * kCR], sum);
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] = fmaf(f, x[e], acc[e]);
    }
  }
  if (g) {
#pragma unroll
    for (int e = 0; e < 8; e++) got[g][e][r] = acc[e];
    got[g][8][r] = sum;
    got[g][9][r] = M;
  }
  __syncthreads();
  if (g || !here) return;
  float all = M;
#pragma unroll
  for (uint32_t i = 1; i < kJoin; i++) all = fmaxf(all, got[i][9][r]);
  const float ref = all == -INFINITY ? 0.0f : all, f0 = exp2f(M - ref);
  sum *= f0;
#pragma unroll
  for (int e = 0; e < 8; e++) acc[e] *= f0;
#pragma unroll
  for (uint32_t i = 1; i < kJoin; i++) {
    const float f = exp2f(got[i][9][r] - ref);
    sum = fmaf(f, got[i][8][r], sum);
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = fmaf(f, got[i][e][r], acc[e]);
  }
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  __half *out = reinterpret_cast<__half *>(j.out.base) + (uint64_t)(first + (r0 + r) / hpg) * j.out.ld + (uint64_t)(head * hpg + (r0 + r) % hpg) * j.out.ldh + oh * DV + d0;
  uint32_t y[4];
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = pack2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if (j.out.wide) {
    *reinterpret_cast<uint4 *>(out) = make_uint4(y[0], y[1], y[2], y[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) out[e] = __ushort_as_half((unsigned short)(y[e / 2] >> (16 * (e & 1))));
  }
}

// whether the workspace has this much scratch, or the device the memory for it (as far as one can tell before asking): the one that
// is there is not given up in vain
bool room_for(p0_ctx *c, uint64_t scratch) {
  const uint64_t need = c->ws_cnt_bytes + scratch;
  if (need <= c->ws_bytes) return true;
  size_t left = 0, all = 0;
  if (cudaMemGetInfo(&left, &all) != cudaSuccess) { cudaGetLastError(); return true; }
  return need + (16ull << 20) <= (uint64_t)left + c->ws_bytes;
}

// *taken stays false where there is no memory for the pages as f16: the form for few rows needs none
template <int D>
p0_status prompt_launch(p0_ctx *c, AttnJob &j, uint64_t wide_bytes, bool *taken) {
  using C = Cfg<D>;
  const uint32_t R = j.v.rows, G = (uint32_t)c->sm_count / 2;
  const size_t smem = C::kSmem + ((size_t)R + 1) * 8;
  uint32_t *cnt;
  void *ws;
  const size_t desc = ((size_t)G * sizeof(uint4) + 255) / 256 * 256, parts = ((size_t)G * 2 * kRB * (C::kDV + 2) * 4 + 255) / 256 * 256;
  // in place and with the output in parts, a unit writes where another reads q: both work from a copy
  const bool in_place = C::kParts > 1 && j.q.base == j.out.base;
  const uint64_t q_bytes = ((uint64_t)(j.v.n - 1) * j.q.ld + (uint64_t)(j.hpg * j.v.nkv - 1) * j.q.ldh + D) * 2u;
  const uint64_t scratch = desc + parts + wide_bytes + (in_place ? q_bytes : 0u);
  if (!room_for(c, scratch)) return P0_OK;
  p0_status st = p0_workspace(c, 0, scratch, &cnt, &ws);
  if (st == P0_ENOMEM) return P0_OK;
  *taken = true;
  if (st) return st;
  j.units = j.v.nkv * C::kParts;
  if (in_place) {
    uint8_t *copy = (uint8_t *)ws + desc + parts + wide_bytes;
    if ((st = p0_cuda(c, cudaMemcpyAsync(copy, j.q.base, q_bytes, cudaMemcpyDeviceToDevice, c->stream), "kv4Attn in place"))) return st;
    j.q.base = copy;
  }
  j.desc = (uint4 *)ws;
  j.part = (float *)((uint8_t *)ws + desc);
  j.wide = (uint8_t *)ws + desc + parts;
  const auto kern = kv4_prompt_kernel<D>;
  // q as [tokens][heads][dims]: where 128 rows are whole tokens' heads, or some of one token's, a block is a box of it
  CUtensorMap qm = {};
  const auto encode = tensor_map_encoder();
  if (encode && j.q.wide && (j.hpg & (j.hpg - 1u)) == 0u) {
    const uint32_t heads = j.hpg < kCR ? j.hpg : kCR;
    const cuuint64_t size[3] = {(cuuint64_t)D, (cuuint64_t)j.hpg * j.v.nkv, j.v.n}, stride[2] = {(cuuint64_t)j.q.ldh * 2u, (cuuint64_t)j.q.ld * 2u};
    const cuuint32_t box[3] = {64, heads, kCR / heads}, one[3] = {1, 1, 1};
    j.qbox = encode(&qm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<uint8_t *>(j.q.base), size, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) { cudaGetLastError(); return p0_fail(c, P0_EDEVICE, "kv4Attn: the prompt kernel does not fit this device"); }
  launch_dep(kv4_widen_kernel<D>, dim3((unsigned)c->sm_count * 4u), dim3(kET), ((size_t)R + 1) * 4, c->stream, j);
  if ((st = p0_launched(c, "kv4Attn pages"))) return st;
  launch_dep(kern, dim3(2 * G), dim3(kThreads), smem, c->stream, j, qm);
  if ((st = p0_launched(c, "kv4Attn prompt"))) return st;
  // four threads a row where units are in many parts (16 rows' heads of 30000 keys, D = 256: 57 us with one, 45 with four), one
  // where they are in two or three (3 x 2048 of 5003 tokens: 110 with one, 126 with four)
  const uint64_t units = ((uint64_t)j.v.n * j.hpg / kRB + 1u) * j.units;
  if (units * 4u <= G) launch_dep(kv4_prompt_join_kernel<D, 4>, dim3(G, C::kDV / 8, 2), dim3(kCR * 4), 0, c->stream, j);
  else launch_dep(kv4_prompt_join_kernel<D, 1>, dim3(G, C::kDV / 8, 2), dim3(kCR), 0, c->stream, j);
  return p0_launched(c, "kv4Attn join");
}

}  // namespace

// Taken where the sequences have 64 query rows a KV head on average (128 at 512 dims): one sequence of 1200 keys, 64 rows of 256
// dims, 22 us against 32 of the form for few rows; 24 of 6000 keys, 70 against 76; 32 rows of 1200 keys, 23 against 19. (One
// sequence of 30000 keys and 64 rows: 46 against 50; 512 dims, 24 of 6000, 64 rows: 165 against 114, 256 rows: 152 against 269.)
// And where the pages that the call may see take no more than 4 GB as f16: of each sequence all that its table row holds, or with a
// window those of the sinks, of the window before its first new token, and of its new tokens (T / 64 and a page's ends more).
p0_status kv4_attn_prompt(p0_ctx *c, AttnJob &j, bool *taken) {
  *taken = false;
  const uint64_t rows = (uint64_t)j.v.n * j.hpg, D = j.v.D, R = j.v.rows;
  if (rows / R < (D == 512 ? 128 : 64) || R > 256) return P0_OK;
  uint64_t pages = R * j.v.ld;
  if (j.window) {
    const uint64_t seen = R * ((j.sinks + kPage - 1) / kPage + j.window / kPage + 3u) + j.v.n / kPage;
    if (seen < pages) pages = seen;
  }
  const uint64_t wide = pages * j.v.nkv * D * 256;
  if (wide > (4ull << 30)) return P0_OK;
  switch (D) {
    case 64: return prompt_launch<64>(c, j, wide, taken);
    case 128: return prompt_launch<128>(c, j, wide, taken);
    case 256: return prompt_launch<256>(c, j, wide, taken);
    default: return prompt_launch<512>(c, j, wide, taken);
  }
}
