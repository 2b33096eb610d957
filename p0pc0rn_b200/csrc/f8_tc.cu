// f8_tc.cu -- gemmF8 on tcgen05: the form for many tokens.
//
// A pair of CTAs computes tiles of 256 tokens x 256 columns (gated: 128 of w and the same 128 of u), each CTA 128 of the tokens.
// Per block of 128 k one warp brings 128 rows of x and 128 of weights (64 of each block of columns) as 128-byte rows (TMA, 128-byte
// swizzle), one thread of the even CTA issues the pair's four MMAs (tcgen05, kind::f8f6f4, 256 x 256 x 32) into one of two buffers of
// tensor memory, and eight warps add the block's sums, scaled, to the tile's in their registers: 128 columns of a token to a thread,
// each times xs[b, m] * ws[n / 128, b]. While a tile's results are stored, the next tile's first two blocks are computed.
//
// What bounds it: a block takes 965 cycles where its MMAs take 512. A CTA's two buffers fill tensor memory, and a buffer's round (MMAs, 420
// cycles of commit, wait and arrival, the warps' reading) bounds it at about 700; the warps themselves, two to a scheduler, need 800 to 900: loads
// of 64 columns (90 cycles each), FMAs (284 for both), waits, arrivals, the next scales. Hence the pairs of FMAs (half the instructions to fetch), scales that
// are loaded four blocks ahead, waits that were looked at before, and the waits of the issuing warp at once. 4096 tokens, 12288 x 4096: 203 us
// (2.03 PFLOP/s), 238 in long runs (1.55 GHz at the power limit); 32760, 6720 x 2240: 505 and 595; 1031 gated, 8960 x 2240: 80 us.
#include "f8_gemm.cuh"

namespace {

using namespace f8tc;

constexpr uint32_t kSums = 256, kThreads = kSums + 128;   // warps 0: copies; 1: MMAs; 2: what landed; 3: none (a warpgroup changes its registers as one); 4-11: sums
constexpr uint32_t kBox = 128 * 128, kHalf = 64 * 128, kStage = kBox + 2 * kHalf;
constexpr uint32_t kOut = 2 * 32 * 128;   // a warp's results on their way: two boxes of 32 rows of 128 bytes
constexpr uint32_t kGroup = 8;            // row tiles whose x stays in L2 while the columns pass
template <bool GATED>
struct Cfg {
  static constexpr uint32_t kStages = GATED ? 6 : 5;
  static constexpr uint32_t kSmem = 1024 + kStages * kStage + (GATED ? 0 : kSums / 32 * kOut);
};

struct TcJob {
  GemmJob j;
  F8Mat y;                 // gated: the codes
  uint32_t mt, nt, tiles;  // tiles of 256 tokens, of 256 (gated: 128) columns
  bool wide;               // gated: rows of y start on 32-byte boundaries; else: y is stored by tensor copies
  uint32_t *err;
};

// a 2D tile into this CTA's shared memory, its bytes counted by the even CTA's barrier
__device__ __forceinline__ void tma_load_pair(void *dst, const void *tmap, uint32_t bar, int32_t c0, int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"(tmap), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ uint32_t even_bar(uint64_t *bar) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tc::smem_u32(bar)));
  return r;
}
// a word of CTA `rank` of the pair, at this place in shared memory
__device__ __forceinline__ void store_rank(uint32_t *p, uint32_t rank, uint32_t v) {
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n st.shared::cluster.u32 [a], %2;\n}" ::"r"(tc::smem_u32(p)), "r"(rank), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t load_rank(const uint32_t *p, uint32_t rank) {
  uint32_t v;
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.u32 %0, [a];\n}" : "=r"(v) : "r"(tc::smem_u32(p)), "r"(rank) : "memory");
  return v;
}
// counts bytes on a barrier as a copy would
__device__ __forceinline__ void complete_tx(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(bytes) : "memory");
}
// a 2D tile out of shared memory; rows beyond the matrix are not stored, nor whole 16 bytes beyond a row
__device__ __forceinline__ void tma_store(const void *tmap, const void *src, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tmap), "r"(tc::smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}
// D (+)= A * B of e4m3 codes on the pair, K = 32; one thread of the even CTA issues
__device__ __forceinline__ void mma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void store32(void *p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
               "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// 64 columns of tensor memory as 32 pairs
__device__ __forceinline__ void tmem_ld64(uint32_t t, uint64_t (&d)[32]) {
  asm volatile(
      "{\n .reg .b32 r<64>;\n"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {r0,r1,r2,r3,r4,r5,r6,r7,r8,r9,r10,r11,r12,r13,r14,r15,r16,r17,r18,r19,r20,r21,r22,r23,r24,r25,r26,r27,r28,r29,r30,r31,"
      "r32,r33,r34,r35,r36,r37,r38,r39,r40,r41,r42,r43,r44,r45,r46,r47,r48,r49,r50,r51,r52,r53,r54,r55,r56,r57,r58,r59,r60,r61,r62,r63}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      "mov.b64 %0, {r0,r1};\nmov.b64 %1, {r2,r3};\nmov.b64 %2, {r4,r5};\nmov.b64 %3, {r6,r7};\nmov.b64 %4, {r8,r9};\nmov.b64 %5, {r10,r11};\nmov.b64 %6, {r12,r13};\nmov.b64 %7, {r14,r15};\n"
      "mov.b64 %8, {r16,r17};\nmov.b64 %9, {r18,r19};\nmov.b64 %10, {r20,r21};\nmov.b64 %11, {r22,r23};\nmov.b64 %12, {r24,r25};\nmov.b64 %13, {r26,r27};\nmov.b64 %14, {r28,r29};\nmov.b64 %15, {r30,r31};\n"
      "mov.b64 %16, {r32,r33};\nmov.b64 %17, {r34,r35};\nmov.b64 %18, {r36,r37};\nmov.b64 %19, {r38,r39};\nmov.b64 %20, {r40,r41};\nmov.b64 %21, {r42,r43};\nmov.b64 %22, {r44,r45};\nmov.b64 %23, {r46,r47};\n"
      "mov.b64 %24, {r48,r49};\nmov.b64 %25, {r50,r51};\nmov.b64 %26, {r52,r53};\nmov.b64 %27, {r54,r55};\nmov.b64 %28, {r56,r57};\nmov.b64 %29, {r58,r59};\nmov.b64 %30, {r60,r61};\nmov.b64 %31, {r62,r63};\n}"
      : "=l"(d[0]), "=l"(d[1]), "=l"(d[2]), "=l"(d[3]), "=l"(d[4]), "=l"(d[5]), "=l"(d[6]), "=l"(d[7]), "=l"(d[8]), "=l"(d[9]), "=l"(d[10]), "=l"(d[11]),
        "=l"(d[12]), "=l"(d[13]), "=l"(d[14]), "=l"(d[15]), "=l"(d[16]), "=l"(d[17]), "=l"(d[18]), "=l"(d[19]), "=l"(d[20]), "=l"(d[21]), "=l"(d[22]),
        "=l"(d[23]), "=l"(d[24]), "=l"(d[25]), "=l"(d[26]), "=l"(d[27]), "=l"(d[28]), "=l"(d[29]), "=l"(d[30]), "=l"(d[31])
      : "r"(t)
      : "memory");
}
// tile t: its row and column of tiles. Column by column within groups of kGroup rows
__device__ __forceinline__ uint2 tile_at(const TcJob &q, uint32_t t) {
  const uint32_t per = kGroup * q.nt, grp = t / per, r0 = grp * kGroup, rows = min(kGroup, q.mt - r0), in = t - grp * per;
  return make_uint2(r0 + in % rows, in / rows);
}

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    f8_tc_kernel(TcJob q, const __grid_constant__ CUtensorMap xm, const __grid_constant__ CUtensorMap wm, const __grid_constant__ CUtensorMap um) {
  constexpr uint32_t NS = Cfg<GATED>::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u), *out = ring + NS * kStage;
  // full (even CTA's): both CTAs' rows of a stage are there; ready: that was seen; empty: its MMAs are done; dfull: a block's sums are there;
  // dread: both CTAs' warps have read them
  __shared__ __align__(8) uint64_t full[NS], ready[NS], empty[NS], dfull[2], dread[2], mdone;
  __shared__ uint32_t tmem_slot, abort_word, issued_word, failed_word;   // failed_word: abort_word of either CTA
  __shared__ float peak[GATED ? 2 : 1][2][GATED ? 128 : 1];   // [tile parity][half of the columns][row]
  volatile uint32_t *abort_flag = &abort_word;
  const GemmJob &j = q.j;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = tc::cluster_rank(), first = blockIdx.x >> 1, step = gridDim.x >> 1;
  if (tid == 0) {
    for (uint32_t i = 0; i < NS; i++) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&ready[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&dfull[i], 1);
      tc::mbar_init(&dread[i], 2 * kSums / 32);
    }
    tc::mbar_init(&mdone, 1);
    abort_word = failed_word = 0u;
    tc::fence_mbar_init();
  }
  if (warp == 0) {
    if (elect()) {   // the maps are this launch's own
      tc::prefetch_tmap(&xm);
      tc::prefetch_tmap(&wm);
      if (GATED || q.wide) tc::prefetch_tmap(&um);
    }
    __syncwarp();
    tc::tmem_alloc_pair(&tmem_slot, 512);
    tc::tmem_relinquish_pair();
  }
  tc::fence_before();
  tc::cluster_sync();
  tc::fence_after();
  const uint32_t tmem = tmem_slot;
  dep_enter();
  uint32_t issued = 0;   // stages used so far (copies)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");   // 256 x 232 + 128 x 40 = 384 x 168
    bool ok = true;
    uint32_t s = 0, round = 0;
    if (warp == 0) {
      // ---------------------------------------------------------- copies
      for (uint32_t t = first; t < q.tiles && ok; t += step) {
        const uint2 at = tile_at(q, t);
        const int32_t m0 = (int32_t)(at.x * 256u + rank * 128u), n0 = (int32_t)((GATED ? at.y * 128u : at.y * 256u) + rank * 64u);
        for (uint32_t kb = 0; kb < j.KB; kb++) {
          if (round && !(ok = warp_wait(&empty[s], (round & 1u) ^ 1u, abort_flag, q.err, 0x8f1u, j.polls[rank]))) break;
          if (elect()) {
            if (rank == 0) tc::mbar_expect_tx(&full[s], 2 * kStage);
            const uint32_t bar = even_bar(&full[s]);
            tma_load_pair(ring + s * kStage, &xm, bar, (int32_t)(kb * 128u), m0);
            tma_load_pair(ring + s * kStage + kBox, &wm, bar, (int32_t)(kb * 128u), n0);
            tma_load_pair(ring + s * kStage + kBox + kHalf, GATED ? &um : &wm, bar, (int32_t)(kb * 128u), GATED ? n0 : n0 + 128);
          }
          __syncwarp();
          issued++;
          if (++s == NS) s = 0, round++;
        }
      }
      if (lane == 0) issued_word = issued;
      // the last MMAs signal both CTAs that their stages are free: neither leaves before that has arrived (the results take longer)
      if (ok && lane < NS && lane < issued) tc::mbar_wait(&empty[lane], ((issued - 1u - lane) / NS) & 1u, abort_flag, q.err, 0x8f7u, P0_SPIN_LIMIT);
      __syncwarp();
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- the pair's MMAs
      constexpr uint32_t idesc = tc::idesc_f16_f32(256, 256);   // e4m3 has the format number 0, too
      uint32_t c = 0;
      for (uint32_t t = first; t < q.tiles && ok; t += step)
        for (uint32_t kb = 0; kb < j.KB; kb++, c++) {
          const uint64_t ad = tc::desc_sw128(tc::smem_u32(ring + s * kStage)), bd = tc::desc_sw128(tc::smem_u32(ring + s * kStage + kBox));
          if (!(ok = warp_wait_two(&ready[s], round & 1u, c >= 2u ? &dread[c & 1u] : nullptr, ((c >> 1) - 1u) & 1u, abort_flag, q.err, 0x8f3u, P0_SPIN_LIMIT))) break;
          tc::fence_after();
          if (elect()) {
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) mma_f8_pair(tmem + (c & 1u) * 256u, ad + i * 2u, bd + i * 2u, idesc, i != 0u);
            tc::mma_commit_pair(&dfull[c & 1u]);
            tc::mma_commit_pair(&empty[s]);
          }
          __syncwarp();
          if (++s == NS) s = 0, round++;
        }
    } else if (warp == 2 && rank == 0) {
      // ---------------------------------------------------------- what landed: the odd CTA's copies complete the even one's barrier, so its phases
      // are acquired over the cluster, ahead of the warp whose every wait delays MMAs
      for (uint32_t t = first; t < q.tiles && ok; t += step)
        for (uint32_t kb = 0; kb < j.KB; kb++) {
          if (!(ok = __all_sync(0xffffffffu, tc::mbar_wait_cluster(&full[s], round & 1u, abort_flag, q.err, 0x8f2u, P0_SPIN_LIMIT)))) break;
          if (elect()) tc::mbar_arrive(&ready[s]);
          __syncwarp();
          if (++s == NS) s = 0, round++;
        }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ------------------------------------------------------------ sums: row r of this CTA's, columns 64 h .. + 63 of either block of 128
    const uint32_t r = (warp & 3u) * 32u + lane, h = (warp >> 2) - 1u, base = tmem + (((warp & 3u) * 32u) << 16) + 128u * h;
    const uint32_t KB = j.KB, NB = (j.N + 127u) / 128u;
    // scales ahead of their use: x's of the next four blocks (x[i]: of this tile's next block whose number is i by 4, or if there is none of the next
    // tile's block i), the weights' of 32, one a lane
    float x[4] = {}, wc[2], wn[2] = {};
    uint32_t wt = first, wk = 0;
    const auto row_of = [&](uint32_t t) { return min(tile_at(q, t).x * 256u + rank * 128u + r, j.M - 1u); };
    uint32_t row = 0, row_next = row_of(first);
    const auto ahead_w = [&]() {
      if (wt >= q.tiles) return;
      const uint32_t col = tile_at(q, wt).y;
      if (wk + lane < KB) {
        wn[0] = j.w.s[(uint64_t)(GATED ? col : 2u * col) * j.w.s_ld + wk + lane];
        wn[1] = GATED ? j.u.s[(uint64_t)col * j.u.s_ld + wk + lane] : j.w.s[(uint64_t)min(2u * col + 1u, NB - 1u) * j.w.s_ld + wk + lane];
      }
      if ((wk += 32u) >= KB) wk = 0, wt += step;
    };
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
      if (i < KB) x[i] = j.x.s[(uint64_t)i * j.x.s_ld + row_next];
    ahead_w();
    bool ok = true, hot = false;   // hot: the next block's sums were seen
    uint32_t c = 0, parity = 0;
    for (uint32_t t = first; t < q.tiles; t += step, parity ^= 1u) {
      __syncwarp();
      const uint2 at = tile_at(q, t);
      row = row_next;
      row_next = row_of(t + step < q.tiles ? t + step : t);
      uint64_t sum[2][32];   // pairs of columns
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int i = 0; i < 32; i++) sum[a][i] = 0ull;
#pragma unroll 1
      for (uint32_t k0 = 0; k0 < KB; k0 += 4u) {
        if ((k0 & 31u) == 0u) {
          wc[0] = wn[0];
          wc[1] = wn[1];
          ahead_w();
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
          if (k0 + i >= KB || !ok) break;
          const uint64_t f[2] = {twice(x[i] * __shfl_sync(0xffffffffu, wc[0], (k0 + i) & 31u)), twice(x[i] * __shfl_sync(0xffffffffu, wc[1], (k0 + i) & 31u))};
          const bool here = k0 + i + 4u < KB;
          x[i] = j.x.s[(uint64_t)(here ? k0 + i + 4u : i) * j.x.s_ld + (here ? row : row_next)];
          if (!__all_sync(0xffffffffu, hot)) ok = warp_wait(&dfull[c & 1u], (c >> 1) & 1u, abort_flag, q.err, 0x8f4u, P0_SPIN_LIMIT);
          if (!ok) break;
          tc::fence_after();
#pragma unroll
          for (int a = 0; a < 2; a++) {
            uint64_t d[32];
            tmem_ld64(base + (c & 1u) * 256u + 64u * a, d);
            if (a) {
              tc::fence_before();
              __syncwarp();
              if (lane == 0) tc::mbar_arrive_peer(&dread[c & 1u], 0);
              c++;
              hot = tc::mbar_test(&dfull[c & 1u], (c >> 1) & 1u);
            }
#pragma unroll
            for (int e = 0; e < 32; e++) fma2(sum[a][e], d[e], f[a]);
          }
        }
      }
      float acc[2][64];
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int i = 0; i < 32; i++) asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[a][2 * i]), "=f"(acc[a][2 * i + 1]) : "l"(sum[a][i]));
      const uint32_t mw = at.x * 256u + rank * 128u + (warp & 3u) * 32u, m = mw + lane;   // the warp's first row, this thread's
      if (GATED) {
        const uint32_t n0 = at.y * 128u + 64u * h;
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 64; i++) {
          acc[0][i] = n0 + i < j.N ? f8_gate(acc[0][i], j.epi) * acc[1][i] : 0.0f;
          a = fmaxf(a, fabsf(acc[0][i]));
        }
        peak[parity][h][r] = a;
        asm volatile("bar.sync 1, %0;" ::"n"(kSums) : "memory");
        if (!ok || m >= j.M) continue;
        a = f8_hold(fmaxf(a, peak[parity][h ^ 1u][r]));
        const float inv = __fdiv_rn(448.0f, a);
        uint8_t *row = q.y.q + (uint64_t)m * q.y.ld;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float *v = &acc[0][32 * i + 4 * e];
            w[e] = f8_codes4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
          }
          const uint32_t n = n0 + 32u * i;
          if (n + 32u <= j.N) {
            if (q.wide) {
              store32(row + n, w);
            } else {
              *reinterpret_cast<uint4 *>(row + n) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4 *>(row + n + 16) = make_uint4(w[4], w[5], w[6], w[7]);
            }
          } else {
#pragma unroll
            for (uint32_t e = 0; e < 32; e++)
              if (n + e < j.N) row[n + e] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
          }
        }
        if (h == 0) q.y.s[(uint64_t)at.y * q.y.s_ld + m] = __fdiv_rn(a, 448.0f);
      } else if (ok) {
        if (j.bv)
#pragma unroll
          for (int a = 0; a < 4; a++) {   // a lane loads the bias of one of 32 columns
            const uint32_t n = at.y * 256u + 128u * (a >> 1) + 64u * h + 32u * (a & 1) + lane;
            const float b = n < j.N ? j.bv[n] : 0.0f;
#pragma unroll
            for (int i = 0; i < 32; i++) acc[a >> 1][32 * (a & 1) + i] += __shfl_sync(0xffffffffu, b, i);
          }
        // through shared memory, in boxes of 32 rows of 128 bytes (64 f16 columns, 32 f32), 16-byte chunk i of row r at i ^ (r % 8)
        const bool f16 = j.epi == P0_F8EPI_F16;
        uint8_t *stg = out + (warp - 4u) * kOut;
#pragma unroll
        for (int a = 0; a < 2; a++) {
          const uint32_t n0 = at.y * 256u + 128u * a + 64u * h;
          if (q.wide && lane == 0 && (a == 0 || !f16)) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // what stood there has been read
          __syncwarp();
          if (f16) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const float *v = &acc[a][8 * i];
              *reinterpret_cast<uint4 *>(stg + a * 4096 + lane * 128u + ((i ^ (lane & 7u)) * 16u)) =
                  make_uint4(half2_bits(v[0], v[1]), half2_bits(v[2], v[3]), half2_bits(v[4], v[5]), half2_bits(v[6], v[7]));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; i++)
              *reinterpret_cast<float4 *>(stg + (i >> 3) * 4096 + lane * 128u + (((i & 7) ^ (lane & 7u)) * 16u)) = *reinterpret_cast<const float4 *>(&acc[a][4 * i]);
          }
          if (q.wide) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && mw < j.M) {
              if (f16) {
                if (n0 < j.N) tma_store(&um, stg + a * 4096, (int32_t)n0, (int32_t)mw);
              } else {
                for (uint32_t i = 0; i < 2; i++)
                  if (n0 + 32u * i < j.N) tma_store(&um, stg + i * 4096u, (int32_t)(n0 + 32u * i), (int32_t)mw);
              }
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {   // rows that do not start or end on 16 bytes: a lane a column, row by row
            __syncwarp();
            for (uint32_t row = 0; row < 32u && mw + row < j.M; row++)
#pragma unroll
              for (uint32_t i = 0; i < 2; i++) {
                const uint32_t e = lane + 32u * i;
                if (n0 + e >= j.N) continue;
                const uint64_t to = (uint64_t)(mw + row) * j.y_ld + n0 + e;
                if (f16) reinterpret_cast<__half *>(j.y)[to] = *reinterpret_cast<const __half *>(stg + a * 4096 + row * 128u + (((e >> 3) ^ (row & 7u)) * 16u) + (e & 7u) * 2u);
                else reinterpret_cast<float *>(j.y)[to] = *reinterpret_cast<const float *>(stg + i * 4096u + row * 128u + (((lane >> 2) ^ (row & 7u)) * 16u) + (lane & 3u) * 4u);
              }
            __syncwarp();
          }
        }
      }
    }
    if (!GATED && q.wide && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncthreads();
  if (tid < 2 && abort_word) store_rank(&failed_word, tid, 1u);
  __syncwarp();
  tc::fence_before();
  tc::cluster_sync();   // neither CTA frees its tensor memory or exits while the other may still use it
  if (failed_word) {    // a wait gave up (q.err says which): nothing may be in flight when the pair leaves. Both CTAs' warps have ended their loops. Bounded
    volatile uint32_t never = 0;
    if (warp == 0 && lane == 0 && rank == 0) {
      const uint32_t mine = issued_word, theirs = load_rank(&issued_word, 1);
      for (uint32_t i = 0; i < NS; i++) {
        // uses of stage i. They differ by one at most: a stage is free again for both when its MMAs have read both CTAs' halves
        const uint32_t a = mine > i ? (mine - 1u - i) / NS + 1u : 0u, b = theirs > i ? (theirs - 1u - i) / NS + 1u : 0u;
        if (a > b) complete_tx(&full[i], kStage);             // the odd CTA's half was expected and does not come
        else if (b > a) tc::mbar_expect_tx(&full[i], kStage);   // its half comes, with none from here
        never = 0;
        if (a || b) tc::mbar_wait(&full[i], (max(a, b) - 1u) & 1u, &never, q.err, 0x18f5u, kDrain);
      }
    }
    if (warp == 1) {   // a commit is for what its own thread issued: the elected one, as above. It arrives in both CTAs
      if (rank == 0 && elect()) tc::mma_commit_pair(&mdone);
      __syncwarp();
      warp_wait(&mdone, 0, &never, q.err, 0x18f6u, kDrain);
    }
    __syncwarp();
    tc::cluster_sync();
  }
  if (warp == 0) {
    tc::fence_after();
    tc::tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace

p0_status f8_tc_launch(p0_ctx *c, const GemmJob &j, const F8Mat &y, const char *op) {
  const bool gated = j.epi >= P0_F8EPI_SWIGLU, f16 = j.epi == P0_F8EPI_F16;
  TcJob q{j, y};
  q.mt = (j.M + 255u) / 256u;
  q.nt = gated ? (j.N + 127u) / 128u : (j.N + 255u) / 256u;
  q.tiles = q.mt * q.nt;
  q.err = c->d_err;
  CUtensorMap xm, wm, um = {};   // um: u, or the results
  if (!f8_box_map(&xm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, j.x.q, j.M, j.K, j.x.ld, 128) || !f8_box_map(&wm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, j.w.q, j.N, j.K, j.w.ld, 64) ||
      (gated && !f8_box_map(&um, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, j.u.q, j.N, j.K, j.u.ld, 64)))
    return p0_fail(c, P0_EDEVICE, "%s: tensor map encode failed", op);
  const uint32_t es = f16 ? 2 : 4;
  if (gated) q.wide = (uintptr_t)y.q % 32 == 0 && y.ld % 32 == 0;
  // a tensor copy ends a row in whole 16 bytes: a row that ends inside of them is stored the other way, or what lies behind it would be lost
  else q.wide = (uintptr_t)j.y % 16 == 0 && j.y_ld * es % 16 == 0 && j.N * es % 16 == 0 && f8_box_map(&um, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, es, j.y, j.M, j.N, j.y_ld, 32);
  const auto kern = gated ? f8_tc_kernel<true> : f8_tc_kernel<false>;
  const uint32_t smem = gated ? Cfg<true>::kSmem : Cfg<false>::kSmem, pairs = (uint32_t)c->sm_count / 2u;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return p0_cuda(c, e, op);
  launch_dep(kern, dim3(2u * (q.tiles < pairs ? q.tiles : pairs)), dim3(kThreads), smem, c->stream, q, xm, wm, um);
  return p0_launched(c, op);
}
