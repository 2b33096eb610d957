// f8_mid.cu -- gemmF8 on tcgen05 where tokens are few or tiles too few for f8_tc.cu: bound by the weights' bytes.
//
// A CTA computes 128 weight rows (gated: of w and of u) times TN tokens: weights are the MMA's rows, so that tensor cores and sums do
// the work of TN tokens, not of 128. Per block of 128 k one warp brings the weights' rows and the tokens' (TMA, 128-byte swizzle), one
// issues four MMAs (128 x TN x 32) into tensor memory, one brings the block's TN scales of x (cp.async, 4 bytes
// each: they need no alignment), and four warps a matrix add the block's sums to those in their registers: TN tokens of a weight row to a
// thread, each times xs[b, m] * ws[n / 128, b].
// A cluster of S CTAs shares a tile's blocks of k. Each leaves its sums in its shared memory as [token][row]; then a warp takes a
// token's 128 columns, adds the S parts in order (over distributed shared memory) and stores them; of a gated call it knows all 128
// columns of the block of codes.
// 16 tokens, 8192 x 2048: 7.4 us, of which the weights take 2.6 at the copy rate (the loop runs at it: 620 cycles a block over 128 CTAs) and 5 go by
// before the first block and after the last, in the cluster's barriers most of all; 8192 x 8192: 15.6 us, 4.3 TB/s. 100 tokens, 6720 x 2240: 10.8 us. Groups
// of blocks (64 sums to a wait) took 64 tokens from 10.0 to 9.4 us (now 8.9), eight warps for 128 tokens 8192 x 8192 from 24.1 to 22.3 (now 21.9).
#include "f8_gemm.cuh"

namespace {

using namespace f8tc;

constexpr uint32_t kW = 128 * 128;        // a stage's rows of one matrix
constexpr uint32_t kScales = 4;           // groups of blocks whose scales are on their way

template <int TN, int MATS>
struct Cfg {
  static constexpr uint32_t kParts = TN == 128 ? 2 : 1;    // of a matrix's tokens: 64 at most to a thread
  static constexpr uint32_t kSets = MATS * kParts, kThreads = 128 + 128 * kSets;   // warps 0: copies; 1: MMAs; 2: scales; 3: none; then four a part: sums
  static constexpr uint32_t kStage = MATS * kW + TN * 128, kFit = 200u * 1024 / kStage, kStages = kFit < 6 ? kFit : 6;
  static constexpr uint32_t kTile = TN * 512;              // a matrix's sums as f32
  static constexpr uint32_t kG = TN < 64 ? 64 / TN : 1;    // blocks of a group: its sums are waited for and read at once
  static constexpr uint32_t kSmem = 1024 + kStages * kStage;
  static constexpr uint32_t kCols = 2 * kG * TN * MATS;
  static_assert(MATS * kTile <= kStages * kStage, "the sums take the ring's place");
};

struct MidJob {
  GemmJob j;
  F8Mat y;              // gated: the codes
  uint32_t nblk, S;     // blocks of 128 rows; CTAs that share a tile's k
  bool wide;            // four columns of y can be stored at once
  uint32_t *err;
};

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 4 bytes to shared memory, zeros where there is nothing
__device__ __forceinline__ void copy4(void *dst, const void *src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(there ? 4u : 0u) : "memory");
}
// this thread's arrival once its copies so far have landed
__device__ __forceinline__ void copies_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float4 remote4(const void *p, uint32_t rank) {
  float4 v;
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n}"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(tc::smem_u32(p)), "r"(rank)
               : "memory");
  return v;
}
// or zeros: a predicated load, no branch
__device__ __forceinline__ float4 remote4_if(const void *p, uint32_t rank, bool there) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  asm volatile("{\n .reg .b32 a;\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n mapa.shared::cluster.u32 a, %4, %5;\n @p ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n}"
               : "+f"(v.x), "+f"(v.y), "+f"(v.z), "+f"(v.w)
               : "r"(tc::smem_u32(p)), "r"(rank), "r"((uint32_t)there)
               : "memory");
  return v;
}
template <int TN, int MATS>
__global__ void __launch_bounds__(Cfg<TN, MATS>::kThreads, 1)
    f8_mid_kernel(MidJob q, const __grid_constant__ CUtensorMap xm, const __grid_constant__ CUtensorMap wm, const __grid_constant__ CUtensorMap um) {
  using C = Cfg<TN, MATS>;
  constexpr uint32_t NS = C::kStages, G = C::kG;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ __align__(16) float scales[kScales][G * TN];
  __shared__ __align__(8) uint64_t full[NS], empty[NS], sfull[kScales], sread[kScales], dfull[2], dread[2], mdone;
  __shared__ uint32_t tmem_slot, abort_word;
  volatile uint32_t *abort_flag = &abort_word;
  const GemmJob &j = q.j;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, S = q.S, rank = blockIdx.x % S, tile = blockIdx.x / S;
  const uint32_t nb = tile % q.nblk, n0 = nb * 128u, m0 = tile / q.nblk * TN;
  const uint32_t k_lo = (uint32_t)((uint64_t)j.KB * rank / S), k_hi = (uint32_t)((uint64_t)j.KB * (rank + 1u) / S);
  if (tid == 0) {
    for (uint32_t i = 0; i < NS; i++) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (uint32_t i = 0; i < kScales; i++) {
      tc::mbar_init(&sfull[i], 32);
      tc::mbar_init(&sread[i], 4 * C::kSets);
    }
    for (uint32_t i = 0; i < 2; i++) {
      tc::mbar_init(&dfull[i], 1);
      tc::mbar_init(&dread[i], 4 * C::kSets);
    }
    tc::mbar_init(&mdone, 1);
    abort_word = 0u;
    tc::fence_mbar_init();
  }
  if (warp == 0) {
    if (elect()) {   // the maps are this launch's own
      tc::prefetch_tmap(&wm);
      tc::prefetch_tmap(&xm);
      if (MATS == 2) tc::prefetch_tmap(&um);
    }
    __syncwarp();
    tc::tmem_alloc(&tmem_slot, C::kCols);
    tc::tmem_relinquish();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_slot;
  dep_enter();
  uint32_t issued = 0;
  bool ok = true;
  if (warp == 0) {
    // ------------------------------------------------------------ copies
    for (uint32_t kb = k_lo; kb < k_hi; kb++) {
      const uint32_t i = kb - k_lo, s = i % NS;
      if (i >= NS && !(ok = warp_wait(&empty[s], (i / NS & 1u) ^ 1u, abort_flag, q.err, 0x8a1u, j.polls[0]))) break;
      if (elect()) {
        uint8_t *to = ring + s * C::kStage;
        tc::mbar_expect_tx(&full[s], C::kStage);
        tc::tma_load_2d(to, &wm, &full[s], (int32_t)(kb * 128u), (int32_t)n0);
        if (MATS == 2) tc::tma_load_2d(to + kW, &um, &full[s], (int32_t)(kb * 128u), (int32_t)n0);
        tc::tma_load_2d(to + MATS * kW, &xm, &full[s], (int32_t)(kb * 128u), (int32_t)m0);
      }
      __syncwarp();
      issued++;
    }
    // the CTA does not leave before the last MMAs have signalled that their stages are free
    if (ok && lane < NS && lane < issued) tc::mbar_wait(&empty[lane], ((issued - 1u - lane) / NS) & 1u, abort_flag, q.err, 0x8a6u, P0_SPIN_LIMIT);
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs
    constexpr uint32_t idesc = tc::idesc_f16_f32(128, TN);   // e4m3 has the format number 0, too
    for (uint32_t kb = k_lo; kb < k_hi; kb++) {
      const uint32_t i = kb - k_lo, s = i % NS, grp = i / G, b = grp & 1u, in = i % G;
      if (!(ok = warp_wait_two(&full[s], i / NS & 1u, in == 0u && grp >= 2u ? &dread[b] : nullptr, ((grp >> 1) - 1u) & 1u, abort_flag, q.err, 0x8a2u, P0_SPIN_LIMIT))) break;
      tc::fence_after();
      if (elect()) {
        const uint64_t xd = tc::desc_sw128(tc::smem_u32(ring + s * C::kStage + MATS * kW));
#pragma unroll
        for (uint32_t a = 0; a < MATS; a++) {
          const uint64_t wd = tc::desc_sw128(tc::smem_u32(ring + s * C::kStage + a * kW));
#pragma unroll
          for (uint32_t e = 0; e < 4; e++) mma_f8(tmem + ((b * MATS + a) * G + in) * TN, wd + e * 2u, xd + e * 2u, idesc, e != 0u);
        }
        if (in == G - 1u || kb + 1u == k_hi) tc::mma_commit(&dfull[b]);
        tc::mma_commit(&empty[s]);
      }
      __syncwarp();
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ x's scales
    for (uint32_t kb = k_lo, grp = 0; kb < k_hi; kb += G, grp++) {
      const uint32_t s = grp % kScales;
      if (!(ok = warp_wait(&sread[s], (grp / kScales & 1u) ^ 1u, abort_flag, q.err, 0x8a4u, j.polls[0]))) break;
#pragma unroll
      for (uint32_t e = lane; e < G * TN; e += 32u) {
        const uint32_t k = kb + e / TN, t = e % TN;
        const bool there = m0 + t < j.M && k < k_hi;
        copy4(&scales[s][e], there ? j.x.s + (uint64_t)k * j.x.s_ld + m0 + t : j.x.s, there);
      }
      copies_arrive(&sfull[s]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= 4) {
    // ------------------------------------------------------------ sums: row r of matrix a, tokens t0 .. t0 + TW - 1
    constexpr uint32_t TW = TN / C::kParts;
    const uint32_t set = (warp >> 2) - 1u, a = set / C::kParts, t0 = set % C::kParts * TW, r = (warp & 3u) * 32u + lane;
    const uint32_t base = tmem + (((warp & 3u) * 32u) << 16) + a * G * TN + t0;
    const float *ws = a ? j.u.s + (uint64_t)nb * j.u.s_ld : j.w.s + (uint64_t)nb * j.w.s_ld;
    uint64_t acc[TW / 2];   // pairs of tokens
    float w[G], wn[G];
#pragma unroll
    for (int e = 0; e < TW / 2; e++) acc[e] = 0ull;
#pragma unroll
    for (uint32_t g = 0; g < G; g++) wn[g] = k_lo + g < k_hi ? ws[k_lo + g] : 0.0f;
    bool hot = false;   // the next group's sums and scales were seen
    for (uint32_t kb = k_lo, grp = 0; kb < k_hi; kb += G, grp++) {
      const uint32_t s = grp % kScales, b = grp & 1u;
#pragma unroll
      for (uint32_t g = 0; g < G; g++) {
        w[g] = wn[g];
        if (kb + G + g < k_hi) wn[g] = ws[kb + G + g];
      }
      if (!__all_sync(0xffffffffu, hot) && !(ok = warp_wait_two(&dfull[b], (grp >> 1) & 1u, &sfull[s], grp / kScales & 1u, abort_flag, q.err, 0x8a5u, P0_SPIN_LIMIT))) break;
      tc::fence_after();
#pragma unroll
      for (uint32_t c0 = 0; c0 < G * TW; c0 += 64u) {
        uint32_t d[2][32];
        tc::tmem_ld32(base + b * MATS * G * TN + c0, d[0]);
        tc::tmem_ld32(base + b * MATS * G * TN + c0 + 32u, d[1]);
        tc::tmem_wait_ld();
        if (c0 + 64u == G * TW) {
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&dread[b]);
          hot = tc::mbar_test(&dfull[b ^ 1u], ((grp + 1u) >> 1) & 1u) && tc::mbar_test(&sfull[(grp + 1u) % kScales], (grp + 1u) / kScales & 1u);
        }
#pragma unroll
        for (uint32_t e = 0; e < 64u; e += 4u) {
          const uint32_t g = (c0 + e) / TW, t = (c0 + e) % TW;
          if (G > 1u && kb + g >= k_hi) break;   // a last group may be short
          const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(&scales[s][t0 + c0 + e]);
          const uint32_t *v = &d[e >> 5][e & 31u];
          fma2(acc[t / 2], pair(v[0], v[1]), mul2(x.x, twice(w[g])));
          fma2(acc[t / 2 + 1], pair(v[2], v[3]), mul2(x.y, twice(w[g])));
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sread[s]);
    }
    // the last block's sums were waited for, so every copy has landed and every MMA has read it: the ring is free
    if (ok) {
      float *to = reinterpret_cast<float *>(ring + a * C::kTile) + t0 * 128u + r;
#pragma unroll
      for (int e = 0; e < TW / 2; e++) {
        float lo, hi;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(acc[e]));
        to[2 * e * 128] = lo;
        to[(2 * e + 1) * 128] = hi;
      }
    }
  }
  __syncthreads();
  const bool failed = abort_word != 0u;
  if (failed) {   // a wait gave up (q.err says which): nothing may be in flight when the CTA leaves. Bounded
    volatile uint32_t never = 0;
    if (warp == 0 && lane == 0)
      for (uint32_t i = 0; i < NS && i < issued; i++) {
        const uint32_t last = (issued - 1u - i) / NS * NS + i;   // the last use of stage i
        never = 0;
        tc::mbar_wait(&full[i], (last / NS) & 1u, &never, q.err, 0x18a7u, kDrain);
      }
    if (warp == 1) {   // a commit is for what its own thread issued: the elected one, as above
      if (elect()) tc::mma_commit(&mdone);
      __syncwarp();
      warp_wait(&mdone, 0, &never, q.err, 0x18a8u, kDrain);
    }
  }
  __syncwarp();
  tc::fence_before();
  if (S > 1u) tc::cluster_sync();   // every part is in place
  else __syncthreads();
  tc::fence_after();
  if (warp == 0) tc::tmem_dealloc(tmem, C::kCols);
  // a token's 128 columns a warp, four a lane
  constexpr uint32_t U = 4;   // tokens whose parts are on their way at once
  const uint32_t stride = S * (C::kThreads / 32u), mend = min((uint32_t)TN, j.M - m0);
  for (uint32_t t0 = rank + S * warp; t0 < mend && !failed; t0 += U * stride) {
    float sums[U][MATS][4];
#pragma unroll
    for (uint32_t i = 0; i < U; i++)
#pragma unroll
      for (uint32_t a = 0; a < MATS; a++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) sums[i][a][e] = 0.0f;
    const auto add = [&](auto part) {   // of token i and matrix a
      float4 p[U][MATS];
#pragma unroll
      for (uint32_t i = 0; i < U; i++)
#pragma unroll
        for (uint32_t a = 0; a < MATS; a++)
          p[i][a] = part(reinterpret_cast<const float *>(ring + a * C::kTile) + min(t0 + i * stride, mend - 1u) * 128u + lane * 4u, t0 + i * stride < mend);
#pragma unroll
      for (uint32_t i = 0; i < U; i++)
#pragma unroll
        for (uint32_t a = 0; a < MATS; a++) {
          sums[i][a][0] += p[i][a].x;
          sums[i][a][1] += p[i][a].y;
          sums[i][a][2] += p[i][a].z;
          sums[i][a][3] += p[i][a].w;
        }
    };
    // Another CTA's parts are read only for tokens that there are: those are used, and so have arrived, before this warp comes to the last
    // barrier. Where all U are there nothing is asked (100 tokens, 6720 x 2240: 10.9 us with the predicates throughout, 10.7 to 10.8 so; N = 8192, K = 2048
    // with reads of absent tokens and now: 16 tokens 7.5 and 7.4, 16 gated 11.4 and 10.7, 64 plain 8.7 and 8.9)
    const bool all = S == 1u || t0 + (U - 1u) * stride < mend;
    for (uint32_t z = 0; z < S; z++) {
      if (all) add([=](const float *at, bool) { return S > 1u ? remote4(at, z) : *reinterpret_cast<const float4 *>(at); });
      else add([=](const float *at, bool there) { return remote4_if(at, z, there); });
    }
#pragma unroll
    for (uint32_t i = 0; i < U; i++) {
      const uint32_t t = t0 + i * stride;
      if (t >= mend) break;
      float (&v)[MATS][4] = sums[i];
      const uint32_t n = n0 + lane * 4u, m = m0 + t;
      if (MATS == 2) {
        float a = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          v[0][e] = n + e < j.N ? f8_gate(v[0][e], j.epi) * v[MATS - 1][e] : 0.0f;
          a = fmaxf(a, fabsf(v[0][e]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        a = f8_hold(a);
        const float inv = __fdiv_rn(448.0f, a);
        const uint32_t codes = f8_codes4(v[0][0] * inv, v[0][1] * inv, v[0][2] * inv, v[0][3] * inv);
        uint8_t *to = q.y.q + (uint64_t)m * q.y.ld + n;
        if (n + 4u <= j.N) *reinterpret_cast<uint32_t *>(to) = codes;
        else
          for (uint32_t e = 0; n + e < j.N; e++) to[e] = (uint8_t)(codes >> (8 * e));
        if (lane == 0) q.y.s[(uint64_t)nb * q.y.s_ld + m] = __fdiv_rn(a, 448.0f);
      } else {
        const uint64_t to = (uint64_t)m * j.y_ld + n;
        if (j.bv)
#pragma unroll
          for (uint32_t e = 0; e < 4; e++)
            if (n + e < j.N) v[0][e] += j.bv[n + e];
        if (j.epi == P0_F8EPI_F16) {
          __half *y = reinterpret_cast<__half *>(j.y) + to;
          if (q.wide && n + 4u <= j.N) {
            const __half2 lo = __floats2half2_rn(v[0][0], v[0][1]), hi = __floats2half2_rn(v[0][2], v[0][3]);
            *reinterpret_cast<uint2 *>(y) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
          } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
              if (n + e < j.N) y[e] = __float2half_rn(v[0][e]);
          }
        } else {
          float *y = reinterpret_cast<float *>(j.y) + to;
          if (q.wide && n + 4u <= j.N) {
            *reinterpret_cast<float4 *>(y) = make_float4(v[0][0], v[0][1], v[0][2], v[0][3]);
          } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
              if (n + e < j.N) y[e] = v[0][e];
          }
        }
      }
    }
  }
  __syncwarp();
  // no CTA leaves while another may read its parts. What was read has been used, so there is nothing to release: a barrier that also waits
  // for the stores of y took 0.3 us more
  if (S > 1u) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

template <int TN, int MATS>
p0_status launch(p0_ctx *c, const MidJob &q, uint32_t tiles, const CUtensorMap &xm, const CUtensorMap &wm, const CUtensorMap &um, const char *op) {
  using C = Cfg<TN, MATS>;
  const auto kern = f8_mid_kernel<TN, MATS>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
  if (e != cudaSuccess) return p0_cuda(c, e, op);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * q.S);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = c->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = q.S;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kern, q, xm, wm, um);
  return p0_launched(c, op);
}

uint32_t tokens_of(uint32_t M) { return M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128; }

}  // namespace

// as many CTAs as there are SMs, two blocks of k each at least; clusters of eight wait long for their SMs (128 tokens, N = K = 2048: 23.5 us
// against 8.8 with four)
uint32_t f8_mid_parts(const p0_ctx *c, uint32_t M, uint32_t N, uint32_t KB) {
  const uint32_t TN = tokens_of(M);
  const uint64_t tiles = (uint64_t)((N + 127u) / 128u) * ((M + TN - 1u) / TN);
  uint32_t S = 1;
  while (S < 4u && tiles * S * 2u <= (uint64_t)c->sm_count && KB >= S * 4u) S *= 2u;
  return S;
}

p0_status f8_mid_launch(p0_ctx *c, const GemmJob &j, const F8Mat &y, const char *op) {
  const bool gated = j.epi >= P0_F8EPI_SWIGLU;
  MidJob q{j, y};
  q.nblk = (j.N + 127u) / 128u;
  q.err = c->d_err;
  const uint32_t es = j.epi == P0_F8EPI_F16 ? 2 : 4;
  q.wide = (uintptr_t)j.y % (4 * es) == 0 && j.y_ld % 4 == 0;
  const uint32_t TN = tokens_of(j.M), tiles = q.nblk * ((j.M + TN - 1u) / TN);
  q.S = f8_mid_parts(c, j.M, j.N, j.KB);
  const auto map = [&](CUtensorMap *m, const F8Mat &a, uint64_t rows, uint32_t box) {
    return f8_box_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.q, rows, j.K, a.ld, box);
  };
  CUtensorMap xm, wm, um = {};
  if (!map(&xm, j.x, j.M, TN) || !map(&wm, j.w, j.N, 128) || (gated && !map(&um, j.u, j.N, 128)))
    return p0_fail(c, P0_EDEVICE, "%s: tensor map encode failed", op);
  if (gated) {   // up to 64 tokens
    if (TN == 16) return launch<16, 2>(c, q, tiles, xm, wm, um, op);
    return TN == 32 ? launch<32, 2>(c, q, tiles, xm, wm, um, op) : launch<64, 2>(c, q, tiles, xm, wm, um, op);
  }
  switch (TN) {
    case 16: return launch<16, 1>(c, q, tiles, xm, wm, um, op);
    case 32: return launch<32, 1>(c, q, tiles, xm, wm, um, op);
    case 64: return launch<64, 1>(c, q, tiles, xm, wm, um, op);
    default: return launch<128, 1>(c, q, tiles, xm, wm, um, op);
  }
}
