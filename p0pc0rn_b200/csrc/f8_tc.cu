// f8_tc.cu -- gemmF8 on tcgen05: the form for many tokens.
//
// A pair of CTAs computes tiles of 256 tokens x 256 columns (gated: 128 of w and the same 128 of u), each CTA 128 of the tokens.
// Per block of 128 k one warp brings 128 rows of x and half of the columns' weights as 128-byte rows (TMA, 128-byte swizzle), one
// thread of the even CTA issues the pair's four MMAs (tcgen05, kind::f8f6f4, 256 x 256 x 32), into one of two buffers of tensor
// memory, and eight warps add the block's sums, scaled, to the tile's in their registers: 128 columns of a token to a thread. The
// scale of a thread's sums is one product, xs[b, m] * ws[n / 128, b], for each 128 columns; x's are loaded two blocks ahead. While a
// tile's results are stored, the next tile's first two blocks are computed.
#include "f8_gemm.cuh"
#include "tc.cuh"

namespace {

constexpr uint32_t kSoft = 256, kThreads = kSoft + 64;   // warps 0-7: sums; 8: copies; 9: MMAs
constexpr uint32_t kStages = 6, kBox = 128 * 128, kStage = 2 * kBox;
constexpr uint32_t kSmem = 1024 + kStages * kStage;
constexpr uint32_t kDrain = 1u << 16;   // polls for what is in flight when a wait has given up
constexpr uint32_t kGroup = 8;          // row tiles whose x stays in L2 while the columns pass

struct TcJob {
  GemmJob j;
  F8Mat y;                 // gated: the codes
  uint32_t mt, nt, tiles;  // tiles of 256 tokens, of 256 (gated: 128) columns
  bool wide;               // rows of y start on 32-byte boundaries
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
// D (+)= A * B of e4m3 codes on the pair, K = 32; one thread of the even CTA issues
__device__ __forceinline__ void mma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// two f32 FMAs: (a0, a1) += (b0, b1) * (s, s)
__device__ __forceinline__ void fma2(float2 &a, uint32_t b0, uint32_t b1, float s) {
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n mov.b64 z, {%0, %1};\n fma.rn.f32x2 z, x, y, z;\n mov.b64 {%0, %1}, z;\n}"
      : "+f"(a.x), "+f"(a.y)
      : "r"(b0), "r"(b1), "f"(s));
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

// tile t: its row and column of tiles. Column by column within groups of kGroup rows
__device__ __forceinline__ uint2 tile_at(const TcJob &q, uint32_t t) {
  const uint32_t per = kGroup * q.nt, grp = t / per, r0 = grp * kGroup, rows = min(kGroup, q.mt - r0), in = t - grp * per;
  return make_uint2(r0 + in % rows, in / rows);
}

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    f8_tc_kernel(TcJob q, const __grid_constant__ CUtensorMap xm, const __grid_constant__ CUtensorMap wm, const __grid_constant__ CUtensorMap um) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  // full (even CTA's): both CTAs' rows of a stage are there; empty: its MMAs are done; dfull: a block's sums are there; dread: both CTAs' warps have read them
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], dfull[2], dread[2], mdone;
  __shared__ uint32_t tmem_slot, abort_word;
  __shared__ float peak[2][2][128];   // gated: [tile parity][half of the columns][row]
  volatile uint32_t *abort_flag = &abort_word;
  const GemmJob &j = q.j;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = tc::cluster_rank(), first = blockIdx.x >> 1, step = gridDim.x >> 1;
  if (tid == 0) {
    for (uint32_t i = 0; i < kStages; i++) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&dfull[i], 1);
      tc::mbar_init(&dread[i], 2 * kSoft / 32);
    }
    tc::mbar_init(&mdone, 1);
    abort_word = 0u;
    tc::fence_mbar_init();
  }
  if (warp == 8) {
    tc::tmem_alloc_pair(&tmem_slot, 512);
    tc::tmem_relinquish_pair();
  }
  tc::fence_before();
  tc::cluster_sync();
  tc::fence_after();
  const uint32_t tmem = tmem_slot;
  dep_enter();
  uint32_t issued = 0;   // stages used so far (copies)
  if (warp == 8) {
    // ------------------------------------------------------------ copies
    if (lane == 0) {
      bool ok = true;
      uint32_t s = 0, round = 0;
      for (uint32_t t = first; t < q.tiles && ok; t += step) {
        const uint2 at = tile_at(q, t);
        const int32_t m0 = (int32_t)(at.x * 256u + rank * 128u), n0 = (int32_t)(GATED ? at.y * 128u : at.y * 256u + rank * 128u);
        for (uint32_t kb = 0; kb < j.KB; kb++) {
          if (!(ok = tc::mbar_wait(&empty[s], (round & 1u) ^ 1u, abort_flag, q.err, 0x8f1u, P0_SPIN_LIMIT))) break;
          if (rank == 0) tc::mbar_expect_tx(&full[s], 2 * kStage);
          const uint32_t bar = even_bar(&full[s]);
          tma_load_pair(ring + s * kStage, &xm, bar, (int32_t)(kb * 128u), m0);
          tma_load_pair(ring + s * kStage + kBox, GATED && rank ? &um : &wm, bar, (int32_t)(kb * 128u), n0);
          issued++;
          if (++s == kStages) s = 0, round++;
        }
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------ the pair's MMAs
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = tc::idesc_f16_f32(256, 256);   // e4m3 has the format number 0, too
      bool ok = true;
      uint32_t s = 0, round = 0, b = 0;
      for (uint32_t t = first; t < q.tiles && ok; t += step)
        for (uint32_t kb = 0; kb < j.KB; kb++, b++) {
          if (!(ok = tc::mbar_wait_cluster(&full[s], round & 1u, abort_flag, q.err, 0x8f2u, P0_SPIN_LIMIT))) break;
          if (b >= 2u && !(ok = tc::mbar_wait(&dread[b & 1u], ((b >> 1) - 1u) & 1u, abort_flag, q.err, 0x8f3u, P0_SPIN_LIMIT))) break;
          tc::fence_after();
          const uint64_t ad = tc::desc_sw128(tc::smem_u32(ring + s * kStage)), bd = tc::desc_sw128(tc::smem_u32(ring + s * kStage + kBox));
#pragma unroll
          for (uint32_t i = 0; i < 4; i++) mma_f8_pair(tmem + (b & 1u) * 256u, ad + i * 2u, bd + i * 2u, idesc, i != 0u);
          tc::mma_commit_pair(&dfull[b & 1u]);
          tc::mma_commit_pair(&empty[s]);
          if (++s == kStages) s = 0, round++;
        }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ sums: row (warp & 3) * 32 + lane, columns 64 h .. + 63 of either half
    const uint32_t r = (warp & 3u) * 32u + lane, h = warp >> 2, base = tmem + (((warp & 3u) * 32u) << 16) + 64u * h;
    const uint32_t NB = (j.N + 127u) / 128u;
    struct Scales {
      float x, w[2];
    } next[2];
    // the scales of block (tile, kb), two ahead of their use
    uint32_t lt = first, lk = 0;
    const float *lx = nullptr, *lw0 = nullptr, *lw1 = nullptr;
    const auto ahead = [&](Scales &s) {
      if (lt >= q.tiles) return;
      if (lk == 0) {
        const uint2 at = tile_at(q, lt);
        lx = j.x.s + min(at.x * 256u + rank * 128u + r, j.M - 1u);
        const uint32_t nb = GATED ? at.y : at.y * 2u;
        lw0 = j.w.s + (uint64_t)nb * j.w.s_ld;
        lw1 = GATED ? j.u.s + (uint64_t)nb * j.u.s_ld : j.w.s + (uint64_t)min(nb + 1u, NB - 1u) * j.w.s_ld;
      }
      s.x = lx[(uint64_t)lk * j.x.s_ld];
      s.w[0] = lw0[lk];
      s.w[1] = lw1[lk];
      if (++lk == j.KB) lk = 0, lt += step;
    };
    next[0] = next[1] = Scales{};
    ahead(next[0]);
    ahead(next[1]);
    bool ok = true;
    uint32_t b = 0, parity = 0;
    for (uint32_t t = first; t < q.tiles; t += step, parity ^= 1u) {
      __syncwarp();
      const uint2 at = tile_at(q, t);
      float2 acc[2][32];
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int i = 0; i < 32; i++) acc[a][i] = make_float2(0.0f, 0.0f);
      for (uint32_t kb = 0; kb < j.KB; kb++, b++) {
        const float f0 = next[0].x * next[0].w[0], f1 = next[0].x * next[0].w[1];
        next[0] = next[1];
        ahead(next[1]);
        ok = __all_sync(0xffffffffu, ok && tc::mbar_wait(&dfull[b & 1u], (b >> 1) & 1u, abort_flag, q.err, 0x8f4u, P0_SPIN_LIMIT));
        if (!ok) break;
        tc::fence_after();
        uint32_t d[2][16];
        tc::tmem_ld16(base + (b & 1u) * 256u, d[0]);
#pragma unroll
        for (int i = 0; i < 8; i++) {   // columns 16 i .. + 15 of the thread's 128
          tc::tmem_wait_ld();
          if (i < 7) tc::tmem_ld16(base + (b & 1u) * 256u + (i + 1 >= 4 ? 128u : 0u) + ((i + 1) & 3) * 16u, d[(i + 1) & 1]);
          const float f = i < 4 ? f0 : f1;
#pragma unroll
          for (int e = 0; e < 8; e++) fma2(acc[i >> 2][(i & 3) * 8 + e], d[i & 1][2 * e], d[i & 1][2 * e + 1], f);
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_peer(&dread[b & 1u], 0);
      }
      const uint32_t m = at.x * 256u + rank * 128u + r;
      if (GATED) {
        const uint32_t n0 = at.y * 128u + 64u * h;
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i++) {
          acc[0][i].x = n0 + 2 * i < j.N ? f8_gate(acc[0][i].x, j.epi) * acc[1][i].x : 0.0f;
          acc[0][i].y = n0 + 2 * i + 1 < j.N ? f8_gate(acc[0][i].y, j.epi) * acc[1][i].y : 0.0f;
          a = fmaxf(a, fmaxf(fabsf(acc[0][i].x), fabsf(acc[0][i].y)));
        }
        peak[parity][h][r] = a;
        asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory");
        if (!ok || m >= j.M) continue;
        a = f8_hold(fmaxf(a, peak[parity][h ^ 1u][r]));
        const float inv = __fdiv_rn(448.0f, a);
        uint8_t *row = q.y.q + (uint64_t)m * q.y.ld;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float2 lo = acc[0][i * 16 + 2 * e], hi = acc[0][i * 16 + 2 * e + 1];
            w[e] = f8_codes4(lo.x * inv, lo.y * inv, hi.x * inv, hi.y * inv);
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
      } else {
        if (!ok || m >= j.M) continue;
#pragma unroll
        for (int a = 0; a < 2; a++) {
          const uint32_t n0 = at.y * 256u + 128u * a + 64u * h;
          if (j.bv)
#pragma unroll
            for (int i = 0; i < 32; i++) {
              acc[a][i].x += n0 + 2 * i < j.N ? j.bv[n0 + 2 * i] : 0.0f;
              acc[a][i].y += n0 + 2 * i + 1 < j.N ? j.bv[n0 + 2 * i + 1] : 0.0f;
            }
          if (j.epi == P0_F8EPI_F16) {
            __half *row = reinterpret_cast<__half *>(j.y) + (uint64_t)m * j.y_ld + n0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; e++) w[e] = half2_bits(acc[a][i * 8 + e].x, acc[a][i * 8 + e].y);
              if (q.wide && n0 + 16u * i + 16u <= j.N) {
                store32(row + 16 * i, w);
              } else {
#pragma unroll
                for (int e = 0; e < 16; e++)
                  if (n0 + 16u * i + e < j.N) row[16 * i + e] = __ushort_as_half((unsigned short)(w[e >> 1] >> (16 * (e & 1))));
              }
            }
          } else {
            float *row = reinterpret_cast<float *>(j.y) + (uint64_t)m * j.y_ld + n0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 4; e++) w[2 * e] = __float_as_uint(acc[a][i * 4 + e].x), w[2 * e + 1] = __float_as_uint(acc[a][i * 4 + e].y);
              if (q.wide && n0 + 8u * i + 8u <= j.N) {
                store32(row + 8 * i, w);
              } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                  if (n0 + 8u * i + e < j.N) row[8 * i + e] = __uint_as_float(w[e]);
              }
            }
          }
        }
      }
    }
  }
  __syncthreads();
  if (abort_word && lane == 0) {   // a wait gave up (q.err says which): nothing may be in flight when the pair leaves. Bounded
    volatile uint32_t never = 0;
    if (warp == 8 && rank == 0)
      for (uint32_t i = 0; i < kStages && i < issued; i++) {
        const uint32_t last = (issued - 1u - i) / kStages * kStages + i;   // the last use of stage i
        never = 0;
        tc::mbar_wait(&full[i], (last / kStages) & 1u, &never, q.err, 0x8f5u, kDrain);
      }
    if (warp == 9 && rank == 0) {
      tc::mma_commit_pair(&mdone);
      tc::mbar_wait(&mdone, 0, &never, q.err, 0x8f6u, kDrain);
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

bool code_map(CUtensorMap *m, const F8Mat &a, uint64_t rows, uint64_t cols) {
  const auto encode = tensor_map_encoder();
  const cuuint64_t size[2] = {cols, rows}, stride[1] = {a.ld};
  const cuuint32_t box[2] = {128, 128}, one[2] = {1, 1};
  return encode && encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a.q, size, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

p0_status f8_tc_launch(p0_ctx *c, const GemmJob &j, const F8Mat &y, const char *op) {
  const bool gated = j.epi >= P0_F8EPI_SWIGLU;
  TcJob q{j, y};
  q.mt = (j.M + 255u) / 256u;
  q.nt = gated ? (j.N + 127u) / 128u : (j.N + 255u) / 256u;
  q.tiles = q.mt * q.nt;
  q.err = c->d_err;
  const uint64_t row_bytes = gated ? y.ld : j.y_ld * (j.epi == P0_F8EPI_F16 ? 2 : 4);
  q.wide = (gated ? (uintptr_t)y.q : (uintptr_t)j.y) % 32 == 0 && row_bytes % 32 == 0;
  CUtensorMap xm, wm, um = {};
  if (!code_map(&xm, j.x, j.M, j.K) || !code_map(&wm, j.w, j.N, j.K) || (gated && !code_map(&um, j.u, j.N, j.K)))
    return p0_fail(c, P0_EDEVICE, "%s: tensor map encode failed", op);
  const auto kern = gated ? f8_tc_kernel<true> : f8_tc_kernel<false>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  if (e != cudaSuccess) return p0_cuda(c, e, op);
  const uint32_t pairs = (uint32_t)c->sm_count / 2u;
  launch_dep(kern, dim3(2u * (q.tiles < pairs ? q.tiles : pairs)), dim3(kThreads), kSmem, c->stream, q, xm, wm, um);
  return p0_launched(c, op);
}
