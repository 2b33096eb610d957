// f8_gemm.cu -- gemmF8: products of matrices in 8 bits. The entry point, and the form for few tokens.
//
// Y[m, n] = sum over blocks b of 128 k:  (xs[b, m] * ws[n / 128, b]) * sum_{k in b} xc[m, k] wc[n, k].
//
// The factor in brackets is rounded to f32 first, one FMA a block and result. Two multiplications instead where f32 does not hold the
// factor (below 2^-126, beyond 2^128) would need a look at every factor and a second way: 4096 tokens, 12288 x 4096 went from 203 to 238 us,
// 128, 8192 x 8192 from 21.8 to 23.1; hence the bounds that the interface states.
// Few tokens: bound by the weights' bytes. A CTA computes 16 weight rows; its warps take blocks of k in turn, a lane loads 16
// bytes of two rows at a time straight into the fragments of mma.sync.m16n8k32 (e4m3, f32 sums): the order of k inside a
// fragment is free as long as both operands share it, so 16 consecutive bytes serve two instructions. Tokens are the n side,
// loaded the same way. Each block's sums are scaled and added in f32; the warps' parts meet in shared memory, in order.
// 1 token, 2048 x 2048: 3.5 us (launch, a round trip to memory, the join); 8 tokens, 8192 x 2048: 6.1 us, 2.8 TB/s; 8192 x 8192: 16 us, 4.2 TB/s.
#include <cstdlib>

#include "f8_gemm.cuh"

namespace {

constexpr int kT = 256, kW = kT / 32;

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes k .. k + 15 of a row of K (a 16-byte boundary); zeros beyond it
__device__ __forceinline__ uint4 codes16(const uint8_t *row, uint32_t k, uint32_t K) {
  if (k + 16u <= K) return *reinterpret_cast<const uint4 *>(row + k);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  for (uint32_t i = 0; k + i < K; i++) w[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3u));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// NT: groups of 8 tokens
template <int NT>
__global__ void __launch_bounds__(kT) f8_few_kernel(GemmJob j) {
  dep_enter();
  constexpr int kOut = NT * 128;   // token * 16 + row
  __shared__ float red[kW][kOut];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, c = lane & 3u;
  const uint32_t n0 = blockIdx.x * 16u;
  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[t][i] = 0.0f;
  const uint64_t r0 = min(n0 + g, j.N - 1u), r1 = min(n0 + g + 8u, j.N - 1u);   // rows beyond the last: their sums are not stored
#pragma unroll 2
  for (uint32_t kb = warp; kb < j.KB; kb += kW) {
    const uint32_t k = kb * kF8Block + c * 16u;
    uint4 x[NT][2];
    float xs[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const uint32_t m = t * 8u + g;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        x[t][h] = m < j.M ? codes16(j.x.q + (uint64_t)m * j.x.ld, k + h * 64u, j.K) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t mc = t * 8u + 2u * c + h;
        xs[t][h] = mc < j.M ? j.x.s[(uint64_t)kb * j.x.s_ld + mc] : 0.0f;
      }
    }
    uint4 w0[2], w1[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      w0[h] = codes16(j.w.q + r0 * j.w.ld, k + h * 64u, j.K);
      w1[h] = codes16(j.w.q + r1 * j.w.ld, k + h * 64u, j.K);
    }
    const float ws = j.w.s[(uint64_t)(n0 / kF8Block) * j.w.s_ld + kb];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; h++) {
        mma_e4m3(d, w0[h].x, w1[h].x, w0[h].y, w1[h].y, x[t][h].x, x[t][h].y);
        mma_e4m3(d, w0[h].z, w1[h].z, w0[h].w, w1[h].w, x[t][h].z, x[t][h].w);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) acc[t][i] = fmaf(d[i], xs[t][i & 1] * ws, acc[t][i]);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) red[warp][(t * 8 + 2 * c + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[t][i];
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < kOut; e += kT) {
    const uint32_t m = e / 16u, n = n0 + e % 16u;
    if (m >= j.M || n >= j.N) continue;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < kW; w++) y += red[w][e];
    if (j.bv) y += j.bv[n];
    const uint64_t at = (uint64_t)m * j.y_ld + n;
    if (j.epi == P0_F8EPI_F16) reinterpret_cast<__half *>(j.y)[at] = __float2half_rn(y);
    else reinterpret_cast<float *>(j.y)[at] = y;
  }
}

p0_status few_launch(p0_ctx *c, const GemmJob &j, const char *op) {
  const dim3 grid((j.N + 15u) / 16u);
  if (j.M <= 8) launch_dep(f8_few_kernel<1>, grid, dim3(kT), 0, c->stream, j);
  else launch_dep(f8_few_kernel<2>, grid, dim3(kT), 0, c->stream, j);
  return p0_launched(c, op);
}

}  // namespace

extern "C" p0_status p0_gemm_f8(p0_ctx *c, const p0_gemm_f8_args *a) {
  if (!c || !a) return P0_EINVAL;
  const char *op = "gemmF8";
  if (a->epi > P0_F8EPI_GEGLU) return p0_fail(c, P0_EINVAL, "%s: epilogue %u", op, a->epi);
  const bool gated = a->epi >= P0_F8EPI_SWIGLU;
  if (gated && !a->u.buf.id) return p0_fail(c, P0_EINVAL, "%s: a gated epilogue needs u", op);
  if (!gated && a->u.buf.id) return p0_fail(c, P0_EINVAL, "%s: u without a gated epilogue", op);
  if (gated && a->bv.id) return p0_fail(c, P0_EINVAL, "%s: bv with a gated epilogue", op);
  if (!a->M || !a->N) return P0_OK;
  if (!a->K) return p0_fail(c, P0_EINVAL, "%s: K is 0", op);
  const uint64_t M = a->M, N = a->N, K = a->K;
  if (K > (1u << 24) || N > (1u << 24) || M > (1u << 24) || ((N + 15) / 16) * ((M + 7) / 8) >= (1ull << 31))
    return p0_fail(c, P0_EINVAL, "%s: M %u, N %u, K %u", op, a->M, a->N, a->K);
  GemmJob j{};
  j.M = a->M;
  j.N = a->N;
  j.K = a->K;
  j.KB = (a->K + kF8Block - 1) / kF8Block;
  j.epi = a->epi;
  j.polls[0] = j.polls[1] = P0_SPIN_LIMIT;
  if (const char *limit = getenv("P0MM_F8_POLLS")) {   // for tests of what follows a wait that gives up: one limit, or two
    char *odd;
    j.polls[0] = j.polls[1] = (uint32_t)strtoul(limit, &odd, 10);
    if (*odd == ',') j.polls[1] = (uint32_t)strtoul(odd + 1, nullptr, 10);
  }
  p0_status st;
  if ((st = f8_view(c, a->x, M, K, false, op, "x", &j.x))) return st;
  if ((st = f8_view(c, a->w, N, K, true, op, "w", &j.w))) return st;
  if (gated && (st = f8_view(c, a->u, N, K, true, op, "u", &j.u))) return st;
  F8Mat y{};
  uint64_t yn, ysn = 0;
  if (gated) {
    if ((st = f8_view(c, a->y, M, N, false, op, "y", &y))) return st;
    yn = f8_code_bytes(y, M, N);
    ysn = f8_scale_bytes(y, M, N, false);
  } else {
    const uint8_t *p;
    uint32_t ld;
    const uint32_t type = a->epi == P0_F8EPI_F16 ? P0_F16 : P0_F32;
    if ((st = f8_rows(c, a->y.buf, a->y.off, a->y.ld, M, N, type, op, "y", &p, &ld, nullptr))) return st;
    j.y = (uint8_t *)p;
    j.y_ld = ld;
    yn = ((M - 1) * ld + N) * (type == P0_F16 ? 2 : 4);
  }
  P0Range rb;
  if ((st = p0_range(c, a->bv, (uint64_t)a->bv_off * 4, N * 4, op, "bv", &rb, true))) return st;
  if ((uintptr_t)rb.base % 4) return p0_fail(c, P0_EALIGN, "%s: bv must be 4-byte aligned", op);
  j.bv = (const float *)rb.base;
  const void *yp = gated ? (const void *)y.q : (const void *)j.y;
  const auto over = [&](const void *p, uint64_t n) { return f8_meet(yp, yn, p, n) || (ysn && f8_meet(y.s, ysn, p, n)); };
  if (over(j.x.q, f8_code_bytes(j.x, M, K)) || over(j.x.s, f8_scale_bytes(j.x, M, K, false)) || over(j.w.q, f8_code_bytes(j.w, N, K)) ||
      over(j.w.s, f8_scale_bytes(j.w, N, K, true)) || (gated && (over(j.u.q, f8_code_bytes(j.u, N, K)) || over(j.u.s, f8_scale_bytes(j.u, N, K, true)))) ||
      (j.bv && over(j.bv, N * 4)) || (gated && f8_meet(y.q, yn, y.s, ysn)))
    return p0_fail(c, P0_EINVAL, "%s: y must not lie over the inputs", op);
  DeviceGuard guard(c->device);
  // Up to 8 tokens and k of 8192 the form without tensor memory is the faster one (8 tokens, 8192 x 2048: 6.1 us against 7.4; 1 token, 2048 x
  // 16384: 19 against 14.6), for small matrices up to 16 (2048 x 2048: 4.3 against 6.0). f8_mid.cu up to 128 tokens (128, 8192 x 2048: 10.7
  // against 12.6 us of f8_tc.cu) and where its clusters share k, as then few of the other's tiles there are (256, 2048 x 8192: 15.1 against 32.5; 512, 4096 x
  // 2048, where they do not: 14.4 against 12.5). Gated, with twice the stages' bytes, up to 64 (64: 13.9 against 17.1; 100: 29 against 18.6)
  if (!gated && ((M <= 8 && j.KB <= 64) || (M <= 16 && N <= 4096 && j.KB <= 32))) return few_launch(c, j, op);
  if (gated ? M <= 64 : M <= 128 || f8_mid_parts(c, j.M, j.N, j.KB) > 1) return f8_mid_launch(c, j, y, op);
  return f8_tc_launch(c, j, y, op);
}
