// f8.cu -- packF8 (values to e4m3 codes with a scale for each block of 128) and normF8 (residual, RMS norm, codes).
//
// Both are bound by memory. Half a warp holds a row's block of 128 columns, eight to a lane: 16-byte loads of f16 (two of f32),
// the block's maximum by four shuffles, 8-byte stores of codes.
#include "f8.cuh"

namespace {

constexpr int kT = 256;

struct Vals {
  float v[8];
};
// x[k .. k + 7] of a row of K; zeros beyond it
template <bool F16, bool WIDE>
__device__ __forceinline__ Vals load8(const void *row, uint32_t k, uint32_t K) {
  Vals r;
  if (WIDE && k + 8u <= K) {
    if (F16) {
      const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const __half *>(row) + k);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        r.v[2 * i] = f.x;
        r.v[2 * i + 1] = f.y;
      }
    } else {
      const float4 a = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(row) + k);
      const float4 b = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(row) + k + 4);
      r.v[0] = a.x, r.v[1] = a.y, r.v[2] = a.z, r.v[3] = a.w, r.v[4] = b.x, r.v[5] = b.y, r.v[6] = b.z, r.v[7] = b.w;
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; i++)
      r.v[i] = k + i >= K ? 0.0f : F16 ? __half2float(reinterpret_cast<const __half *>(row)[k + i]) : reinterpret_cast<const float *>(row)[k + i];
  }
  return r;
}
template <bool F16, bool WIDE>
__device__ __forceinline__ void store8(void *row, uint32_t k, uint32_t K, const Vals &x) {
  if (WIDE && k + 8u <= K) {
    if (F16) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const __half2 h = __floats2half2_rn(x.v[2 * i], x.v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
      *reinterpret_cast<uint4 *>(reinterpret_cast<__half *>(row) + k) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      float *p = reinterpret_cast<float *>(row) + k;
      *reinterpret_cast<float4 *>(p) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
      *reinterpret_cast<float4 *>(p + 4) = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; i++)
      if (k + i < K) {
        if (F16) reinterpret_cast<__half *>(row)[k + i] = __float2half_rn(x.v[i]);
        else reinterpret_cast<float *>(row)[k + i] = x.v[i];
      }
  }
}
// codes of x[k .. k + 7]; rows of codes start on 16-byte boundaries
__device__ __forceinline__ void store_codes(uint8_t *row, uint32_t k, uint32_t K, const Vals &x, float inv) {
  const uint32_t lo = f8_codes4(x.v[0] * inv, x.v[1] * inv, x.v[2] * inv, x.v[3] * inv);
  const uint32_t hi = f8_codes4(x.v[4] * inv, x.v[5] * inv, x.v[6] * inv, x.v[7] * inv);
  if (k + 8u <= K) {
    *reinterpret_cast<uint2 *>(row + k) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; i++)
      if (k + i < K) row[k + i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}
__device__ __forceinline__ float max8(const Vals &x) {
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) a = fmaxf(a, fabsf(x.v[i]));   // fmaxf leaves NaN aside
  return a;
}
// the maximum over half a warp
__device__ __forceinline__ float half_max(float a) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// ---------------------------------------------------------------- packF8, blocks of a row
struct PackJob {
  const uint8_t *x;
  uint64_t ld;
  uint32_t M, K, KB, units;   // units = M * KB
  F8Mat y;
};
template <bool F16, bool WIDE>
__global__ void __launch_bounds__(kT) f8_pack_rows_kernel(PackJob j) {
  dep_enter();
  constexpr uint32_t U = 4;   // blocks of a half warp on their way at once
  const uint32_t l = threadIdx.x & 15u, es = F16 ? 2u : 4u, halves = gridDim.x * (kT / 16);
  for (uint64_t u0 = blockIdx.x * (kT / 16) + (threadIdx.x >> 4); __any_sync(0xffffffffu, u0 < j.units); u0 += (uint64_t)halves * U) {
    Vals x[U];
    uint32_t m[U], kb[U];
#pragma unroll
    for (uint32_t i = 0; i < U; i++) {
      const uint64_t u = u0 + (uint64_t)i * halves;
      const bool here = u < j.units;
      m[i] = here ? (uint32_t)u / j.KB : 0u;
      kb[i] = here ? (uint32_t)u - m[i] * j.KB : j.KB;   // beyond the row: zeros, nothing stored
      x[i] = load8<F16, WIDE>(j.x + (uint64_t)m[i] * j.ld * es, kb[i] * kF8Block + l * 8u, j.K);
    }
#pragma unroll
    for (uint32_t i = 0; i < U; i++) {
      const float a = f8_hold(half_max(max8(x[i])));
      if (kb[i] == j.KB) continue;
      store_codes(j.y.q + (uint64_t)m[i] * j.y.ld, kb[i] * kF8Block + l * 8u, j.K, x[i], __fdiv_rn(448.0f, a));
      if (l == 0) j.y.s[(uint64_t)kb[i] * j.y.s_ld + m[i]] = __fdiv_rn(a, 448.0f);
    }
  }
}

// ---------------------------------------------------------------- packF8, tiles of 128 x 128: one a CTA
template <bool F16, bool WIDE>
__global__ void __launch_bounds__(kT) f8_pack_tiles_kernel(PackJob j) {
  dep_enter();
  __shared__ float red[kT / 32];
  const uint32_t l = threadIdx.x & 15u, es = F16 ? 2u : 4u, nb = blockIdx.x / j.KB, kb = blockIdx.x % j.KB;
  const uint32_t k = kb * kF8Block + l * 8u;
  Vals x[8];
#pragma unroll
  for (uint32_t i = 0; i < 8; i++) {
    const uint32_t m = nb * kF8Block + i * 16u + (threadIdx.x >> 4);
    x[i] = load8<F16, WIDE>(j.x + (uint64_t)min(m, j.M - 1u) * j.ld * es, m < j.M ? k : j.K, j.K);
  }
  float a = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < 8; i++) a = fmaxf(a, max8(x[i]));
  a = half_max(a);
  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 16));
  if ((threadIdx.x & 31u) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kT / 32; i++) a = fmaxf(a, red[i]);
  a = f8_hold(a);
  const float inv = __fdiv_rn(448.0f, a);
#pragma unroll
  for (uint32_t i = 0; i < 8; i++) {
    const uint32_t m = nb * kF8Block + i * 16u + (threadIdx.x >> 4);
    if (m < j.M) store_codes(j.y.q + (uint64_t)m * j.y.ld, k, j.K, x[i], inv);
  }
  if (threadIdx.x == 0) j.y.s[(uint64_t)nb * j.y.s_ld + kb] = __fdiv_rn(a, 448.0f);
}

// ---------------------------------------------------------------- normF8
// tv = the sum of the partial rows in order; with pw: tv * rsqrt(mean tv^2 + eps) * pw; h = (x + tv) * scale, rounded to the
// stream's type; st = rsqrt(mean h^2 + eps); codes of (h * st) * w. A row is held in registers by blockDim.x threads, NB blocks
// to a half warp; blockDim.y rows a CTA.
struct NormJob {
  const uint8_t *x, *t;
  uint8_t *h;
  const float *pw, *w;
  float *st;
  uint64_t x_ld, t_ld, t_ldm, h_ld;
  uint32_t parts, M, D;
  float eps, scale;
  bool store;
  F8Mat y;
};
// the sum of one float per thread over a row's threads
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const uint32_t warps = blockDim.x >> 5;
  if (warps == 1) return v;
  float *r = red + threadIdx.y * warps;
  if ((threadIdx.x & 31u) == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (uint32_t i = 0; i < warps; i++) s += r[i];
  return s;
}
template <bool XF16, bool TF16, bool WIDE, int NB>
__global__ void __launch_bounds__(1024) f8_norm_kernel(NormJob j) {
  dep_enter();
  __shared__ float red[2][32];
  const uint32_t l = threadIdx.x & 15u, half = threadIdx.x >> 4, halves = blockDim.x >> 4;
  const uint32_t m = blockIdx.x * blockDim.y + threadIdx.y;
  const bool here = m < j.M;
  const uint32_t mr = here ? m : j.M - 1u, D = here ? j.D : 0u;   // a row beyond the last one: nothing is read or stored
  const uint8_t *xr = j.x + (uint64_t)mr * j.x_ld * (XF16 ? 2u : 4u);
  Vals h[NB], tv[NB];
#pragma unroll
  for (int b = 0; b < NB; b++) h[b] = load8<XF16, WIDE>(xr, (half + b * halves) * kF8Block + l * 8u, D);
#pragma unroll
  for (int b = 0; b < NB; b++) tv[b] = Vals{};
  for (uint32_t p = 0; p < j.parts; p++) {
    const uint8_t *tr = j.t + ((uint64_t)p * j.t_ld + (uint64_t)mr * j.t_ldm) * (TF16 ? 2u : 4u);
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const Vals t = load8<TF16, WIDE>(tr, (half + b * halves) * kF8Block + l * 8u, D);
#pragma unroll
      for (int i = 0; i < 8; i++) tv[b].v[i] += t.v[i];
    }
  }
  if (j.pw) {
    float s = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 8; i++) s = fmaf(tv[b].v[i], tv[b].v[i], s);
    const float rs = rsqrtf(row_sum(s, red[0]) / (float)j.D + j.eps);
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const Vals w = load8<false, WIDE>(j.pw, (half + b * halves) * kF8Block + l * 8u, D);
#pragma unroll
      for (int i = 0; i < 8; i++) tv[b].v[i] = __fmul_rn(__fmul_rn(tv[b].v[i], rs), w.v[i]);
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; b++) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float v = __fmul_rn(__fadd_rn(h[b].v[i], tv[b].v[i]), j.scale);
      if (XF16) v = __half2float(__float2half_rn(v));
      h[b].v[i] = v;
      s = fmaf(v, v, s);
    }
    if (j.store) store8<XF16, WIDE>(j.h + (uint64_t)mr * j.h_ld * (XF16 ? 2u : 4u), (half + b * halves) * kF8Block + l * 8u, D, h[b]);
  }
  const float st = rsqrtf(row_sum(s, red[1]) / (float)j.D + j.eps);
  if (here && j.st && threadIdx.x == 0) j.st[m] = st;
#pragma unroll
  for (int b = 0; b < NB; b++) {
    const uint32_t kb = half + b * halves, k = kb * kF8Block + l * 8u;
    const Vals w = load8<false, WIDE>(j.w, k, D);
#pragma unroll
    for (int i = 0; i < 8; i++) h[b].v[i] = __fmul_rn(__fmul_rn(h[b].v[i], st), w.v[i]);
    const float a = f8_hold(half_max(max8(h[b])));
    if (kb * kF8Block >= D) continue;
    store_codes(j.y.q + (uint64_t)mr * j.y.ld, k, D, h[b], __fdiv_rn(448.0f, a));
    if (l == 0) j.y.s[(uint64_t)kb * j.y.s_ld + m] = __fdiv_rn(a, 448.0f);
  }
}

template <bool XF16, bool TF16, bool WIDE>
void norm_launch(p0_ctx *c, const NormJob &j) {
  // a step of blockDim.x threads covers 8 columns a thread. Few rows: as many threads a row as it has columns for. Many: two blocks
  // a half warp, rows of up to 512 columns several a CTA
  const uint32_t D = j.D;
  const bool few = j.M <= 2u * (uint32_t)c->sm_count;
  const uint32_t nb = D > 8192 || (!few && D > 256) ? 2u : 1u;
  const uint32_t T = ((D + 8u * nb - 1u) / (8u * nb) + 31u) / 32u * 32u, R = T <= 64 && !few ? 256u / T : 1u;
  const dim3 grid((j.M + R - 1u) / R), block(T, R);
  auto go = [&](auto kern) { launch_dep(kern, grid, block, 0, c->stream, j); };
  if (nb == 1) go(f8_norm_kernel<XF16, TF16, WIDE, 1>);
  else go(f8_norm_kernel<XF16, TF16, WIDE, 2>);
}

void pack_rows_launch(p0_ctx *c, const PackJob &j, bool f16, bool wide) {
  const uint64_t want = ((uint64_t)j.units + kT / 16 - 1) / (kT / 16), most = (uint64_t)c->sm_count * 8u;
  const dim3 grid((unsigned)(want < most ? want : most));
  auto go = [&](auto kern) { launch_dep(kern, grid, dim3(kT), 0, c->stream, j); };
  if (f16) wide ? go(f8_pack_rows_kernel<true, true>) : go(f8_pack_rows_kernel<true, false>);
  else wide ? go(f8_pack_rows_kernel<false, true>) : go(f8_pack_rows_kernel<false, false>);
}

}  // namespace

p0_status f8_rows(p0_ctx *c, p0_buf b, uint64_t off, uint32_t ld, uint64_t rows, uint64_t cols, uint32_t type, const char *op, const char *name,
                  const uint8_t **out, uint32_t *out_ld, bool *wide) {
  const uint64_t es = type == P0_F16 ? 2 : 4, l = ld ? ld : cols;
  if (l < cols) return p0_fail(c, P0_EINVAL, "%s: %s row stride %u < %llu", op, name, ld, (unsigned long long)cols);
  if (off > (1ull << 60)) return p0_fail(c, P0_EINVAL, "%s: %s offset %llu", op, name, (unsigned long long)off);
  P0Range r;
  p0_status st = p0_range(c, b, off * es, ((rows - 1) * l + cols) * es, op, name, &r);
  if (st) return st;
  if ((uintptr_t)r.base % es) return p0_fail(c, P0_EALIGN, "%s: %s must be %u-byte aligned", op, name, (unsigned)es);
  *out = r.base;
  *out_ld = (uint32_t)l;
  if (wide) *wide = (uintptr_t)r.base % 16 == 0 && (rows == 1 || l * es % 16 == 0);
  return P0_OK;
}

p0_status f8_view(p0_ctx *c, const p0_f8 &m, uint64_t rows, uint64_t cols, bool tile, const char *op, const char *name, F8Mat *out) {
  const uint64_t kb = (cols + kF8Block - 1) / kF8Block, nb = (rows + kF8Block - 1) / kF8Block;
  const uint64_t ld = m.ld ? m.ld : (cols + 15) / 16 * 16, s_ld = m.s_ld ? m.s_ld : tile ? kb : (rows + 3) / 4 * 4, s_cols = tile ? kb : rows;
  if (ld < cols) return p0_fail(c, P0_EINVAL, "%s: %s row stride %u < %llu", op, name, m.ld, (unsigned long long)cols);
  if (s_ld < s_cols) return p0_fail(c, P0_EINVAL, "%s: %s.s row stride %u < %llu", op, name, m.s_ld, (unsigned long long)s_cols);
  if (ld % 16) return p0_fail(c, P0_EALIGN, "%s: %s rows must start on 16-byte boundaries (ld %% 16)", op, name);
  if (m.s_off > (1ull << 60)) return p0_fail(c, P0_EINVAL, "%s: %s.s offset %llu", op, name, (unsigned long long)m.s_off);
  P0Range r, s;
  p0_status st;
  if ((st = p0_range(c, m.buf, m.off, (rows - 1) * ld + cols, op, name, &r))) return st;
  if ((uintptr_t)r.base % 16) return p0_fail(c, P0_EALIGN, "%s: %s rows must start on 16-byte boundaries (off)", op, name);
  char sn[48];
  snprintf(sn, sizeof sn, "%s.s", name);
  if ((st = p0_range(c, m.s, m.s_off * 4, (((tile ? nb : kb) - 1) * s_ld + s_cols) * 4, op, sn, &s))) return st;
  if ((uintptr_t)s.base % 4) return p0_fail(c, P0_EALIGN, "%s: %s must be 4-byte aligned", op, sn);
  out->q = (uint8_t *)r.base;
  out->s = (float *)s.base;
  out->ld = (uint32_t)ld;
  out->s_ld = (uint32_t)s_ld;
  return P0_OK;
}

p0_status f8_pack_rows(p0_ctx *c, const float *x, uint64_t ld, uint32_t M, uint32_t K, const F8Mat &y, const char *op) {
  PackJob j{(const uint8_t *)x, ld, M, K, (K + kF8Block - 1) / kF8Block, 0, y};
  j.units = M * j.KB;
  pack_rows_launch(c, j, false, ld % 4 == 0);
  return p0_launched(c, op);
}

extern "C" {

p0_status p0_pack_f8(p0_ctx *c, const p0_pack_f8_args *a) {
  if (!c || !a) return P0_EINVAL;
  const char *op = "packF8";
  if (a->type > P0_F16) return p0_fail(c, P0_EINVAL, "%s: type %u", op, a->type);
  if (a->block > P0_F8_TILE) return p0_fail(c, P0_EINVAL, "%s: block %u", op, a->block);
  if (!a->M || !a->K) return P0_OK;
  const bool tile = a->block == P0_F8_TILE;
  PackJob j{};
  j.M = a->M;
  j.K = a->K;
  j.KB = (a->K + kF8Block - 1) / kF8Block;
  const uint64_t units = (uint64_t)(tile ? (a->M + kF8Block - 1) / kF8Block : a->M) * j.KB;
  if (a->K > (1u << 24) || a->M > (1u << 28) || units >= (1ull << 31)) return p0_fail(c, P0_EINVAL, "%s: %u x %u values", op, a->M, a->K);
  j.units = (uint32_t)units;
  p0_status st;
  uint32_t ld;
  bool wide;
  if ((st = f8_rows(c, a->x, a->x_off, a->x_ld, a->M, a->K, a->type, op, "x", &j.x, &ld, &wide))) return st;
  if ((st = f8_view(c, a->y, a->M, a->K, tile, op, "y", &j.y))) return st;
  j.ld = ld;
  const uint64_t xn = ((uint64_t)(a->M - 1) * ld + a->K) * (a->type == P0_F16 ? 2 : 4), qn = f8_code_bytes(j.y, a->M, a->K), sn = f8_scale_bytes(j.y, a->M, a->K, tile);
  if (f8_meet(j.x, xn, j.y.q, qn) || f8_meet(j.x, xn, j.y.s, sn) || f8_meet(j.y.q, qn, j.y.s, sn))
    return p0_fail(c, P0_EINVAL, "%s: x, y and its scales must not lie over one another", op);
  DeviceGuard guard(c->device);
  const bool f16 = a->type == P0_F16;
  if (!tile) {
    pack_rows_launch(c, j, f16, wide);
    return p0_launched(c, op);
  }
  auto go = [&](auto kern) { launch_dep(kern, dim3(j.units), dim3(kT), 0, c->stream, j); };
  if (f16) wide ? go(f8_pack_tiles_kernel<true, true>) : go(f8_pack_tiles_kernel<true, false>);
  else wide ? go(f8_pack_tiles_kernel<false, true>) : go(f8_pack_tiles_kernel<false, false>);
  return p0_launched(c, op);
}

p0_status p0_norm_f8(p0_ctx *c, const p0_norm_f8_args *a) {
  if (!c || !a) return P0_EINVAL;
  const char *op = "normF8";
  if (a->type > P0_F16) return p0_fail(c, P0_EINVAL, "%s: type %u", op, a->type);
  if (a->t_type > P0_F16) return p0_fail(c, P0_EINVAL, "%s: t.type %u", op, a->t_type);
  if (a->pw.id && !a->t.id) return p0_fail(c, P0_EINVAL, "%s: pw without t", op);
  if (!a->M || !a->D) return P0_OK;
  if (a->D > P0_F8_MAX_D) return p0_fail(c, P0_EINVAL, "%s: D > %u", op, P0_F8_MAX_D);
  if (a->M > (1u << 28)) return p0_fail(c, P0_EINVAL, "%s: %u rows", op, a->M);
  const uint64_t M = a->M, D = a->D, es = a->type == P0_F16 ? 2 : 4, ts = a->t_type == P0_F16 ? 2 : 4;
  NormJob j{};
  p0_status st;
  uint32_t ld;
  bool wide, w1 = true, w2 = true;
  if ((st = f8_rows(c, a->x, a->x_off, a->x_ld, M, D, a->type, op, "x", &j.x, &ld, &wide))) return st;
  j.x_ld = ld;
  const uint64_t xn = ((M - 1) * ld + D) * es;
  uint64_t tn = 0;
  if (a->t.id) {
    const uint64_t n = a->t_n ? a->t_n : 1, ldm = a->t_ldm ? a->t_ldm : D, lp = a->t_ld ? a->t_ld : M * ldm;
    if (ldm < D) return p0_fail(c, P0_EINVAL, "%s: t row stride %u < %u", op, a->t_ldm, a->D);
    if (n > 1024 || lp > (1ull << 40) || a->t_off > (1ull << 60)) return p0_fail(c, P0_EINVAL, "%s: %u partial sums of t, %llu apart", op, a->t_n, (unsigned long long)lp);
    P0Range r;
    tn = ((n - 1) * lp + (M - 1) * ldm + D) * ts;
    if ((st = p0_range(c, a->t, a->t_off * ts, tn, op, "t", &r))) return st;
    if ((uintptr_t)r.base % ts) return p0_fail(c, P0_EALIGN, "%s: t must be %u-byte aligned", op, (unsigned)ts);
    j.t = r.base;
    j.t_ld = lp;
    j.t_ldm = ldm;
    j.parts = (uint32_t)n;
    w1 = (uintptr_t)r.base % 16 == 0 && (M == 1 || ldm * ts % 16 == 0) && (n == 1 || lp * ts % 16 == 0);
  }
  j.scale = a->scale;
  const uint8_t *h = j.x;
  uint32_t h_ld = ld;
  if (a->h.id && (st = f8_rows(c, a->h, a->h_off, a->h_ld, M, D, a->type, op, "h", &h, &h_ld, &w2))) return st;
  j.h = (uint8_t *)h;
  j.h_ld = h_ld;
  const bool in_place = h == j.x && h_ld == ld;
  j.store = !in_place || j.parts || a->scale != 1.0f;
  const uint64_t hn = ((M - 1) * h_ld + D) * es;
  P0Range rw, rp, rs;
  if ((st = p0_range(c, a->w, (uint64_t)a->w_off * 4, D * 4, op, "w", &rw))) return st;
  if ((st = p0_range(c, a->pw, (uint64_t)a->pw_off * 4, D * 4, op, "pw", &rp, true))) return st;
  if ((st = p0_range(c, a->st, (uint64_t)a->st_off * 4, M * 4, op, "st", &rs, true))) return st;
  if ((uintptr_t)rw.base % 4 || (uintptr_t)rp.base % 4 || (uintptr_t)rs.base % 4) return p0_fail(c, P0_EALIGN, "%s: w, pw and st must be 4-byte aligned", op);
  j.w = (const float *)rw.base;
  j.pw = (const float *)rp.base;
  j.st = (float *)rs.base;
  if ((st = f8_view(c, a->y, M, D, false, op, "y", &j.y))) return st;
  // what is written lies over nothing else, but h over x where both are the same rows
  struct { const void *p; uint64_t n; } in[4] = {{j.x, xn}, {j.t, tn}, {j.w, D * 4}, {j.pw, j.pw ? D * 4 : 0}};
  struct { const void *p; uint64_t n; } out[4] = {{j.h, j.store ? hn : 0}, {j.y.q, f8_code_bytes(j.y, M, D)}, {j.y.s, f8_scale_bytes(j.y, M, D, false)}, {j.st, j.st ? M * 4 : 0}};
  for (int o = 0; o < 4; o++) {
    for (int i = 0; i < 4; i++)
      if (out[o].n && in[i].n && !(o == 0 && i == 0 && in_place) && f8_meet(out[o].p, out[o].n, in[i].p, in[i].n))
        return p0_fail(c, P0_EINVAL, "%s: an output lies over an input (h may be x itself)", op);
    for (int i = 0; i < o; i++)
      if (out[o].n && out[i].n && f8_meet(out[o].p, out[o].n, out[i].p, out[i].n)) return p0_fail(c, P0_EINVAL, "%s: two outputs lie over one another", op);
  }
  j.M = a->M;
  j.D = a->D;
  j.eps = a->eps != 0.0f ? a->eps : 1e-6f;
  wide = wide && w1 && w2 && (uintptr_t)j.w % 16 == 0 && (uintptr_t)j.pw % 16 == 0;
  DeviceGuard guard(c->device);
  const bool xf = a->type == P0_F16, tf = a->t_type == P0_F16;
  if (wide) {
    if (xf) tf ? norm_launch<true, true, true>(c, j) : norm_launch<true, false, true>(c, j);
    else tf ? norm_launch<false, true, true>(c, j) : norm_launch<false, false, true>(c, j);
  } else {
    if (xf) tf ? norm_launch<true, true, false>(c, j) : norm_launch<true, false, false>(c, j);
    else tf ? norm_launch<false, true, false>(c, j) : norm_launch<false, false, false>(c, j);
  }
  return p0_launched(c, op);
}

}  // extern "C"
