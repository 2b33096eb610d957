// f8.cu -- packF8 (values to e4m3 codes with a scale for each block of 128) and normF8 (residual, RMS norm, codes).
//
// Both are bound by memory. Eight lanes hold a row's block of 128 columns, sixteen to a lane (columns 8 l .. and 64 + 8 l ..): 16-byte
// loads of f16 (two of f32), the block's maximum by three shuffles, 8-byte stores of codes. What a block costs besides (two rounded
// divisions, its place) is shared by sixteen columns a lane (4096 x 12288 f16: 47 us with eight, 29.2 with sixteen, 5.2 TB/s).
#include "f8.cuh"

namespace {

constexpr int kT = 256;

// eight columns as they lie in memory, and as f32
template <bool F16>
struct Raw {
  uint4 w[F16 ? 1 : 2];
};
struct Vals {
  float v[8];
};
// x[k .. k + 7] of a row of K; zeros beyond it. WIDE: rows start on 16-byte boundaries
template <bool F16, bool WIDE>
__device__ __forceinline__ Raw<F16> load8(const void *row, uint32_t k, uint32_t K) {
  Raw<F16> r;
  if (WIDE && k + 8u <= K) {
    const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(row) + (uint64_t)k * (F16 ? 2u : 4u));
    r.w[0] = p[0];
    if (!F16) r.w[F16 ? 0 : 1] = p[1];
  } else {
    uint32_t w[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; i++)
      w[i] = k + i >= K ? 0u : F16 ? (uint32_t)reinterpret_cast<const uint16_t *>(row)[k + i] : reinterpret_cast<const uint32_t *>(row)[k + i];
    if (F16) {
      r.w[0] = make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16), w[6] | (w[7] << 16));
    } else {
      r.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
      r.w[F16 ? 0 : 1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  return r;
}
template <bool F16>
__device__ __forceinline__ Vals vals(const Raw<F16> &r) {
  Vals x;
  const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[F16 ? 0 : 1].x, r.w[F16 ? 0 : 1].y, r.w[F16 ? 0 : 1].z, r.w[F16 ? 0 : 1].w};
  if (F16) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x.v[2 * i] = f.x;
      x.v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x.v[i] = __uint_as_float(w[i]);
  }
  return x;
}
template <bool F16>
__device__ __forceinline__ void store8(void *row, uint32_t k, uint32_t K, const Vals &x) {
#pragma unroll
  for (uint32_t i = 0; i < 8; i++)
    if (k + i < K) {
      if (F16) reinterpret_cast<__half *>(row)[k + i] = __float2half_rn(x.v[i]);
      else reinterpret_cast<float *>(row)[k + i] = x.v[i];
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
// the maximum over eight lanes
__device__ __forceinline__ float eight_max(float a) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// ---------------------------------------------------------------- packF8, blocks of a row
struct PackJob {
  const uint8_t *x;
  uint64_t ld;
  uint32_t M, K, KB, units;   // units = M * KB
  uint32_t magic;             // u / KB = umulhi(u, magic) (+ 1 where the remainder says so) for u < 2^31
  F8Mat y;
};
template <bool F16, bool WIDE>
__global__ void __launch_bounds__(kT) f8_pack_rows_kernel(PackJob j) {
  dep_enter();
  constexpr uint32_t U = F16 ? 4 : 2;   // blocks of eight lanes on their way at once: 128 bytes a lane
  const uint32_t l = threadIdx.x & 7u, es = F16 ? 2u : 4u, eights = gridDim.x * (kT / 8);
  for (uint64_t u0 = blockIdx.x * (kT / 8) + (threadIdx.x >> 3); __any_sync(0xffffffffu, u0 < j.units); u0 += (uint64_t)eights * U) {
    Raw<F16> x[U][2];
    uint32_t m[U], kb[U];
#pragma unroll
    for (uint32_t i = 0; i < U; i++) {
      const uint64_t u = u0 + (uint64_t)i * eights;
      const bool here = u < j.units;
      uint32_t d = j.KB == 1u ? (uint32_t)u : __umulhi((uint32_t)u, j.magic);
      if ((uint32_t)u - d * j.KB >= j.KB) d++;
      m[i] = here ? d : 0u;
      kb[i] = here ? (uint32_t)u - d * j.KB : j.KB;   // beyond the row: zeros, nothing stored
      const uint8_t *row = j.x + (uint64_t)m[i] * j.ld * es;
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) x[i][g] = load8<F16, WIDE>(row, kb[i] * kF8Block + g * 64u + l * 8u, j.K);
    }
#pragma unroll
    for (uint32_t i = 0; i < U; i++) {
      const Vals v[2] = {vals<F16>(x[i][0]), vals<F16>(x[i][1])};
      const float a = f8_hold(eight_max(fmaxf(max8(v[0]), max8(v[1]))));
      if (kb[i] == j.KB) continue;
      const float inv = __fdiv_rn(448.0f, a);
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) store_codes(j.y.q + (uint64_t)m[i] * j.y.ld, kb[i] * kF8Block + g * 64u + l * 8u, j.K, v[g], inv);
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
  Raw<F16> x[8];
#pragma unroll
  for (uint32_t i = 0; i < 8; i++) {
    const uint32_t m = nb * kF8Block + i * 16u + (threadIdx.x >> 4);
    x[i] = load8<F16, WIDE>(j.x + (uint64_t)min(m, j.M - 1u) * j.ld * es, m < j.M ? k : j.K, j.K);
  }
  float a = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < 8; i++) a = fmaxf(a, max8(vals<F16>(x[i])));
  a = eight_max(a);
  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 8));
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
    if (m < j.M) store_codes(j.y.q + (uint64_t)m * j.y.ld, k, j.K, vals<F16>(x[i]), inv);
  }
  if (threadIdx.x == 0) j.y.s[(uint64_t)nb * j.y.s_ld + kb] = __fdiv_rn(a, 448.0f);
}

// ---------------------------------------------------------------- normF8
// tv = the sum of the partial rows in order; with pw: tv * rsqrt(mean tv^2 + eps) * pw; h = (x + tv) * scale, rounded to the
// stream's type; st = rsqrt(mean h^2 + eps); codes of (h * st) * w. blockDim.x threads hold a row, 16 columns each, and take rows in
// turn (blockDim.y of them a CTA). Rows that start on 16 bytes come through shared memory (RING): every warp copies (cp.async) the 512 columns that
// it will read itself, up to two rows ahead, so that no warp waits for another one and no register holds what is on its way. Its lanes copy for one
// another: a row's copies have landed for all of them behind one __syncwarp, and its place is overwritten behind the next. With the
// next row in registers instead, few CTAs fit an SM (190 us for 32760 rows of 2240 in f16), and loads of the weights, which return in
// order behind the next row's, held up each row. Now 95 us, 5.4 TB/s, at 76 % of the issue slots (in long runs 104 at 1.81 GHz); 2051 rows of 1536, f32 +
// f16 with both norms: 13.1; 4096 of 16384, f32 + f32, with room for one row a thread: 161, 5.4 TB/s. Rows that start anywhere, or D % 8 != 0, go value by
// value: 4096 rows of 2241 in f16 55 us, of 2240 17.
struct NormJob {
  const uint8_t *x, *t;
  uint8_t *h;
  const float *pw, *w;
  float *st;
  uint64_t x_ld, t_ld, t_ldm, h_ld;
  uint32_t parts, M, D, nbuf;   // nbuf: rows that a thread has room for
  float eps, scale;
  bool store, wsm;              // wsm: the norms' weights are kept in shared memory
  F8Mat y;
};
// the sum of one float per thread over a row's threads; red: a place for its warps that no sum since the last but one has used
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const uint32_t warps = blockDim.x >> 5;
  if (warps == 1u) return v;
  if ((threadIdx.x & 31u) == 0) red[threadIdx.x >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(1u + threadIdx.y), "r"(blockDim.x) : "memory");
  // the warps' sums, one a lane, by the same tree in every warp
  v = (threadIdx.x & 31u) < warps ? red[threadIdx.x & 31u] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void copy16(uint4 *dst, const uint8_t *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
// x += t, times scale, rounded to f16 where the stream has that type; what is stored of it
template <bool F16>
__device__ __forceinline__ Raw<F16> settle(Vals &x, const Vals &t, float scale) {
  Raw<F16> r;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; i++) x.v[i] = __fadd_rn(x.v[i], t.v[i]);
  if (scale != 1.0f)
#pragma unroll
    for (int i = 0; i < 8; i++) x.v[i] = __fmul_rn(x.v[i], scale);
  if (F16) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __half2 h = __floats2half2_rn(x.v[2 * i], x.v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
      const float2 f = __half22float2(h);
      x.v[2 * i] = f.x;
      x.v[2 * i + 1] = f.y;
    }
    r.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = __float_as_uint(x.v[i]);
    r.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
    r.w[F16 ? 0 : 1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  return r;
}
enum { kScalar = 0, kDirect = 1, kRing = 2 };   // rows that start anywhere; on 16 bytes, loaded as they are needed; ahead
template <bool XF16, bool TF16, int MODE, bool POST>
__global__ void __launch_bounds__(MODE == kDirect ? 512 : 1024) f8_norm_kernel(NormJob j) {
  dep_enter();
  constexpr bool RING = MODE == kRing, WIDE = MODE != kScalar;
  constexpr uint32_t xs = XF16 ? 2 : 4, ts = TF16 ? 2 : 4, XC = xs, TC = ts;   // 16 columns are as many chunks of 16 bytes as a value has bytes
  extern __shared__ uint4 sm[];
  __shared__ float red[3][64];   // of each sum in turn, [row of the CTA][warp]
  const uint32_t l = threadIdx.x & 7u, kb = threadIdx.x >> 3, k0 = kb * kF8Block + l * 8u, step = gridDim.x * blockDim.y;
  const uint32_t T = blockDim.x * blockDim.y;
  const bool in[2] = {k0 < j.D, k0 + 64u < j.D};   // where rows start on 16 bytes, D is a multiple of 8
  uint32_t turn = 0;
  const auto place = [&]() {
    float *p = red[turn] + threadIdx.y * (blockDim.x >> 5);
    turn = turn == 2u ? 0u : turn + 1u;
    return p;
  };
  // shared memory: places of rows [x | t], each warp's 512 columns together, then (wsm) [chunk][thread of a row] of w and pw. Columns beyond D stay zeros
  const uint32_t lane = threadIdx.x & 31u, wx = (threadIdx.x >> 5) * 32u * XC, wt = blockDim.x * XC + (threadIdx.x >> 5) * 32u * TC;   // a warp's chunks of a place
  uint4 *const own = sm + threadIdx.y * blockDim.x * (XC + TC), *const wat = sm + (RING ? j.nbuf * (XC + TC) * T : 0u) + threadIdx.x;
  if (RING) {
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (uint32_t c = threadIdx.y * blockDim.x + threadIdx.x; c < j.nbuf * (XC + TC) * T; c += T) sm[c] = zero;
    if (j.wsm && threadIdx.y == 0)
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) {
        Raw<false> w = load8<false, true>(j.w, k0 + g * 64u, j.D);
        wat[2u * g * blockDim.x] = w.w[0], wat[(2u * g + 1u) * blockDim.x] = w.w[1];
        if (!POST) continue;
        w = load8<false, true>(j.pw, k0 + g * 64u, j.D);
        wat[(4u + 2u * g) * blockDim.x] = w.w[0], wat[(5u + 2u * g) * blockDim.x] = w.w[1];
      }
    __syncthreads();
  }
  Raw<false> wr[2] = {}, pr[2] = {};   // kDirect: the norms' weights
  if (MODE == kDirect)
#pragma unroll
    for (uint32_t g = 0; g < 2; g++) {
      wr[g] = load8<false, true>(j.w, k0 + g * 64u, j.D);
      if (POST) pr[g] = load8<false, true>(j.pw, k0 + g * 64u, j.D);
    }
  // 8 values of f32 weights, of group g
  const auto weights = [&](const float *w, uint32_t chunk, uint32_t g) {
    if (MODE == kDirect) return vals<false>(chunk ? pr[g] : wr[g]);
    Raw<false> r;
    if (RING && j.wsm) r.w[0] = wat[(chunk + 2u * g) * blockDim.x], r.w[1] = wat[(chunk + 2u * g + 1u) * blockDim.x];
    else r = load8<false, WIDE>(w, k0 + g * 64u, j.D);
    return vals<false>(r);
  };
  uint32_t m = blockIdx.x * blockDim.y + threadIdx.y, mf = m;   // the row to work on, to fetch
  uint32_t into = 0, from = 0;                                  // their places
  const uint32_t cx = (threadIdx.x >> 5) * 512u + lane * (16u / xs), ct = (threadIdx.x >> 5) * 512u + lane * (16u / ts);   // columns of a lane's first chunks
  const uint8_t *xf = j.x + ((uint64_t)m * j.x_ld + cx) * xs, *tf = j.t + ((uint64_t)m * j.t_ldm + ct) * ts;
  const auto fetch = [&]() {
    if (mf < j.M) {
      uint4 *to = own + into * (XC + TC) * T;
#pragma unroll
      for (uint32_t c = 0; c < XC; c++)
        if (cx + c * (512u / xs) < j.D) copy16(to + wx + c * 32u + lane, xf + c * 512u);
      if (j.parts)
#pragma unroll
        for (uint32_t c = 0; c < TC; c++)
          if (ct + c * (512u / ts) < j.D) copy16(to + wt + c * 32u + lane, tf + c * 512u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    into = into + 1u == j.nbuf ? 0u : into + 1u;
    mf += step;
    xf += (uint64_t)step * j.x_ld * xs;
    tf += (uint64_t)step * j.t_ldm * ts;
  };
  if (RING)
    for (uint32_t i = 0; i + 1u < j.nbuf; i++) fetch();
  uint8_t *hp = j.h + ((uint64_t)m * j.h_ld + k0) * xs, *yp = j.y.q + (uint64_t)m * j.y.ld;
  for (; m < j.M; m += step, hp += (uint64_t)step * j.h_ld * xs, yp += (uint64_t)step * j.y.ld) {   // the threads of a row go together
    Vals h[2], tv[2];
    if (RING) {
      fetch();
      if (j.nbuf == 3u) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else if (j.nbuf == 2u) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();   // a warp's lanes copied for one another
      const uint4 *at = own + from * (XC + TC) * T;
      from = from + 1u == j.nbuf ? 0u : from + 1u;
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) {
        Raw<XF16> x;
        Raw<TF16> t;
#pragma unroll
        for (uint32_t c = 0; c < XC / 2; c++) x.w[c] = at[wx + (lane >> 3) * (8u * XC) + g * (4u * XC) + l * (XC / 2) + c];
        h[g] = vals<XF16>(x);
        tv[g] = Vals{};
        if (!j.parts) continue;
#pragma unroll
        for (uint32_t c = 0; c < TC / 2; c++) t.w[c] = at[wt + (lane >> 3) * (8u * TC) + g * (4u * TC) + l * (TC / 2) + c];
        tv[g] = vals<TF16>(t);
      }
    } else {
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) {
        h[g] = vals<XF16>(load8<XF16, WIDE>(j.x + (uint64_t)m * j.x_ld * xs, k0 + g * 64u, j.D));
        tv[g] = j.parts ? vals<TF16>(load8<TF16, WIDE>(j.t + (uint64_t)m * j.t_ldm * ts, k0 + g * 64u, j.D)) : Vals{};
      }
    }
    for (uint32_t p = 1; p < j.parts; p++)
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) {
        const Vals t = vals<TF16>(load8<TF16, WIDE>(j.t + ((uint64_t)p * j.t_ld + (uint64_t)m * j.t_ldm) * ts, k0 + g * 64u, j.D));
#pragma unroll
        for (int i = 0; i < 8; i++) tv[g].v[i] += t.v[i];
      }
    if (POST) {
      float s = 0.0f;
#pragma unroll
      for (uint32_t g = 0; g < 2; g++)
#pragma unroll
        for (int i = 0; i < 8; i++) s = fmaf(tv[g].v[i], tv[g].v[i], s);
      const float rs = rsqrtf(row_sum(s, place()) / (float)j.D + j.eps);
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) {
        const Vals w = weights(j.pw, 4, g);
#pragma unroll
        for (int i = 0; i < 8; i++) tv[g].v[i] = __fmul_rn(__fmul_rn(tv[g].v[i], rs), w.v[i]);
      }
    }
    float s = 0.0f;
#pragma unroll
    for (uint32_t g = 0; g < 2; g++) {
      const Raw<XF16> r = settle<XF16>(h[g], tv[g], j.scale);
#pragma unroll
      for (int i = 0; i < 8; i++) s = fmaf(h[g].v[i], h[g].v[i], s);
      if (!j.store) continue;
      if (WIDE) {
        if (!in[g]) continue;
        uint4 *to = reinterpret_cast<uint4 *>(hp + g * 64u * xs);
        to[0] = r.w[0];
        if (!XF16) to[1] = r.w[XF16 ? 0 : 1];
      } else {
        store8<XF16>(j.h + (uint64_t)m * j.h_ld * xs, k0 + g * 64u, j.D, h[g]);
      }
    }
    const float st = rsqrtf(row_sum(s, place()) / (float)j.D + j.eps);
    if (j.st && threadIdx.x == 0) j.st[m] = st;
#pragma unroll
    for (uint32_t g = 0; g < 2; g++) {
      const Vals w = weights(j.w, 0, g);
#pragma unroll
      for (int i = 0; i < 8; i++) h[g].v[i] = __fmul_rn(__fmul_rn(h[g].v[i], st), w.v[i]);
    }
    const float a = f8_hold(eight_max(fmaxf(max8(h[0]), max8(h[1])))), inv = __fdiv_rn(448.0f, a);
    if (in[0]) {
#pragma unroll
      for (uint32_t g = 0; g < 2; g++) store_codes(yp, k0 + g * 64u, j.D, h[g], inv);
    }
    if (l == 0 && in[0]) j.y.s[(uint64_t)kb * j.y.s_ld + m] = __fdiv_rn(a, 448.0f);
    __syncwarp();
  }
  if (RING) asm volatile("cp.async.wait_all;" ::: "memory");
}

template <bool XF16, bool TF16>
p0_status norm_launch(p0_ctx *c, NormJob &j, bool wide, const char *op) {
  // several rows a CTA where they are short; as many CTAs as an SM holds, each with its rows in turn
  const uint32_t T = (j.D + 511u) / 512u * 32u, R = T <= 160u ? 320u / T : 1u, ctas = (j.M + R - 1u) / R;
  const uint32_t row = T * R * 16u * ((XF16 ? 2u : 4u) + (TF16 ? 2u : 4u)), ws = T * 64u * (j.pw ? 2u : 1u);
  uint32_t per = 1024u / (T * R), smem = 0;
  const auto go = [&](auto kern, dim3 grid, dim3 block) {
    const cudaError_t e = smem ? p0_smem_limit((const void *)kern, 768) : cudaSuccess;   // 768: red
    if (e != cudaSuccess) return p0_cuda(c, e, op);
    launch_dep(kern, grid, block, smem, c->stream, j);
    return p0_launched(c, op);
  };
  if (!wide) return j.pw ? go(f8_norm_kernel<XF16, TF16, kScalar, true>, dim3(ctas), dim3(T, R)) : go(f8_norm_kernel<XF16, TF16, kScalar, false>, dim3(ctas), dim3(T, R));
  // a row a CTA and nothing to fetch ahead: 148 rows of 2560, 4.0 us against 6.0; beyond, starting CTAs costs more (300 of 4096: 7.8 against 5.4)
  if (j.M <= (uint32_t)c->sm_count && T <= 512u)
    return j.pw ? go(f8_norm_kernel<XF16, TF16, kDirect, true>, dim3(j.M), dim3(T)) : go(f8_norm_kernel<XF16, TF16, kDirect, false>, dim3(j.M), dim3(T));
  // room for three rows where it does not cost CTAs, two else; one for the longest in f32
  const uint32_t all = 220u * 1024u;
  j.wsm = row + ws <= all;
  const uint32_t w = j.wsm ? ws : 0u;
  j.nbuf = (3u * row + w) * per <= all ? 3u : 2u * row + w <= all ? 2u : 1u;
  smem = j.nbuf * row + w;
  if (per > all / smem) per = all / smem;
  const uint32_t fit = (uint32_t)c->sm_count * per;
  return j.pw ? go(f8_norm_kernel<XF16, TF16, kRing, true>, dim3(ctas < fit ? ctas : fit), dim3(T, R))
              : go(f8_norm_kernel<XF16, TF16, kRing, false>, dim3(ctas < fit ? ctas : fit), dim3(T, R));
}

void pack_rows_launch(p0_ctx *c, PackJob j, bool f16, bool wide) {
  j.magic = (uint32_t)((1ull << 32) / j.KB);   // one too small at most
  const uint64_t want = ((uint64_t)j.units + kT / 8 - 1) / (kT / 8), most = (uint64_t)c->sm_count * 8u;
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
  const bool in_place = h == j.x && (h_ld == ld || M == 1);   // the stride of one row is not looked at
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
  wide = wide && w1 && w2 && (uintptr_t)j.w % 16 == 0 && (uintptr_t)j.pw % 16 == 0 && D % 8 == 0;
  DeviceGuard guard(c->device);
  const bool xf = a->type == P0_F16, tf = a->t_type == P0_F16;
  if (xf) return tf ? norm_launch<true, true>(c, j, wide, op) : norm_launch<true, false>(c, j, wide, op);
  return tf ? norm_launch<false, true>(c, j, wide, op) : norm_launch<false, false>(c, j, wide, op);
}

}  // extern "C"
