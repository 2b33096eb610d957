// f8_gemm.cuh -- what the forms of gemmF8 share: the job, and pieces of the two that use tcgen05.
#pragma once
#include "f8.cuh"
#include "tc.cuh"

struct GemmJob {
  F8Mat x, w, u;
  const float *bv;
  uint8_t *y;              // f16 or f32 rows of y_ld
  uint64_t y_ld;
  uint32_t M, N, K, KB, epi;
  uint32_t polls[2];       // after which the copies' waits give up (of a pair's even and odd CTA). The others' limit is a constant: with an
                           // argument few tokens took 0.2 us more
};

// the form for many tokens (f8_tc.cu); y: where the codes of a gated call go
p0_status f8_tc_launch(p0_ctx *c, const GemmJob &j, const F8Mat &y, const char *op);
// the form for few tokens or tiles (f8_mid.cu), and into how many parts it splits the blocks of k
p0_status f8_mid_launch(p0_ctx *c, const GemmJob &j, const F8Mat &y, const char *op);
uint32_t f8_mid_parts(const p0_ctx *c, uint32_t M, uint32_t N, uint32_t KB);

// the gate of a gated epilogue: silu, or the tanh form of gelu as x * sigmoid(2 z), z = sqrt(2 / pi) (x + 0.044715 x^3)
// e^-z = 2^hi 2^lo with hi + lo = -z log2(e) in two f32 (1.44269504 is log2(e) in f32, 1.92596303e-8 what that is too small by), 2^lo = 1 + lo ln 2 (lo is
// below 2^-17): off by 1.25 * 2^-22, the gate by 2.5 * 2^-22, where z is exact. A plain __expf's error grows with z and moved one code in 60000
// to its neighbour; expf and a rounded division took the gated form for many tokens from 78 to 93 us (1031 tokens, N = 8960, K = 2240)
__device__ __forceinline__ float f8_gate(float x, uint32_t epi) {
  const float z = epi == P0_F8EPI_SWIGLU ? x : 1.5957691216057308f * fmaf(0.044715f * x, x * x, x);
  const float zc = fminf(fmaxf(z, -88.0f), 88.0f);   // beyond it the gate is 0 (a quotient by more than 2^126 is, from z = -87.3 on: x * gate is below 2^-119) or 1
  const float hi = -1.44269504f * zc, lo = fmaf(-1.44269504f, zc, -hi) - 1.92596303e-8f * zc;
  float p;
  asm("ex2.approx.f32 %0, %1;" : "=f"(p) : "f"(hi));
  return __fdividef(x, 1.0f + fmaf(p, lo * 0.693147181f, p));
}

// a matrix of codes or of results, in boxes of rows of 128 bytes, in the 128-byte swizzle
inline bool f8_box_map(CUtensorMap *m, CUtensorMapDataType type, uint32_t es, const void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  const auto encode = tensor_map_encoder();
  const cuuint64_t size[2] = {cols, rows}, stride[1] = {ld * es};
  const cuuint32_t box[2] = {128 / es, box_rows}, one[2] = {1, 1};
  return encode && encode(m, type, 2, const_cast<void *>(base), size, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace f8tc {

constexpr uint32_t kDrain = 1u << 16;   // polls for what is in flight when a wait has given up

// one lane of a converged warp. What it issues to the tensor core and the copy engine costs a few cycles each; under a condition on the
// lane's number the compiler cannot tell that there is one lane, and the many tokens' loop took 1050 cycles a block instead of 830
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}" : "=r"(p));
  return p != 0u;
}
// a warp's waits: every lane returns the same
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort, uint32_t *err, uint32_t code, uint32_t polls) {
  return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort, err, code, polls));
}
// for two phases (y may be null): a wait that is over costs its latency, here once for both
__device__ __forceinline__ bool warp_wait_two(uint64_t *x, uint32_t px, uint64_t *y, uint32_t py, volatile uint32_t *abort, uint32_t *err, uint32_t code,
                                              uint32_t polls) {
  bool ok = false;
  for (uint32_t i = 0; i < polls; i++) {
    const bool a = tc::mbar_try(x, px), b = !y || tc::mbar_try(y, py);
    if (a && b) {
      ok = true;
      break;
    }
    if (*abort) break;
  }
  if (!ok && !*abort) {
    *abort = 1u;
    atomicOr(err, code);
  }
  return __all_sync(0xffffffffu, ok);
}

// pairs of f32 in 64 bits: the instructions that take two at once leave issue slots (and instruction fetches) to others
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t twice(float f) { return pair(__float_as_uint(f), __float_as_uint(f)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void fma2(uint64_t &a, uint64_t d, uint64_t f) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(d), "l"(f)); }

}  // namespace f8tc
