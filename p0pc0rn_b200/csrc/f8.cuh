// f8.cuh -- matrices in 8 bits (e4m3 codes with an f32 scale for each block of 128): their views, checks and the quantiser's
// steps, which packF8, normF8 and gemmF8 share.
//
// a = the largest |x| of a block, held within [2^-100, the largest f32] (NaN aside), s = a / 448, code = e4m3(x * (448 / a)),
// each step in f32: the code is off by half a step of x / s (2^-4 of it, or 2^-10 below 2^-6), s by 2^-24 of it. The floor gives a
// block of zeros a scale and keeps 448 / a finite; an infinity becomes 448 * s; NaN stays NaN (code 0x7f).
#pragma once
#include <cuda_fp16.h>

#include "internal.h"
#include "launch.cuh"

constexpr uint32_t kF8Block = 128;

struct F8Mat {
  uint8_t *q;
  float *s;
  uint32_t ld, s_ld;
};

// the calling thread's device for the length of a call: the context's, then again what it was
struct DeviceGuard {
  int was = -1;
  explicit DeviceGuard(int device) {
    int cur = -1;
    if (cudaGetDevice(&cur) == cudaSuccess && cur != device) {
      was = cur;
      cudaSetDevice(device);
    }
  }
  ~DeviceGuard() {
    if (was >= 0) cudaSetDevice(was);
  }
};

// a code matrix [rows][cols] with its scales: by row ([cols / 128][s_ld >= rows]) or by tile ([rows / 128][s_ld >= cols / 128])
p0_status f8_view(p0_ctx *c, const p0_f8 &m, uint64_t rows, uint64_t cols, bool tile, const char *op, const char *name, F8Mat *out);
// rows of f32 or f16: [rows][ld >= cols], off and ld in elements. *wide: rows start on 16-byte boundaries
p0_status f8_rows(p0_ctx *c, p0_buf b, uint64_t off, uint32_t ld, uint64_t rows, uint64_t cols, uint32_t type, const char *op, const char *name,
                  const uint8_t **out, uint32_t *out_ld, bool *wide);
// whether the bytes [a, a + na) and [b, b + nb) meet
inline bool f8_meet(const void *a, uint64_t na, const void *b, uint64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + nb && y < x + na;
}
inline uint64_t f8_code_bytes(const F8Mat &m, uint64_t rows, uint64_t cols) { return (rows - 1) * m.ld + cols; }
inline uint64_t f8_scale_bytes(const F8Mat &m, uint64_t rows, uint64_t cols, bool tile) {
  const uint64_t kb = (cols + kF8Block - 1) / kF8Block, nb = (rows + kF8Block - 1) / kF8Block;
  return tile ? ((nb - 1) * m.s_ld + kb) * 4 : ((kb - 1) * m.s_ld + rows) * 4;
}
__device__ __forceinline__ float f8_hold(float a) { return fminf(fmaxf(a, 0x1p-100f), 3.402823466e38f); }
// two values to two e4m3 codes, round to nearest even, held at +-448; lo in the low byte
__device__ __forceinline__ uint32_t f8_codes2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t f8_codes4(float a, float b, float c, float d) { return f8_codes2(a, b) | (f8_codes2(c, d) << 16); }
