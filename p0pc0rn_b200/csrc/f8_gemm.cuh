// f8_gemm.cuh -- what the forms of gemmF8 share.
#pragma once
#include "f8.cuh"

struct GemmJob {
  F8Mat x, w, u;
  const float *bv;
  uint8_t *y;              // f16 or f32 rows of y_ld
  uint64_t y_ld;
  uint32_t M, N, K, KB, epi;
};

// the form for many tokens (f8_tc.cu); y: where the codes of a gated call go
p0_status f8_tc_launch(p0_ctx *c, const GemmJob &j, const F8Mat &y, const char *op);
// where tokens or tiles are few (f8_mid.cu)
p0_status f8_mid_launch(p0_ctx *c, const GemmJob &j, const F8Mat &y, const char *op);
