// kv.cuh -- the paged 4-bit cache as the kernels see it: a layer's view, where a token's row lies, its new tokens, and
// the host checks that every operator over it shares. The layout is described at p0_kv in include/p0mm.h.
#pragma once
#include <cuda_fp16.h>

#include "internal.h"

constexpr uint32_t kPage = P0_KV_PAGE;      // tokens per page
constexpr uint32_t kKvMaxRows = 1024;       // sequences per call: the kernels keep a word per sequence in shared memory

// one layer of the cache; head h's K records start at pool + page * stride + h * 2 * part, its V records `part` later
struct KvView {
  const uint8_t *pool;
  uint64_t stride;
  const uint32_t *table, *len, *cu;   // cu: cumulative new tokens [rows + 1], or null: T per sequence
  uint32_t ld, pages, rows, nkv, D, n, T;
};

// the tokens [lo, lo + count) of the call that belong to sequence b. A cu that decreases or passes n gives no tokens
// out of range (it may give a token to several sequences: claims_fit).
__device__ __forceinline__ uint32_t kv_tokens(const KvView &v, uint32_t b, uint32_t &lo) {
  uint32_t hi;
  if (v.cu) {
    lo = min(v.cu[b], v.n);
    hi = min(v.cu[b + 1], v.n);
  } else {
    lo = min(b * v.T, v.n);
    hi = min(lo + v.T, v.n);
  }
  return hi > lo ? hi - lo : 0u;
}
// the sequence's length, held at what its table row can map
__device__ __forceinline__ uint32_t kv_len(const KvView &v, uint32_t b) { return min(v.len[b], v.ld * kPage); }

// the position of the call's token i in its sequence b, or false where it has none (a token of no sequence, or a
// sequence shorter than its new tokens)
__device__ __forceinline__ bool kv_place(const KvView &v, uint32_t i, uint32_t &b, uint32_t &pos) {
  if (v.cu) {
    uint32_t lo = 0, hi = v.rows;   // the last b with cu[b] <= i
    while (hi - lo > 1) {
      const uint32_t m = (lo + hi) >> 1;
      if (v.cu[m] <= i) lo = m; else hi = m;
    }
    b = lo;
  } else {
    b = i / v.T;
  }
  if (b >= v.rows) return false;
  uint32_t first;
  const uint32_t count = kv_tokens(v, b, first), n = kv_len(v, b);
  if (i < first || i - first >= count) return false;
  const uint32_t back = count - (i - first);   // 1 for the last new token
  if (back > n) return false;
  pos = n - back;
  return true;
}

// kv_deq2: the codes in the low nibbles of a word's halves -> f16(q * s + mn) of both, each rounded once
__device__ __forceinline__ uint32_t kv_fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// (w & mask) | 0x64006400: 1024 + the masked code of both halves (one lop3; written as two operators it takes two)
__device__ __forceinline__ uint32_t kv_code2(uint32_t w, uint32_t mask) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(0x64006400u));
  return d;
}
__device__ __forceinline__ uint32_t kv_sub1024(uint32_t x) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x64006400u));   // (1024 + q) - 1024, exact
  return d;
}
__device__ __forceinline__ uint32_t kv_deq2(uint32_t w, uint32_t s2, uint32_t mn2) {
  return kv_fma2(kv_sub1024(kv_code2(w, 0x000F000Fu)), s2, mn2);
}
// the four pairs of a word, nibbles 0..3 of its halves. A nibble one place up makes 1024 + 16 q, which one fma turns into q
// as exactly as the subtraction does: one shift a word instead of three
__device__ __forceinline__ void kv_deq8(uint32_t w, uint32_t s2, uint32_t mn2, uint32_t *v) {
  const uint32_t w8 = w >> 8;
  v[0] = kv_deq2(w, s2, mn2);
  v[1] = kv_fma2(kv_fma2(kv_code2(w, 0x00F000F0u), 0x2C002C00u, 0xD400D400u), s2, mn2);   // x / 16 - 64
  v[2] = kv_deq2(w8, s2, mn2);
  v[3] = kv_fma2(kv_fma2(kv_code2(w8, 0x00F000F0u), 0x2C002C00u, 0xD400D400u), s2, mn2);
}

// the host side: resolves and checks a view (layer: its D and nkv too), the new tokens' layout, and rows of values
p0_status kv_view(p0_ctx *c, const p0_kv &kv, bool layer, const char *op, KvView *v);
p0_status kv_new_tokens(p0_ctx *c, uint32_t n, uint32_t T, p0_buf cu, uint32_t cu_off, const char *op, KvView *v);
struct KvRows {
  uint8_t *base;
  uint64_t ld, ldh;    // elements from token to token and from head to head
  bool wide;           // every 8-element run that starts at a multiple of 8 may be read 16 bytes at a time
};
p0_status kv_rows(p0_ctx *c, const p0_rows &r, uint32_t n, uint32_t heads, uint32_t D, uint32_t type, const char *op, const char *name, KvRows *out);
