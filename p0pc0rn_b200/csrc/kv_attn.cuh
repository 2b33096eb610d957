// kv_attn.cuh -- what the forms of kv4Attn share: the call's arguments, what a row block sees, how the work is cut into
// equal runs from the lengths on the device, and how parts of a unit are joined.
#pragma once
#include "kv.cuh"
#include "launch.cuh"
#include "tc.cuh"

struct AttnJob {
  KvView v;
  KvRows q, out;
  uint32_t hpg, window, sinks, units;   // units: of a row block (KV heads; times the parts that an output row is cut into)
  float scale;
  bool qbox;          // the prompt form: q has a tensor map
  uint32_t *err;
  float *part;        // [grid][2][rows of a block][D + 2]
  uint4 *desc;        // [grid]: (1 + last run, b, first row, KV head) of the unit that this run begins and others end
  uint8_t *wide;      // the prompt form: pages as f16 tiles
};

// what a unit's rows see: pages [0, sink_pages) and [from, last], or nothing (n = 0)
struct Span {
  uint32_t sink_pages, from, n;
  uint32_t first_pos, end;   // first key inside the first row's window; one past the last row's position
};
// positions of rows t0 and t1 (0 <= t0 <= t1 < T): len - T + t, which may be negative; all below 2^31, as the window
__device__ __forceinline__ Span span_of(uint32_t len, uint32_t T, uint32_t t0, uint32_t t1, uint32_t window, uint32_t sinks) {
  Span s;
  const int32_t p1 = (int32_t)(len - T + t1), p0 = (int32_t)(len - T + t0), w0 = p0 - (int32_t)window + 1;
  s.end = p1 < 0 ? 0u : (uint32_t)p1 + 1u;
  s.first_pos = window && p0 >= 0 && w0 > 0 ? (uint32_t)w0 : 0u;
  s.from = s.first_pos / kPage;
  s.sink_pages = min((sinks + kPage - 1) / kPage, s.from);
  s.n = s.end ? s.sink_pages + (s.end - 1) / kPage + 1 - s.from : 0u;
  return s;
}
__device__ __forceinline__ uint32_t page_at(const Span &s, uint32_t i) { return i < s.sink_pages ? i : s.from + (i - s.sink_pages); }

// in place, inclusive sums of v[0 .. n) by one warp
__device__ __forceinline__ void warp_sums(uint32_t *v, uint32_t n) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t carry = 0;
  for (uint32_t b0 = 0; b0 < n; b0 += 32) {
    uint32_t x = b0 + lane < n ? v[b0 + lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= (uint32_t)o) x += u;
    }
    if (b0 + lane < n) v[b0 + lane] = x + carry;
    carry += __shfl_sync(0xffffffffu, x, 31);
  }
}

// Sequences that claim more than the call's n tokens between them (a cu that goes up and down) claim some twice. The host
// counts work for n tokens, so such a call has none. A whole warp
__device__ __forceinline__ bool claims_fit(const KvView &view) {
  if (!view.cu) return true;
  uint64_t claimed = 0;
#pragma unroll 1
  for (uint32_t b = threadIdx.x & 31u; b < view.rows; b += 32) {
    uint32_t lo;
    claimed += kv_tokens(view, b, lo);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) claimed += __shfl_xor_sync(0xffffffffu, claimed, o);
  return claimed <= view.n;
}

// Work. The query rows that share a KV head (new tokens x query heads of its group) form blocks of RB; a unit is one row
// block of one sequence and KV head (or part of its output), its items are the runs of PP pages that any of its rows sees (one item where there are
// none: zeros are to be written), after E items that stand for what beginning and ending a unit costs. pre[b] = items
// before sequence b; [rows + 1] shared words. Every thread of the CTA.
template <uint32_t RB, uint32_t PP, uint32_t E>
__device__ __forceinline__ uint32_t unit_items(const AttnJob &j, uint32_t len, uint32_t T, uint32_t r0, Span &s) {
  const uint32_t rows = T * j.hpg;
  s = span_of(len, T, r0 / j.hpg, min(rows - 1, r0 + RB - 1) / j.hpg, j.window, j.sinks);
  return max(1u, (s.n + PP - 1) / PP) + E;
}
template <uint32_t RB, uint32_t PP, uint32_t E>
__device__ __forceinline__ void plan_items(const AttnJob &j, uint32_t *pre) {
  const uint32_t R = j.v.rows;
  if (!j.v.cu && j.v.T * j.hpg <= RB) {   // one block a sequence: a thread each
    for (uint32_t b = threadIdx.x; b < R; b += blockDim.x) {
      uint32_t lo;
      const uint32_t T = kv_tokens(j.v, b, lo);
      Span s;
      pre[b + 1] = T ? unit_items<RB, PP, E>(j, kv_len(j.v, b), T, 0, s) * j.units : 0u;
    }
  } else {                                 // a warp each
    for (uint32_t b = threadIdx.x >> 5; b < R; b += blockDim.x >> 5) {
      uint32_t lo, items = 0;
      const uint32_t T = kv_tokens(j.v, b, lo), len = kv_len(j.v, b);
      for (uint32_t r = (threadIdx.x & 31u) * RB; r < T * j.hpg; r += 32u * RB) {
        Span s;
        items += unit_items<RB, PP, E>(j, len, T, r, s);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) items += __shfl_xor_sync(0xffffffffu, items, o);
      if ((threadIdx.x & 31u) == 0) pre[b + 1] = items * j.units;
    }
  }
  if (threadIdx.x == 0) pre[0] = 0u;
  __syncthreads();
  if (threadIdx.x < 32) {
    if (claims_fit(j.v)) warp_sums(pre + 1, R);
    else
      for (uint32_t b = threadIdx.x; b < R; b += 32) pre[b + 1] = 0u;
  }
  __syncthreads();
}
// the last b with pre[b] <= at (a sequence with items of its own, or one before it)
__device__ __forceinline__ uint32_t find_sequence(const uint32_t *pre, uint32_t R, uint32_t at) {
  uint32_t a = 0, e = R;
  while (e - a > 1) {
    const uint32_t m = (a + e) >> 1;
    if (pre[m] <= at) a = m; else e = m;
  }
  return a;
}

struct Unit {
  uint32_t first, T, len, rows;      // of its sequence: first token of the call, new tokens, length, query rows
  uint32_t r0, head, begin, n;       // first row, KV head (times parts, plus part), first item and items
  Span s;
};
// the unit of item `at` of sequence b: row blocks in order, each with its KV heads in order. A whole warp.
template <uint32_t RB, uint32_t PP, uint32_t E>
__device__ __forceinline__ Unit find_unit(const AttnJob &j, const uint32_t *pre, uint32_t b, uint32_t at) {
  Unit u;
  u.T = kv_tokens(j.v, b, u.first);
  u.len = kv_len(j.v, b);
  u.rows = u.T * j.hpg;
  const uint32_t lane = threadIdx.x & 31u, units = j.units;
  uint32_t base = pre[b];
  for (uint32_t r = 0; r < u.rows; r += 32u * RB) {
    const uint32_t r0 = r + lane * RB;
    Span s;
    const uint32_t n = r0 < u.rows ? unit_items<RB, PP, E>(j, u.len, u.T, r0, s) : 0u;
    uint32_t sum = n * units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= (uint32_t)o) sum += v;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, at < base + sum);
    if (hit) {
      const int k = __ffs(hit) - 1;
      u.r0 = r + k * RB;
      u.n = __shfl_sync(0xffffffffu, n, k);
      base += __shfl_sync(0xffffffffu, sum, k) - u.n * units;
      u.head = (at - base) / u.n;
      u.begin = base + u.head * u.n;
      unit_items<RB, PP, E>(j, u.len, u.T, u.r0, u.s);
      return u;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  u.r0 = u.head = u.begin = 0;   // not reached: `at` lies in sequence b
  u.n = 1;
  u.s = span_of(0, 1, 0, 0, 0, 0);
  return u;
}
// runs end where total * (c + 1) / G does: the run of item i
__device__ __forceinline__ uint32_t run_of(uint32_t i, uint32_t total, uint32_t G) { return (uint32_t)((((uint64_t)i + 1u) * G - 1u) / total); }

// the prompt form (kv_prompt.cu): f16, many new tokens; P0_OK with *taken = false, and j as it was, where it does not serve the call
p0_status kv4_attn_prompt(p0_ctx *c, AttnJob &j, bool *taken);
