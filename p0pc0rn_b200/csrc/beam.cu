// beam.cu -- beamSelect: the k best continuations of every group of k beams over the vocabulary (no counterpart in the
// reference, which decodes one hypothesis by argmax / argmaxM, engine/llm/lops.js:416-436).
//   lse_b = log sum_v exp(x[b, v]),  c[b, v] = score[b] + (x[b, v] - lse_b),  the k largest c, ties to the lowest b * V + v
// One pass over the logits (they are the only traffic that counts: 4 bytes per candidate). A CTA takes a part of a row, 4096
// logits (a chunk) at a time in registers, and keeps per thread the running (max, sum exp), per thread and chunk the maximum
// in shared memory: six instructions a logit. The (k + 1)-th largest of the threads' maxima is a bound that k + 1 logits
// reach; the few (thread, chunk) pairs whose maximum reaches it are read again (out of L2), and what reaches it is ranked.
// Where equal logits make the list too long, the CTA goes over its part again with keys that order equal values too.
// A second kernel merges: lse per row, then the group's k best among the kept ones. Within a row c does not decrease as x
// grows, so every candidate above the k-th best c has been kept; candidates that round to the very same c as the k-th best
// may not have been, and where that can be (a part's last kept one ties with it) the merge looks the row's logits up again
// in index order.
// 128 rows of 262144 logits, 8 beams: 32.3 us, 4.2 TB/s; the scan (29.8 us, 54 % of DRAM, 41 % of the issue slots) has no loads on their
// way while a part is ranked, the merge none of the logits. 4 rows of 4099: 8.8 us, two launches.
#include "internal.h"
#include "launch.cuh"

namespace {

constexpr int kT = 256, kPer = 16;               // threads, logits per thread
constexpr uint32_t kChunk = kT * kPer;
constexpr uint32_t kMaxBeams = 16;
constexpr uint32_t kMaxKept = kMaxBeams + 1, kMaxList = 1024;   // >= kMaxKept * (kPer + 1): what one chunk can add to the kept ones
constexpr uint32_t kMaxChunks = 16, kMaxPairs = 256;   // chunks of a part; its (thread, chunk) pairs to be read again

// an f32 as a whole number of the same order; NaN and -inf, which never win, come below all others as 0
__device__ __forceinline__ uint32_t ordered(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);   // -0 as +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// larger value first, then the lower index; 0 for what never wins
__device__ __forceinline__ uint64_t key_of(float x, uint32_t idx) {
  const uint32_t o = ordered(x);
  return o ? (uint64_t)o << 32 | (0xffffffffu - idx) : 0ull;
}
__device__ __forceinline__ uint32_t key_idx(uint64_t k) { return 0xffffffffu - (uint32_t)k; }
__device__ __forceinline__ float key_val(uint64_t k) { return from_ordered((uint32_t)(k >> 32)); }

// the lanes' keys, largest in lane 0
__device__ __forceinline__ uint64_t warp_sort(uint64_t k) {
  const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
  for (uint32_t size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (uint32_t step = size >> 1; step > 0; step >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, k, step);
      const bool first = (lane & step) == 0, down = (lane & size) == 0;   // the pair's lower lane; a run that falls
      k = (k > o) == (first == down) ? k : o;
    }
  return k;
}

// The n-th largest of the threads' keys (n <= 32; 1 where fewer than n threads have one): a lower bound of the n-th
// largest of everything that the threads looked at. tops: [threads / 32 * n] shared keys.
__device__ __forceinline__ uint64_t nth_of_threads(uint64_t mine, uint32_t n, uint64_t *tops, uint64_t *found) {
  const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5, m = (blockDim.x >> 5) * n;
  const uint64_t s = warp_sort(mine);
  if (lane < n) tops[w * n + lane] = s;
  if (threadIdx.x == 0) *found = 1ull;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < m; i += blockDim.x) {
    const uint64_t k = tops[i];
    uint32_t above = 0;
    for (uint32_t j = 0; j < m; j++) above += tops[j] > k;
    if (k && above == n - 1) *found = k;
  }
  __syncthreads();
  return *found;
}

struct BeamJob {
  const float *logits;
  uint64_t ld;
  const float *score;
  const uint32_t *fin;
  uint32_t groups, beams, V, eos, nchunk, nsplit;   // chunks and parts of a row
  uint64_t *keys;      // [rows][nsplit][beams + 1]
  float2 *stat;        // [rows][nsplit] (max, sum exp(x - max))
  uint32_t *parent, *token, *fin_out;
  float *score_out;
};

// a thread's logits of a chunk; -inf beyond V
template <bool WIDE>
__device__ __forceinline__ void load_chunk(const float *x, uint32_t base, uint32_t V, float (&v)[kPer]) {
  if (WIDE && base + kChunk <= V) {   // a whole chunk: no looks at V
    const float4 *p = reinterpret_cast<const float4 *>(x + base) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < kPer / 4; i++) {
      const float4 f = __ldcs(p + i * kT);
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
  } else if (WIDE) {
#pragma unroll
    for (int i = 0; i < kPer / 4; i++) {
      const uint32_t at = base + (i * kT + threadIdx.x) * 4u;
      const float4 f = at < V ? __ldcs(reinterpret_cast<const float4 *>(x + at)) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint32_t at = base + i * kT + threadIdx.x;
      v[i] = at < V ? __ldcs(x + at) : -INFINITY;
    }
  }
}
template <bool WIDE>
__device__ __forceinline__ uint32_t index_of(uint32_t base, int i) {   // grows with i: the first of equal values has the lowest
  return WIDE ? base + ((i / 4) * kT + threadIdx.x) * 4u + (i & 3) : base + i * kT + threadIdx.x;
}
template <bool WIDE>
__device__ __forceinline__ uint64_t best_key(const float (&v)[kPer], uint32_t base) {
  float mx = -INFINITY;
  uint32_t at = 0;
#pragma unroll
  for (int i = 0; i < kPer; i++)
    if (v[i] > mx) { mx = v[i]; at = index_of<WIDE>(base, i); }
  return key_of(mx, at);
}
// exp(x) for x <= 0, where the error of x * log2(e), 2^-24 of it, weighs less the smaller the result is: three instructions
__device__ __forceinline__ float exp_below(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504088896340736f));
  return y;
}
// the n largest keys of list[0 .. c) (zeros are none), in order, to kept; zeros after them
__device__ __forceinline__ void keep_best(const uint64_t *list, uint32_t c, uint32_t n, uint64_t *kept) {
  if (threadIdx.x < n) kept[threadIdx.x] = 0ull;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < c; i += kT) {
    const uint64_t k = list[i];
    uint32_t above = 0;
    for (uint32_t q = 0; q < c; q++) above += list[q] > k;
    if (k && above < n) kept[above] = k;
  }
  __syncthreads();
}

template <bool WIDE>
__global__ void __launch_bounds__(kT, 4) beam_scan_kernel(BeamJob j) {
  dep_enter();
  __shared__ uint64_t tops[kT / 32 * kMaxKept], list[kMaxList], kept[kMaxKept], found;
  __shared__ float red[2][kT / 32], top[kMaxChunks][kT];
  __shared__ uint32_t count, n_pairs, pairs[kMaxPairs];
  const uint32_t row = blockIdx.y, part = blockIdx.x, n = j.beams + 1, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  if (j.fin && j.fin[row]) return;   // a finished beam has one candidate, whatever its logits
  const float *x = j.logits + row * j.ld;
  const uint32_t c0 = (uint32_t)((uint64_t)j.nchunk * part / j.nsplit), c1 = (uint32_t)((uint64_t)j.nchunk * (part + 1) / j.nsplit);
  if (threadIdx.x == 0) count = n_pairs = 0u;
  // m: the thread's maximum so far, s: its sum of exp(x - m). A NaN or +inf makes s, its row's lse and every c NaN
  float m = -INFINITY, s = 0.0f, v[kPer], next[kPer];
  load_chunk<WIDE>(x, c0 * kChunk, j.V, next);
#pragma unroll 2   // the two buffers change places without moves
  for (uint32_t ch = c0; ch < c1; ch++) {
#pragma unroll
    for (int i = 0; i < kPer; i++) v[i] = next[i];
    if (ch + 1 < c1) load_chunk<WIDE>(x, (ch + 1) * kChunk, j.V, next);
    float y[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 4; i < kPer; i++) y[i & 3] = fmaxf(y[i & 3], v[i]);
    float mx = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));   // of the numbers (fmaxf passes NaN by)
    mx = fmaxf(mx, -INFINITY);
    top[ch - c0][threadIdx.x] = mx;
    if (mx > m) {
      s *= expf(m - mx);   // 0 while the thread has seen nothing (exp(-inf))
      m = mx;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    float t0 = 0.0f, t1 = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
      t0 += exp_below(v[i] - ref);
      t1 += exp_below(v[i + 1] - ref);
    }
    s += t0 + t1;
  }
  // the bound; 0 where fewer than n threads have a candidate: all are kept
  uint64_t thr = nth_of_threads(key_of(m, threadIdx.x), n, tops, &found);
  const uint32_t least = max((uint32_t)(thr >> 32), 1u);
  if (ordered(m) >= least) {
    for (uint32_t ch = 0; ch < c1 - c0; ch++) {
      if (ordered(top[ch][threadIdx.x]) < least) continue;
      const uint32_t q = atomicAdd(&n_pairs, 1u);
      if (q < kMaxPairs) pairs[q] = ch << 16 | threadIdx.x;
    }
  }
  __syncthreads();
  for (uint32_t p = threadIdx.x / kPer; p < min(n_pairs, kMaxPairs); p += kT / kPer) {   // a lane per logit of the pair
    const uint32_t i = threadIdx.x % kPer, th = pairs[p] & 0xffffu, base = (c0 + (pairs[p] >> 16)) * kChunk;
    const uint32_t at = WIDE ? base + ((i / 4) * kT + th) * 4u + (i & 3u) : base + i * kT + th;
    const float f = at < j.V ? x[at] : -INFINITY;
    if (ordered(f) >= least) {
      const uint32_t q = atomicAdd(&count, 1u);
      if (q < kMaxList) list[q] = key_of(f, at);
    }
  }
  __syncthreads();
  uint32_t c = n_pairs > kMaxPairs ? kMaxList + 1u : count;
  __syncthreads();
  if (c > kMaxList) {   // again, slowly: the kept ones join every chunk's candidates, and the bound rises with them
    if (threadIdx.x < n) kept[threadIdx.x] = 0ull;
    for (uint32_t ch = c0; ch < c1; ch++) {
      load_chunk<WIDE>(x, ch * kChunk, j.V, v);
      if (threadIdx.x == 0) count = n;
      if (threadIdx.x < n) list[threadIdx.x] = kept[threadIdx.x];   // by the thread that cleared or ranked it, or after its barrier
      const uint64_t mine = best_key<WIDE>(v, ch * kChunk);
      thr = nth_of_threads(mine, n, tops, &found);
      if (mine && mine >= thr) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
          const uint64_t k = key_of(v[i], index_of<WIDE>(ch * kChunk, i));
          if (k && k >= thr) list[atomicAdd(&count, 1u)] = k;   // at most n threads hold such keys, kPer each
        }
      }
      __syncthreads();
      c = count;
      __syncthreads();
      keep_best(list, c, n, kept);
    }
  } else {
    keep_best(list, c, n, kept);
  }
  uint64_t *out = j.keys + ((uint64_t)row * j.nsplit + part) * n;
  // the part's (m, s)
  float w = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
  if (lane == 0) red[0][warp] = w;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kT / 32; i++) w = fmaxf(w, red[0][i]);
  s *= m == -INFINITY ? 1.0f : expf(m - w);   // a thread of -inf alone has s = 0, or NaN
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[1][warp] = s;
  __syncthreads();
  if (threadIdx.x < n) out[threadIdx.x] = kept[threadIdx.x];
  if (threadIdx.x == 0) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < kT / 32; i++) s += red[1][i];
    j.stat[(uint64_t)row * j.nsplit + part] = make_float2(w, s);
  }
}

// one CTA per group
constexpr int kMT = 512, kHeld = 4;          // keys that a thread holds between the passes
constexpr uint32_t kMaxSplit = 256;
constexpr uint32_t kMaxMerge = kMaxBeams * ((kMaxBeams * kMaxSplit * kMaxKept + kMT - 1) / kMT);   // keys that can pass the bound
__global__ void __launch_bounds__(kMT) beam_merge_kernel(BeamJob j) {
  dep_enter();
  __shared__ float lse[kMaxBeams], score[kMaxBeams];
  __shared__ uint32_t fin[kMaxBeams];
  __shared__ uint64_t tops[kMT / 32 * kMaxBeams], found, best[kMaxBeams], list[kMaxMerge];
  __shared__ uint32_t n_list, tied, warp_n[kMT / 32];
  const uint32_t g = blockIdx.x, k = j.beams, n = k + 1, r0 = g * k, nc = j.nsplit, V = j.V, M = k * nc * n;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint64_t *keys = j.keys + (uint64_t)r0 * nc * n;
  uint64_t held[kHeld];   // on their way while lse is computed
#pragma unroll
  for (int i = 0; i < kHeld; i++) {
    const uint32_t at = threadIdx.x + i * kMT;
    held[i] = at < M ? keys[at] : 0ull;
  }
  for (uint32_t b = warp; b < k; b += kMT / 32) {
    const bool done = j.fin && j.fin[r0 + b];
    const float sc = j.score[r0 + b];
    const float2 *st = j.stat + (uint64_t)(r0 + b) * nc;
    float m = -INFINITY, s = 0.0f;
    if (!done) {
      for (uint32_t i = lane; i < nc; i += 32) m = fmaxf(m, st[i].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float ref = m == -INFINITY ? 0.0f : m;
      for (uint32_t i = lane; i < nc; i += 32) s += st[i].y * expf(st[i].x - ref);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) {
      lse[b] = m + logf(s);
      score[b] = sc;
      fin[b] = done;
    }
  }
  if (threadIdx.x < kMaxBeams) best[threadIdx.x] = 0ull;
  if (threadIdx.x == 0) { n_list = 0u; tied = 0u; }
  __syncthreads();
  // the kept logit at `at` ([beam][part][rank]) as a key of c, then of the lowest b * V + v. A finished beam's one candidate
  // stands in its first place (the scan has written nothing for it)
  const auto c_of = [&](uint32_t b, float x) { return __fadd_rn(score[b], __fsub_rn(x, lse[b])); };
  const auto c_key = [&](uint32_t at, uint64_t kx) {
    const uint32_t b = at / (nc * n);
    if (fin[b]) return at % (nc * n) == 0 ? key_of(score[b], b * V + j.eos) : 0ull;
    return kx ? key_of(c_of(b, key_val(kx)), b * V + key_idx(kx)) : 0ull;
  };
  uint64_t mine = 0;
#pragma unroll
  for (int i = 0; i < kHeld; i++) {
    const uint32_t at = threadIdx.x + i * kMT;
    held[i] = at < M ? c_key(at, held[i]) : 0ull;
    if (held[i] > mine) mine = held[i];
  }
  for (uint32_t at = threadIdx.x + kHeld * kMT; at < M; at += kMT) {
    const uint64_t c = c_key(at, keys[at]);
    if (c > mine) mine = c;
  }
  const uint64_t thr = nth_of_threads(mine, k, tops, &found);
  if (mine >= thr) {   // at most k threads, M / kMT keys each
#pragma unroll
    for (int i = 0; i < kHeld; i++)
      if (held[i] >= thr) list[atomicAdd(&n_list, 1u)] = held[i];
    for (uint32_t at = threadIdx.x + kHeld * kMT; at < M; at += kMT) {
      const uint64_t c = c_key(at, keys[at]);
      if (c >= thr) list[atomicAdd(&n_list, 1u)] = c;
    }
  }
  __syncthreads();
  const uint32_t nl = n_list;
  for (uint32_t i = threadIdx.x; i < nl; i += kMT) {
    uint32_t above = 0;
    for (uint32_t q = 0; q < nl; q++) above += list[q] > list[i];
    if (above < k) best[above] = list[i];
  }
  __syncthreads();
  const uint32_t last = (uint32_t)(best[k - 1] >> 32);   // the k-th best c, 0 where there are fewer candidates
  if (last) {   // where a part's last kept logit has that c, more of them may follow in the part
#pragma unroll
    for (int i = 0; i < kHeld; i++)
      if ((threadIdx.x + i * kMT) % n == n - 1 && (uint32_t)(held[i] >> 32) == last) tied = 1u;
    for (uint32_t at = threadIdx.x + kHeld * kMT; at < M; at += kMT)
      if (at % n == n - 1 && (uint32_t)(c_key(at, keys[at]) >> 32) == last) tied = 1u;
  }
  __syncthreads();
  if (tied && last) {
    // every candidate above the k-th best c is in the list; those that equal it are taken in index order
    uint32_t a = 0;
    for (uint32_t i = 0; i < k; i++) a += (uint32_t)(best[i] >> 32) > last;
    __syncthreads();
    for (uint32_t b = 0; b < k && a < k; b++) {
      if (fin[b]) {
        if (ordered(score[b]) == last) {
          if (threadIdx.x == 0) best[a] = key_of(score[b], b * V + j.eos);
          a++;
        }
        continue;
      }
      const float *x = j.logits + (uint64_t)(r0 + b) * j.ld;
      for (uint32_t v0 = 0; v0 < V && a < k; v0 += kMT) {
        const uint32_t v = v0 + threadIdx.x;
        const bool hit = v < V && ordered(c_of(b, x[v])) == last;
        const uint32_t votes = __ballot_sync(0xffffffffu, hit);
        if (lane == 0) warp_n[warp] = __popc(votes);
        __syncthreads();
        uint32_t at = a, all = 0;
        for (uint32_t w = 0; w < kMT / 32; w++) {
          if (w < warp) at += warp_n[w];
          all += warp_n[w];
        }
        at += __popc(votes & ((1u << lane) - 1u));
        if (hit && at < k) best[at] = (uint64_t)last << 32 | (0xffffffffu - (b * V + v));
        a += all;
        __syncthreads();
      }
    }
    __syncthreads();
  }
  if (threadIdx.x < k) {
    const uint64_t c = best[threadIdx.x];
    const uint32_t r = r0 + threadIdx.x, b = key_idx(c) / V, v = key_idx(c) % V;
    j.parent[r] = c ? r0 + b : P0_KV_NONE;
    j.token[r] = c ? v : P0_KV_NONE;
    j.score_out[r] = c ? key_val(c) : -INFINITY;
    if (j.fin_out) j.fin_out[r] = c ? (uint32_t)(fin[b] || v == j.eos) : 0u;
  }
}

}  // namespace

extern "C" p0_status p0_beam_select(p0_ctx *c, const p0_beam_args *a) {
  if (!c || !a) return P0_EINVAL;
  const char *op = "beamSelect";
  if (!a->groups) return P0_OK;
  if (!a->beams || a->beams > kMaxBeams) return p0_fail(c, P0_EINVAL, "%s: %u beams (1 to %u)", op, a->beams, kMaxBeams);
  if (!a->V || (uint64_t)a->beams * a->V >= 0xffffffffull) return p0_fail(c, P0_EINVAL, "%s: %u beams of %u tokens pass 32 bits", op, a->beams, a->V);
  const uint64_t ld = a->ld ? a->ld : a->V, R = (uint64_t)a->groups * a->beams;
  if (ld < a->V) return p0_fail(c, P0_EINVAL, "%s: row stride %u < V %u", op, a->ld, a->V);
  if (R > 65535) return p0_fail(c, P0_EINVAL, "%s: %llu rows (at most 65535)", op, (unsigned long long)R);
  if (a->fin.id && a->eos >= a->V) return p0_fail(c, P0_EINVAL, "%s: eos %u outside the vocabulary of %u", op, a->eos, a->V);
  if (a->off > (1ull << 60)) return p0_fail(c, P0_EINVAL, "%s: logits offset", op);
  BeamJob j = {};
  if (a->V > kMaxSplit * kMaxChunks * kChunk) return p0_fail(c, P0_EINVAL, "%s: a vocabulary of %u (at most %u)", op, a->V, kMaxSplit * kMaxChunks * kChunk);
  // parts per row: as few rounds of chunks as the resident CTAs allow, counting a part's own work as three of them
  j.nchunk = (a->V - 1) / kChunk + 1;
  const uint64_t slots = (uint64_t)c->sm_count * 4;
  uint64_t best = ~0ull;
  for (uint32_t ns = 1; ns <= j.nchunk && ns <= kMaxSplit; ns++) {
    const uint64_t cost = ((R * ns + slots - 1) / slots) * ((j.nchunk + ns - 1) / ns + 3);
    if (cost < best && (j.nchunk + ns - 1) / ns <= kMaxChunks) { best = cost; j.nsplit = ns; }
  }
  P0Range rl, rs, rf, rp, rt, ro, rfo;
  p0_status st;
  if ((st = p0_range(c, a->logits, a->off * 4, ((R - 1) * ld + a->V) * 4, op, "logits", &rl))) return st;
  if ((st = p0_range(c, a->score, 0, R * 4, op, "score", &rs))) return st;
  if ((st = p0_range(c, a->fin, 0, R * 4, op, "fin", &rf, true))) return st;
  if ((st = p0_range(c, a->parent, 0, R * 4, op, "parent", &rp))) return st;
  if ((st = p0_range(c, a->token, 0, R * 4, op, "token", &rt))) return st;
  if ((st = p0_range(c, a->score_out, 0, R * 4, op, "scoreOut", &ro))) return st;
  if ((st = p0_range(c, a->fin_out, 0, R * 4, op, "finOut", &rfo, true))) return st;
  for (const P0Range *r : {&rl, &rs, &rf, &rp, &rt, &ro, &rfo})
    if ((uintptr_t)r->base % 4) return p0_fail(c, P0_EALIGN, "%s: buffers must be 4-byte aligned", op);
  j.logits = (const float *)rl.base;
  j.ld = ld;
  j.score = (const float *)rs.base;
  j.fin = (const uint32_t *)rf.base;
  j.groups = a->groups;
  j.beams = a->beams;
  j.V = a->V;
  j.eos = a->eos;
  j.parent = (uint32_t *)rp.base;
  j.token = (uint32_t *)rt.base;
  j.score_out = (float *)ro.base;
  j.fin_out = (uint32_t *)rfo.base;
  const uint64_t parts = R * j.nsplit;
  uint32_t *cnt;
  void *ws;
  cudaSetDevice(c->device);
  if ((st = p0_workspace(c, 0, parts * (a->beams + 1) * 8 + parts * 8, &cnt, &ws))) return st;
  j.keys = (uint64_t *)ws;
  j.stat = (float2 *)(j.keys + parts * (a->beams + 1));
  const dim3 grid(j.nsplit, (unsigned)R);
  if ((uintptr_t)rl.base % 16 == 0 && ld % 4 == 0 && a->V % 4 == 0) launch_dep(beam_scan_kernel<true>, grid, dim3(kT), 0, c->stream, j);
  else launch_dep(beam_scan_kernel<false>, grid, dim3(kT), 0, c->stream, j);
  if ((st = p0_launched(c, op))) return st;
  launch_dep(beam_merge_kernel, dim3(a->groups), dim3(kMT), 0, c->stream, j);
  return p0_launched(c, "beamSelect merge");
}
