// beam.cu -- beamSelect: the k best continuations of every group of k beams over the vocabulary (no counterpart in the
// reference, which decodes one hypothesis by argmax / argmaxM, engine/llm/lops.js:416-436).
//   lse_b = log sum_v exp(x[b, v]),  c[b, v] = score[b] + (x[b, v] - lse_b),  the k largest c, ties to the lowest b * V + v
// One pass over the logits (they are the only traffic that counts: 4 bytes per candidate): each CTA takes 4096 logits of
// one row into registers, reduces their (max, sum exp) and keeps the k + 1 largest by (x, lowest index). A second kernel
// merges: lse per row, then the group's k best among the kept ones. Within a row c does not decrease as x grows, so every
// candidate above the k-th best c has been kept; candidates that round to the very same c as the k-th best may not have
// been, and where that can be (a chunk's last kept one ties with it) the merge looks the row's logits up again in index
// order.
#include "internal.h"
#include "launch.cuh"

namespace {

constexpr int kT = 256, kPer = 16;               // threads, logits per thread
constexpr uint32_t kChunk = kT * kPer;
constexpr uint32_t kMaxBeams = 16;
constexpr uint32_t kMaxList = (kMaxBeams + 1) * kPer;

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
  uint32_t groups, beams, V, eos, nchunk;
  uint64_t *keys;      // [rows][nchunk][beams + 1]
  float2 *stat;        // [rows][nchunk] (max, sum exp(x - max))
  uint32_t *parent, *token, *fin_out;
  float *score_out;
};

template <bool WIDE>
__global__ void __launch_bounds__(kT) beam_scan_kernel(BeamJob j) {
  dep_enter();
  __shared__ uint64_t tops[kT / 32 * (kMaxBeams + 1)], list[kMaxList], found;
  __shared__ float red[2][kT / 32];
  __shared__ uint32_t count;
  const uint32_t row = blockIdx.y, chunk = blockIdx.x, n = j.beams + 1, base = chunk * kChunk;
  if (j.fin && j.fin[row]) return;   // a finished beam has one candidate, whatever its logits
  const float *x = j.logits + row * j.ld;
  float v[kPer];
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < kPer / 4; i++) {
      const uint32_t at = base + (i * kT + threadIdx.x) * 4u;
      const float4 f = at < j.V ? __ldcs(reinterpret_cast<const float4 *>(x + at)) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint32_t at = base + i * kT + threadIdx.x;
      v[i] = at < j.V ? __ldcs(x + at) : -INFINITY;
    }
  }
  const auto index = [&](int i) { return WIDE ? base + ((i / 4) * kT + threadIdx.x) * 4u + (i & 3) : base + i * kT + threadIdx.x; };
  float mx = -INFINITY;
  uint32_t at = 0;
#pragma unroll
  for (int i = 0; i < kPer; i++)
    if (v[i] > mx) { mx = v[i]; at = index(i); }   // indexes grow with i: the lowest of equal ones
  if (threadIdx.x == 0) count = 0u;
  float m = mx;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31u) == 0) red[0][threadIdx.x >> 5] = m;
  const uint64_t mine = key_of(mx, at), thr = nth_of_threads(mine, n, tops, &found);
#pragma unroll
  for (int w = 0; w < kT / 32; w++) m = fmaxf(m, red[0][w]);
  // sum exp(x - m): a chunk of -inf alone adds 0, a NaN or +inf makes its row's lse NaN, and with it every c
  float s = 0.0f;
  const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int i = 0; i < kPer; i++) s += expf(v[i] - ref);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31u) == 0) red[1][threadIdx.x >> 5] = s;
  if (mine >= thr) {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint64_t k = key_of(v[i], index(i));
      if (k >= thr) list[atomicAdd(&count, 1u)] = k;   // at most n threads hold such keys, kPer each
    }
  }
  __syncthreads();
  uint64_t *out = j.keys + ((uint64_t)row * j.nchunk + chunk) * n;
  const uint32_t c = count;
  for (uint32_t i = threadIdx.x; i < c; i += kT) {
    uint32_t above = 0;
    for (uint32_t q = 0; q < c; q++) above += list[q] > list[i];
    if (above < n) out[above] = list[i];
  }
  if (threadIdx.x < n && threadIdx.x >= c) out[threadIdx.x] = 0ull;
  if (threadIdx.x == 0) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < kT / 32; w++) s += red[1][w];
    j.stat[(uint64_t)row * j.nchunk + chunk] = make_float2(m, s);
  }
}

// one CTA per group
constexpr int kMT = 512;
constexpr uint32_t kMaxTops = 4096;   // chunks of a group's rows
__global__ void __launch_bounds__(kMT) beam_merge_kernel(BeamJob j) {
  dep_enter();
  __shared__ float lse[kMaxBeams], score[kMaxBeams];
  __shared__ uint32_t fin[kMaxBeams];
  __shared__ uint64_t tops[kMT / 32 * kMaxBeams], found, kth, best[kMaxBeams];
  __shared__ uint64_t list[kMaxBeams * (kMaxBeams + 1)];
  __shared__ uint32_t chosen[kMaxBeams], n_tops, n_list, tied, warp_n[kMT / 32];
  extern __shared__ uint64_t cand[];   // [kMaxTops] chunk tops: c's order << 32 | chunk
  const uint32_t g = blockIdx.x, k = j.beams, n = k + 1, r0 = g * k, nc = j.nchunk, V = j.V;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  for (uint32_t b = warp; b < k; b += kMT / 32) {
    const bool done = j.fin && j.fin[r0 + b];
    float m = -INFINITY, s = 0.0f;
    if (!done) {
      const float2 *st = j.stat + (uint64_t)(r0 + b) * nc;
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
      score[b] = j.score[r0 + b];
      fin[b] = done;
    }
  }
  if (threadIdx.x < kMaxBeams) best[threadIdx.x] = 0ull;
  if (threadIdx.x == 0) { n_tops = 0u; n_list = 0u; tied = 0u; kth = 0ull; }
  __syncthreads();
  // c of a kept logit; its key orders by c, then by the lowest b * V + v
  const auto c_of = [&](uint32_t b, float x) { return __fadd_rn(score[b], __fsub_rn(x, lse[b])); };
  const auto c_key = [&](uint32_t b, uint64_t kx) { return kx ? key_of(c_of(b, key_val(kx)), b * V + key_idx(kx)) : 0ull; };
  const auto kept = [&](uint32_t chunk, uint32_t i) {   // chunk: b * nc + its chunk
    const uint32_t b = chunk / nc;
    if (fin[b]) return chunk % nc == 0 && i == 0 ? key_of(score[b], b * V + j.eos) : 0ull;
    return c_key(b, j.keys[((uint64_t)r0 * nc + chunk) * n + i]);
  };
  // the k-th largest chunk top, by value: at least k candidates are no smaller
  uint64_t mine = 0;
  for (uint32_t i = threadIdx.x; i < k * nc; i += kMT) {
    const uint64_t t = kept(i, 0);
    if (t > mine) mine = t;
  }
  uint32_t bound = (uint32_t)(nth_of_threads(mine, k, tops, &found) >> 32);
  if (!bound) bound = 1u;
  for (uint32_t i = threadIdx.x; i < k * nc; i += kMT) {
    const uint32_t o = (uint32_t)(kept(i, 0) >> 32);
    if (o >= bound) {
      cand[atomicAdd(&n_tops, 1u)] = (uint64_t)o << 32 | i;
    }
  }
  __syncthreads();
  const uint32_t nt = n_tops;
  // the k best of them (by value, any of equal ones)
  for (uint32_t i = threadIdx.x; i < nt; i += kMT) {
    uint32_t above = 0;
    for (uint32_t q = 0; q < nt; q++) above += cand[q] > cand[i];
    if (above < k) chosen[above] = (uint32_t)cand[i];
    if (above == k - 1) kth = cand[i];
  }
  __syncthreads();
  const uint32_t nch = min(nt, k);
  for (uint32_t i = threadIdx.x; i < nch * n; i += kMT) {
    const uint64_t c = kept(chosen[i / n], i % n);
    if (c) list[atomicAdd(&n_list, 1u)] = c;
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
  for (uint32_t i = threadIdx.x; i < nch; i += kMT)
    if (last && (uint32_t)(kept(chosen[i], n - 1) >> 32) == last) tied = 1u;   // more of them may follow in that chunk
  for (uint32_t i = threadIdx.x; i < nt; i += kMT)
    if (cand[i] < kth && (uint32_t)(cand[i] >> 32) == last) tied = 1u;         // or begin in one that was left out
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
  j.nchunk = (a->V - 1) / kChunk + 1;
  if ((uint64_t)a->beams * j.nchunk > kMaxTops)
    return p0_fail(c, P0_EINVAL, "%s: %u beams of %u tokens (at most %u chunks of %u logits in a group)", op, a->beams, a->V, kMaxTops, kChunk);
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
  const uint64_t parts = R * j.nchunk;
  uint32_t *cnt;
  void *ws;
  cudaSetDevice(c->device);
  if ((st = p0_workspace(c, 0, parts * (a->beams + 1) * 8 + parts * 8, &cnt, &ws))) return st;
  j.keys = (uint64_t *)ws;
  j.stat = (float2 *)(j.keys + parts * (a->beams + 1));
  const dim3 grid(j.nchunk, (unsigned)R);
  if ((uintptr_t)rl.base % 16 == 0 && ld % 4 == 0 && a->V % 4 == 0) launch_dep(beam_scan_kernel<true>, grid, dim3(kT), 0, c->stream, j);
  else launch_dep(beam_scan_kernel<false>, grid, dim3(kT), 0, c->stream, j);
  if ((st = p0_launched(c, op))) return st;
  launch_dep(beam_merge_kernel, dim3(a->groups), dim3(kMT), kMaxTops * 8, c->stream, j);
  return p0_launched(c, "beamSelect merge");
}
