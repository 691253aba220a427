// Log probabilities of given tokens, the entropy and the most likely tokens of
// rows of logits, each logit read once.
//
// With m = max_j x_j, s = sum_j exp(x_j - m) and w = sum_j exp(x_j - m) (x_j - m):
//   log p_t = x_t - m - log s,   H = -sum_j p_j log p_j = log s - w / s.
// A logit of -inf (a forbidden token) adds nothing to s or w. A row without a
// logit above -inf has no distribution: its log probabilities are -inf and its
// entropy 0. A NaN or +inf in a row makes its log probabilities and entropy NaN.
// Alternatives are ordered by (logit descending, id ascending).
//
// A CTA of 256 threads takes a slice of a row (the whole row where there are many
// rows), 256 * E logits at a time (a chunk), the next chunk on its way into registers while
// one is used. Each thread carries (m, s, w) of its own logits; parts join under a
// common maximum m' as
//   s' = sum_i a_i s_i,  w' = sum_i a_i (w_i + (m_i - m') s_i),  a_i = exp(m_i - m').
// The `top` largest: in the first chunk the maxima of 64 groups of four threads are
// ranked, and the top-th of them is a threshold that at least `top` logits reach
// and few more (64 -ln(1 - top / 64) of random ones: 24 for 20, 44 for 32); those are
// collected and ranked among themselves, and the top-th is the threshold for what
// follows. Later chunks add what passes it to the candidates, which are ranked
// again, the threshold rising, after 2, 4, 8 ... chunks: between two rankings about
// `top` more come, and the warps run free of each other. (Ranked rarely, nearly
// every warp went through the collection in every chunk: 28 instructions issued a
// logit, 8 of them for the sums.) Chunks with more than kLpCandidates beyond the
// threshold (rising or equal logits) are read again and chosen from one by one. The
// slices of a row are a cluster; its first CTA joins them, ranking out of their lists
// what reaches the largest of the lists' last keys.
//
// Many fp32 rows are bound by memory: 2,047 of 128,256 in 184 to 193 us (two GPUs), 5.4 to
// 5.7 TB/s. Of bf16, with half the bytes for as many exponentials and comparisons, by
// instruction latency: 200 rows with five alternatives in 24.9 us (2.0 TB/s, 15
// instructions a logit), 17.4 without. One row is latency: 9.9 to 10.5 us with twenty.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "mk_device.cuh"

namespace mk {

constexpr int kLogprobsMaxTop = 32;
constexpr int kLpThreads = 256;
constexpr int kLpCandidates = 512;
constexpr int kLpMaxSlices = 16;  // CTAs of a cluster
static_assert(kLpMaxSlices * kLogprobsMaxTop <= kLpCandidates, "a cluster's lists fit the candidates");
constexpr float kLog2e = 1.4426950408889634f;
// Distances below a maximum count as no further than this: their exponential is 0 long before, and 0
// times the distance times a count of logits has to be 0 (logits at the type's lowest value are 3e38
// away: twice that is infinite, and 0 times it a NaN).
constexpr float kLpFar = -1e20f;

struct LogprobsParams {
  const void* logits;   // [rows][ld] fp32 or bf16, the first V columns
  long long ld;
  int rows, V, num_targets, top, slices;
  int slice_len;        // logits of a slice: whole chunks
  const int* targets;   // [rows][num_targets], negative: none
  float* logprobs;      // [rows][num_targets]
  float* entropy;       // [rows]
  int* top_ids;         // [rows][top]
  float* top_logprobs;  // [rows][top]
  int* error;
};

__device__ __forceinline__ float lp_load(const float* x, int64_t i) { return x[i]; }
__device__ __forceinline__ float lp_load(const __nv_bfloat16* x, int64_t i) { return __bfloat162float(x[i]); }

// (logit, id) as one integer that orders as the alternatives do; -0 counts as 0.
__device__ __forceinline__ unsigned long long lp_key(float x, int id) {
  return ((unsigned long long)float_key(x + 0.f) << 32) | (0xFFFFFFFFu - (uint32_t)id);
}
__device__ __forceinline__ float lp_value(unsigned long long key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ int lp_id(unsigned long long key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

struct LpShared {
  float4 stats;  // of the CTA's slice, for the first CTA of its cluster
  unsigned long long cand[kLpCandidates];
  unsigned long long list[kLogprobsMaxTop];
  unsigned long long best[8];
  float group[64];
  float m[8], s[8], w[8];
  float threshold;
  int count;
};

// The first `top` of the n candidates in order into sh.list, which holds 0 before.
__device__ __forceinline__ void lp_rank(LpShared& sh, int top, int n) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kLpThreads) {  // the order they came in does not matter: keys differ
    const unsigned long long mine = sh.cand[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += sh.cand[j] > mine;
    if (rank < top) sh.list[rank] = mine;
  }
  __syncthreads();
}

// The `top` largest of the CTA's keys, in order, into sh.list (0 where there are
// fewer). each(least, f) calls f with the thread's keys, those of values below
// `least` left out if it likes; `best` is the largest of their values, -inf without
// one (a NaN is nobody's largest).
template <typename Each>
__device__ __forceinline__ void lp_select(LpShared& sh, int top, float best, Each each) {
  const int tid = threadIdx.x;
  float q = best;
  q = fmaxf(q, __shfl_xor_sync(0xffffffffu, q, 1));
  q = fmaxf(q, __shfl_xor_sync(0xffffffffu, q, 2));
  if ((tid & 3) == 0) sh.group[tid >> 2] = q;
  if (tid == 0) sh.count = 0;
  if (tid < kLogprobsMaxTop) sh.list[tid] = 0;
  __syncthreads();
  if (tid < 64) {
    const float mine = sh.group[tid];
    int rank = 0;
#pragma unroll 16
    for (int i = 0; i < 64; ++i) rank += sh.group[i] > mine || (sh.group[i] == mine && i < tid);
    if (rank == top - 1) sh.threshold = mine;
  }
  __syncthreads();
  const float thr = sh.threshold;
  const unsigned long long low = (unsigned long long)float_key(thr + 0.f) << 32;
  if (best >= thr) {
    each(thr, [&](unsigned long long k) {
      if (k > low) {  // a value of at least thr: a key's lower half is not 0
        const int at = atomicAdd(&sh.count, 1);
        if (at < kLpCandidates) sh.cand[at] = k;
      }
    });
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= kLpCandidates) {
    lp_rank(sh, top, n);
    return;
  }
  unsigned long long last = ~0ull;
  for (int t = 0; t < top; ++t) {
    unsigned long long b = 0;
    each(-INFINITY, [&](unsigned long long k) {
      if (k < last) b = max(b, k);
    });
    for (int o = 16; o; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    if ((tid & 31) == 0) sh.best[tid >> 5] = b;
    __syncthreads();
    b = 0;
    for (int i = 0; i < 8; ++i) b = max(b, sh.best[i]);
    last = b;
    if (tid == 0) sh.list[t] = b;
    __syncthreads();
    if (!b) break;
  }
}

// The CTA's threads hold (m, s, w): their join, in every thread.
__device__ __forceinline__ void lp_join(LpShared& sh, float& m, float& s, float& w) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float M = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  auto shift = [](float m_, float M_, float& s_, float& w_) {
    const float d = m_ == -INFINITY ? -INFINITY : m_ - M_;  // a part without anything: exp(-inf)
    const float a = __expf(d);
    w_ = a * (w_ + fmaxf(d, kLpFar) * s_);
    s_ = a * s_;
  };
  shift(m, M, s, w);
  s = warp_sum(s);
  w = warp_sum(w);
  if (lane == 0) {
    sh.m[warp] = M;
    sh.s[warp] = s;
    sh.w[warp] = w;
  }
  __syncthreads();
  m = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, sh.m[i]);
  s = w = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float si = sh.s[i], wi = sh.w[i];
    shift(sh.m[i], m, si, wi);
    s += si;
    w += wi;
  }
}

// A row's results from its statistics and the list in sh.list.
template <typename T>
__device__ __forceinline__ void lp_finish(const LogprobsParams& p, const LpShared& sh, int row, float m, float s, float w) {
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.ld;
  const float nan = __uint_as_float(0x7FFFFFFFu);
  const bool none = m == -INFINITY && s == 0.f;    // nothing but -inf (a NaN makes s one)
  // x - m before log s is subtracted: rounded together, m and log s would lose as many of log s's
  // bits as m is larger (all of them at the type's lowest value)
  const float top = none ? 0.f : m, ls = none ? 0.f : logf(s);
  if (threadIdx.x == 0) p.entropy[row] = none ? 0.f : ls - w / s;
  for (int j = threadIdx.x; j < p.num_targets; j += kLpThreads) {
    const int t = p.targets[(int64_t)row * p.num_targets + j];
    float v = 0.f;
    if (t >= p.V) {
      atomicExch(p.error, 1);
      v = nan;
    } else if (t >= 0) {
      v = (lp_load(x, t) - top) - ls;
    }
    p.logprobs[(int64_t)row * p.num_targets + j] = v;
  }
  if (threadIdx.x < p.top) {
    const unsigned long long k = sh.list[threadIdx.x];  // 0 only beside a NaN
    p.top_ids[(int64_t)row * p.top + threadIdx.x] = k ? lp_id(k) : (int)threadIdx.x;
    p.top_logprobs[(int64_t)row * p.top + threadIdx.x] = (lp_value(k) - top) - ls;
  }
}

// One slice of a row. Thread t holds E logits of a chunk, in vectors of 16 bytes
// that neighbouring threads read side by side (kVec: every row starts on 16 bytes).
template <typename T, int E, bool kVec>
__global__ void __launch_bounds__(kLpThreads, E == 16 ? 3 : 4) logprobs_kernel(const __grid_constant__ LogprobsParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ LpShared sh;
  constexpr int N = 16 / (int)sizeof(T);         // logits of a vector
  constexpr int C = kLpThreads * E;              // of a chunk
  static_assert(E % N == 0, "whole vectors");
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.ld;
  const int i0 = slice * p.slice_len, i1 = min(p.V, i0 + p.slice_len);
  auto index = [&](int c0, int e) {
    return kVec ? c0 + ((e / N) * kLpThreads + tid) * N + e % N : c0 + e * kLpThreads + tid;
  };
  // the chunk on its way, and of bf16, whose chunks have half the bytes, the one after it
  // (three CTAs with two in flight: 25.3 us for 200 rows; four with one: 27.5)
  constexpr int W = E * sizeof(T) / 4;
  constexpr bool kTwo = sizeof(T) == 2;
  uint32_t raw[W], after[kTwo ? W : 1];
  auto fetch = [&](auto& raw, int c0) {
    if (kVec && c0 + C <= i1) {
#pragma unroll
      for (int c = 0; c < E / N; ++c) {
        const uint4 u = (reinterpret_cast<const uint4*>(x + c0))[c * kLpThreads + tid];
        raw[4 * c] = u.x;
        raw[4 * c + 1] = u.y;
        raw[4 * c + 2] = u.z;
        raw[4 * c + 3] = u.w;
      }
    } else {  // one by one, -inf past the end
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = index(c0, e);
        if constexpr (sizeof(T) == 4) {
          raw[e] = i < i1 ? reinterpret_cast<const uint32_t*>(x)[i] : 0xFF800000u;
        } else {
          const uint32_t h = i < i1 ? reinterpret_cast<const uint16_t*>(x)[i] : 0xFF80u;
          raw[e / 2] = e & 1 ? raw[e / 2] | h << 16 : h;
        }
      }
    }
  };
  float v[E];
  auto take = [&] {
#pragma unroll
    for (int e = 0; e < E; ++e)
      v[e] = sizeof(T) == 4 ? __uint_as_float(raw[e % (E * sizeof(T) / 4)]) : (e & 1) ? bf_hi(raw[e / 2]) : bf_lo(raw[e / 2]);
  };
  auto largest = [&] {
    float best = v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) best = fmaxf(best, v[e]);
    return best;
  };
  auto own = [&](int c0, float least, auto f) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (v[e] >= least && index(c0, e) < i1) f(lp_key(v[e], index(c0, e)));
  };
  float m = -INFINITY, s = 0.f, w = 0.f;
  float thr = -INFINITY;
  unsigned long long low = 0;
  int kept = 0;
  // the list becomes the candidates; what follows has to beat its last
  auto settle = [&] {
    const unsigned long long mine = tid < p.top ? sh.list[tid] : 0;
    low = sh.list[p.top - 1];
    thr = low ? lp_value(low) : -INFINITY;
    kept = p.top;
    if (!low) {  // fewer so far: as many as there are
      kept = 0;
      for (int t = 0; t < p.top; ++t) kept += sh.list[t] != 0;
    }
    if (tid < p.top) sh.cand[tid] = mine;
    if (tid == 0) sh.count = kept;
    __syncthreads();
  };
  // the chunk in v against the candidates, as a whole
  auto choose = [&](int c0) {
    const unsigned long long old = tid < kept ? sh.cand[tid] : 0;
    const float best = largest();
    __syncthreads();
    lp_select(sh, p.top, old ? fmaxf(best, lp_value(old)) : best, [&](float least, auto f) {
      own(c0, least, f);
      if (old) f(old);
    });
    settle();
  };
  const int chunks = (i1 - i0 + C - 1) / C;
  int from = 0, next = 1;  // the segment of chunks since the list was last settled, and its end
  fetch(raw, i0);
  if (kTwo && chunks > 1) fetch(after, i0 + C);
  for (int c = 0; c < chunks; ++c) {
    const int c0 = i0 + c * C;
    take();
    if constexpr (kTwo) {
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = after[i];
      if (c + 2 < chunks) fetch(after, c0 + 2 * C);
    } else {
      if (c + 1 < chunks) fetch(raw, c0 + C);
    }
    const float best = largest();
    if (best > m) {
      const float a = m == -INFINITY ? 0.f : exp2_approx((m - best) * kLog2e);
      w = m == -INFINITY ? 0.f * s : a * fmaf(fmaxf(m - best, kLpFar), s, w);  // 0 * s: a NaN stays
      s *= a;
      m = best;
    }
    const float mu = m == -INFINITY ? 0.f : m;  // exp(-inf - 0) is 0, and a NaN stays one
    const float2 shift = make_float2(-mu, -mu), base2 = make_float2(kLog2e, kLog2e);
    float2 sx[2] = {make_float2(s, 0.f), make_float2(0.f, 0.f)}, wx[2] = {make_float2(w, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int e = 0; e < E; e += 2) {  // two chains of pairs
      float2 d = add2(make_float2(v[e], v[e + 1]), shift);
      const float2 x2 = mul2(d, base2);
      const float2 a = make_float2(exp2_approx(x2.x), exp2_approx(x2.y));
      d = make_float2(fmaxf(d.x, kLpFar), fmaxf(d.y, kLpFar));  // 0 * -inf adds nothing
      const int c = (e >> 1) & 1;
      sx[c] = add2(sx[c], a);
      wx[c] = fma2(a, d, wx[c]);
    }
    s = (sx[0].x + sx[0].y) + (sx[1].x + sx[1].y);
    w = (wx[0].x + wx[0].y) + (wx[1].x + wx[1].y);
    if (!p.top) continue;
    if (c == 0) {
      choose(c0);
      from = 1;
      next = 2;
      continue;
    }
    if (best >= thr)
      own(c0, thr, [&](unsigned long long k) {
        if (k > low) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kLpCandidates) sh.cand[at] = k;
        }
      });
    if (c + 1 != next && c + 1 != chunks) continue;
    __syncthreads();
    const int n = sh.count;
    if (n <= kLpCandidates) {
      if (tid < kLogprobsMaxTop) sh.list[tid] = 0;
      lp_rank(sh, p.top, n);
      settle();
    } else {
      // more than the list holds: what it had before is still its first entries;
      // the segment's chunks are read once more and chosen from one by one
      __syncthreads();
      for (int r = from; r <= c; ++r) {
        fetch(raw, i0 + r * C);
        take();
        choose(i0 + r * C);
      }
      if (c + 1 < chunks) fetch(raw, c0 + C);
    }
    from = c + 1;
    next = 2 * (c + 1);
  }
  lp_join(sh, m, s, w);
  if (p.slices > 1) {
    if (tid == 0) sh.stats = make_float4(m, s, w, 0.f);
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (slice == 0) {
      auto remote = [&](const void* at, int q) {
        uint32_t a;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(at)), "r"(q));
        return a;
      };
      auto key_of = [&](int q, int i) {
        unsigned long long k;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k) : "r"(remote(&sh.list[i], q)) : "memory");
        return k;
      };
      m = -INFINITY;
      s = w = 0.f;
      if (tid < p.slices) {
        float unused;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(m), "=f"(s), "=f"(w), "=f"(unused)
                     : "r"(remote(&sh.stats, tid))
                     : "memory");
      }
      // a slice's list alone has `top` keys that reach its last: whatever is below the
      // largest of the lasts is out, and little more than `top` keys are left to rank
      unsigned long long key[kLpMaxSlices * kLogprobsMaxTop / kLpThreads], least = 0;
      const int n = p.slices * p.top;
#pragma unroll
      for (int c = 0; c < kLpMaxSlices * kLogprobsMaxTop / kLpThreads; ++c) {
        const int i = c * kLpThreads + tid;
        key[c] = i < n ? key_of(i / p.top, i % p.top) : 0;
        if (i < n && i % p.top == p.top - 1) least = max(least, key[c]);
      }
      for (int o = 16; o; o >>= 1) least = max(least, __shfl_xor_sync(0xffffffffu, least, o));
      if ((tid & 31) == 0) sh.best[tid >> 5] = least;
      if (tid == 0) sh.count = 0;
      lp_join(sh, m, s, w);  // and a barrier for the lines above
#pragma unroll
      for (int i = 0; i < 8; ++i) least = max(least, sh.best[i]);
      least = max(least, 1ull);
      __syncthreads();
      if (tid < kLogprobsMaxTop) sh.list[tid] = 0;  // the keys of this CTA's own list are in registers
#pragma unroll
      for (int c = 0; c < kLpMaxSlices * kLogprobsMaxTop / kLpThreads; ++c)
        if (key[c] >= least) sh.cand[atomicAdd(&sh.count, 1)] = key[c];
      __syncthreads();
      lp_rank(sh, p.top, sh.count);
    }
    // nobody leaves while its list may still be read
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (slice) return;
  }
  lp_finish<T>(p, sh, row, m, s, w);
}

}  // namespace mk
