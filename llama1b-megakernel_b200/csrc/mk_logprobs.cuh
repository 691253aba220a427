// Log probabilities of given tokens, the entropy and the most likely tokens of
// rows of logits.
//
// With m = max_j x_j, s = sum_j exp(x_j - m) and w = sum_j exp(x_j - m) (x_j - m):
//   log p_t = x_t - m - log s,   H = -sum_j p_j log p_j = log s - w / s.
// A logit of -inf (a forbidden token) adds nothing to s or w. A row without a
// logit above -inf has no distribution: its log probabilities are -inf and its
// entropy 0. A NaN or +inf in a row makes its log probabilities and entropy NaN.
// Alternatives are ordered by (logit descending, id ascending).
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "mk_device.cuh"

namespace mk {

constexpr int kLogprobsMaxTop = 32;

struct LogprobsParams {
  const void* logits;   // [rows][ld] fp32 or bf16, the first V columns
  long long ld;
  int rows, V, num_targets, top;
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

template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(const __grid_constant__ LogprobsParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red[8];
  __shared__ unsigned long long redk[8];
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.ld;
  auto sum_of = [&](float v) {
    v = warp_sum(v);
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < 8; ++i) v += red[i];
    __syncthreads();
    return v;
  };
  auto max_of = [&](unsigned long long v) {
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) redk[warp] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < 8; ++i) v = max(v, redk[i]);
    __syncthreads();
    return v;
  };
  float mx = -INFINITY;
  for (int i = tid; i < p.V; i += 256) mx = fmaxf(mx, lp_load(x, i));
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) red[warp] = mx;
  __syncthreads();
  for (int i = 0; i < 8; ++i) mx = fmaxf(mx, red[i]);
  __syncthreads();
  const float m = mx;
  float s = 0.f, w = 0.f;
  for (int i = tid; i < p.V; i += 256) {
    const float d = lp_load(x, i) - m;
    const float e = (d == -INFINITY || m == -INFINITY) ? 0.f : __expf(d);
    s += e;
    if (e != 0.f) w = fmaf(e, d, w);
  }
  s = sum_of(s);
  w = sum_of(w);
  const float lse = m == -INFINITY ? 0.f : m + logf(s);
  if (tid == 0) p.entropy[row] = m == -INFINITY ? 0.f : logf(s) - w / s;
  for (int j = tid; j < p.num_targets; j += 256) {
    const int t = p.targets[(int64_t)row * p.num_targets + j];
    float v = 0.f;
    if (t >= p.V) {
      atomicExch(p.error, 1);
      v = __uint_as_float(0x7FFFFFFFu);
    } else if (t >= 0) {
      v = lp_load(x, t) - lse;
    }
    p.logprobs[(int64_t)row * p.num_targets + j] = v;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < p.V; i += 256) {
      const unsigned long long key = lp_key(lp_load(x, i), i);
      if (key < last) best = max(best, key);
    }
    last = max_of(best);
    const int id = (int)(0xFFFFFFFFu - (uint32_t)last);
    if (tid == 0) {
      p.top_ids[(int64_t)row * p.top + k] = id;
      p.top_logprobs[(int64_t)row * p.top + k] = lp_load(x, id) - lse;
    }
  }
}

}  // namespace mk
