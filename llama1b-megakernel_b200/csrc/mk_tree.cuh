// Attention of drafted tokens over a paged cache.
//
// Sequence b has prefix_b committed positions in its pages and, behind them, n_b
// drafted nodes whose K/V rows sit at positions prefix_b + j. Node i sees every
// committed position and those nodes j whose bit (i, j) is set (itself and its
// ancestors in a tree; j <= i for a chunk of a prompt):
//   s_j = scale q_i . k_j,  p_j = exp(s_j - m),  o = sum p_j v_j / sum p_j,
//   lse = m + log sum p_j,  m = max_j s_j,
// per query head, the sums in fp32. A row that sees nothing gets o = 0 and
// lse = -inf.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "mk_device.cuh"
#include "mk_kv8.cuh"

namespace mk {

constexpr int kTreeMaxNodes = 256;

struct TreeParams {
  const __nv_bfloat16* q;           // [rows][NQ][64]
  KVLayer kv;
  const int* cu_nodes;              // [batch + 1]
  const unsigned long long* mask;   // [rows][words]
  const int* prefix;                // [batch]
  int rows, words, max_nodes, max_len, NQ, group;
  float scale;
  __nv_bfloat16* out;               // [rows][NQ][64]
  float* lse;                       // [rows][NQ] or null
  int* error;
};

// The sequence's rows and lengths; false (and the error word) when they do not
// fit what the call was told.
__device__ __forceinline__ bool tree_sequence(const TreeParams& p, int b, int& row0, int& nodes, int& prefix) {
  row0 = p.cu_nodes[b];
  nodes = p.cu_nodes[b + 1] - row0;
  prefix = p.prefix[b];
  if (row0 < 0 || nodes < 0 || nodes > p.max_nodes || row0 > p.rows - nodes || prefix < 0 ||
      prefix > p.max_len - nodes) {
    atomicExch(p.error, 1);
    return false;
  }
  return true;
}

template <bool kFp8>
__global__ void __launch_bounds__(256) tree_attn_kernel(const __grid_constant__ TreeParams p) {
  pdl_trigger();
  pdl_wait();
  const KVLayer& kv = p.kv;
  const int i = blockIdx.x, g = blockIdx.y, b = blockIdx.z, h = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int row0, nodes, prefix;
  if (!tree_sequence(p, b, row0, nodes, prefix) || i >= nodes || h >= p.group) return;
  const int row = row0 + i, head = g * p.group + h, end = prefix + nodes;
  const uint32_t* q = reinterpret_cast<const uint32_t*>(p.q + ((size_t)row * p.NQ + head) * 64);
  auto value = [&](const uint8_t* pool, const uint8_t* scales, size_t r, int d2) {  // dims 2 d2, 2 d2 + 1
    if (!kFp8) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(pool)[r * 32 + d2];
      return make_float2(bf_lo(w), bf_hi(w));
    }
    float2 f = e4m3x2_to_float2(reinterpret_cast<const uint16_t*>(pool)[r * 32 + d2]);
    const float s = e8m0_value(scales[r]);
    return make_float2(f.x * s, f.y * s);
  };
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int c0 = 0; c0 < end; c0 += 32) {
    const int pos = c0 + lane, j = pos - prefix;
    bool seen = pos < end;
    if (seen && j >= 0) seen = (p.mask[(size_t)row * p.words + (j >> 6)] >> (j & 63)) & 1;
    int page = -1;
    if (pos < end) {
      page = kv.block_tables[(size_t)b * kv.max_blocks + pos / kv.ps];
      if (page < 0 || page >= kv.num_pages) {
        atomicExch(p.error, 1);
        page = -1;
      }
    }
    seen = seen && page >= 0;
    const int64_t r = page >= 0 ? ((int64_t)page * kv.NKV + g) * kv.ps + pos % kv.ps : -1;
    float s = -INFINITY;
    if (seen) {
      s = 0.f;
      for (int d = 0; d < 32; ++d) {
        const float2 k = value(kv.k, kv.k_scales, r, d);
        const uint32_t w = q[d];
        s = fmaf(bf_lo(w), k.x, fmaf(bf_hi(w), k.y, s));
      }
      s *= p.scale;
    }
    float cm = s;
    for (int x = 16; x; x >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, x));
    const float mn = fmaxf(m, cm);
    // a maximum of -inf is taken as 0: exp(-inf) is 0 there, and a NaN score stays one
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = __expf(m - mu);
    const float e = __expf(s - mu);
    l = l * alpha + warp_sum(e);
    m = mn;
    o0 *= alpha;
    o1 *= alpha;
    for (int t = 0; t < 32; ++t) {
      const float pt = __shfl_sync(0xffffffffu, e, t);
      const int64_t rt = __shfl_sync(0xffffffffu, r, t);
      if (!__shfl_sync(0xffffffffu, (int)seen, t)) continue;  // a masked row is not read at all
      const float2 v = value(kv.v, kv.v_scales, rt, lane);
      o0 = fmaf(pt, v.x, o0);
      o1 = fmaf(pt, v.y, o1);
    }
  }
  const bool any = l != 0.f;  // NaN counts as something
  reinterpret_cast<__nv_bfloat162*>(p.out + ((size_t)row * p.NQ + head) * 64)[lane] =
      __floats2bfloat162_rn(any ? o0 / l : 0.f, any ? o1 / l : 0.f);
  if (p.lse && lane == 0) p.lse[(size_t)row * p.NQ + head] = any ? m + logf(l) : -INFINITY;
}

}  // namespace mk
