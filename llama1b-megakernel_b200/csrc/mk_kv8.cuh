// Writing rows into a layer's paged K/V cache, in bf16 or in 8 bits, and
// reading them back.
//
// The 8-bit cache holds e4m3 codes and, for each (position, kv head), one
// E8M0 scale byte: a row x[64] is stored as codes c_d = e4m3(x_d 2^-e) with
//   e = the smallest integer, at least -110, with max|x_d| <= 448 * 2^e,
// and the byte e + 127. Because the scale is a power of two, x 2^-e and c 2^e
// are exact: the one rounding is that of the code (to nearest, ties to even),
// and what a row reads back as is a bf16 number (4 significant bits). A scale
// that maps max|x| onto 448 would not be more precise: the codes are floating
// point, so only values below 2^-6 of the largest code's unit would gain. A row
// holds 65 bytes where bf16 takes 128. A row with an infinity or a NaN gets the
// scale byte 255 (E8M0's NaN) and reads back as NaN, so nothing infinite ever
// turns into a finite number.
//
// New rows come as the q/k/v GEMM writes them, in the packed RoPE-pair order
// (column head * 64 + 2 d + h holds dim d + 32 h), and are rotated here:
//   y_d = x_d c_d - x_{d+32} s_d,  y_{d+32} = x_{d+32} c_{d+32} + x_d s_{d+32}
// from the bf16 table row of the row's position, in fp32: products of two bf16
// numbers are exact there, so a rotated value is rounded once by the sum and
// once by its bf16 or e4m3 store.
//
// Both kernels move bytes. 4,093 rows of 48 heads are written in 13.3 us (47 MB, 3.6
// TB/s; 0.5 more with a head a lane group instead of two): what remains is the latency of two
// rounds of loads (rows, slot and position, then the tables and the page) in three
// waves of CTAs. 32 x 8,191 positions read back in 131 us (5.7 TB/s). One row: 1.8 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "mk_device.cuh"

namespace mk {

// One layer of a paged cache (MkKVLayer with the formats' types erased).
struct KVLayer {
  uint8_t* k;                // [num_pages][NKV][ps][64] bf16 or e4m3
  uint8_t* v;
  uint8_t* k_scales;         // [num_pages][NKV][ps] E8M0 (8-bit cache only)
  uint8_t* v_scales;
  const int* block_tables;   // [batch][max_blocks]
  int ps, num_pages, NKV, max_blocks, batch;
};

constexpr int kScaleNaN = 255;    // E8M0's NaN
constexpr int kMinExponent = -110;

// The scale byte of a row whose largest |x| has these bits.
__device__ __forceinline__ int e8m0_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return kScaleNaN;
  // |x| = (1 + f) 2^k: 448 = 1.75 * 2^8 covers it at e = k - 8 up to f = 0.75
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u);
  return max(e, kMinExponent) + 127;
}

// 2^(127 - byte): the factor a row is divided by its scale with (bytes 17 .. 247 occur).
__device__ __forceinline__ float inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// The scale itself; NaN for byte 255.
__device__ __forceinline__ float e8m0_value(int byte) {
  return byte == kScaleNaN ? __uint_as_float(0x7FFFFFFFu) : byte == 0 ? __uint_as_float(0x00400000u)
                                                                      : __uint_as_float((uint32_t)byte << 23);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two e4m3 codes (low byte first) as floats.
__device__ __forceinline__ float2 e4m3x2_to_float2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

struct KVWriteParams {
  const uint8_t* qkv;        // [rows][(NQ + 2 NKV) * 64] bf16, RoPE-pair order
  const __nv_bfloat16* cos_t;  // [rope_len][64]
  const __nv_bfloat16* sin_t;
  const int* seqs;           // [rows] the row's sequence
  const int* slots;          // [rows] its place in the sequence (-1: a padding row)
  const int* positions;      // [rows] its RoPE position
  int rows, NQ, rope_len;
  KVLayer kv;
  __nv_bfloat16* q_out;      // [rows][NQ][64]
  int* error;
};

// Eight lanes per two neighbouring heads of a row, 16 bytes of qkv (four RoPE pairs) of
// each, so a warp reads full 128-byte lines, a row's largest value is three shuffles away,
// and both heads share the rotation's tables; a lane's results are the dims
// 4 l .. 4 l + 3 and 32 more.
template <bool kFp8>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KVWriteParams p) {
  pdl_trigger();
  pdl_wait();
  const KVLayer& kv = p.kv;
  const uint32_t nh = p.NQ + 2 * kv.NKV, pairs = (nh + 1) / 2;
  // 32 bits: 2^32 of these would be 550 GB of qkv (a 64-bit division was a third of the kernel)
  const uint32_t unit = blockIdx.x * 32u + (threadIdx.x >> 3);
  const int l = threadIdx.x & 7;
  const int row = unit / pairs, h0 = 2 * (unit - row * pairs);
  const bool live = row < p.rows;  // whole groups of eight lanes
  const uint4* src = reinterpret_cast<const uint4*>(p.qkv) + ((size_t)row * nh + h0) * 8 + l;
  uint4 u[2];
  u[0] = live ? src[0] : make_uint4(0, 0, 0, 0);
  u[1] = live && h0 + 1 < nh ? src[8] : make_uint4(0, 0, 0, 0);
  // all that does not wait for another load, then the page, under way with the tables
  const bool rotated = live && h0 < p.NQ + kv.NKV, stored = live && h0 + 1 >= p.NQ;
  const int pos = live ? p.positions[row] : 0;
  const int slot = stored ? p.slots[row] : -1, seq = stored ? p.seqs[row] : 0;
  const int blk = slot / kv.ps, off = slot - blk * kv.ps;
  int page = -1;
  if (slot >= 0 && blk < kv.max_blocks && seq >= 0 && seq < kv.batch)
    page = kv.block_tables[(size_t)seq * kv.max_blocks + blk];
  const bool placed = pos >= 0 && pos < p.rope_len;
  uint2 cs[4] = {};  // cosines of dims 4 l .., 32 + 4 l .., sines of the same
  if (rotated && placed) {
    const uint2* c = reinterpret_cast<const uint2*>(p.cos_t + (size_t)pos * 64) + l;
    const uint2* s = reinterpret_cast<const uint2*>(p.sin_t + (size_t)pos * 64) + l;
    cs[0] = c[0];
    cs[1] = c[8];
    cs[2] = s[0];
    cs[3] = s[8];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int hd = h0 + i;
    float lo[4] = {bf_lo(u[i].x), bf_lo(u[i].y), bf_lo(u[i].z), bf_lo(u[i].w)};
    float hi[4] = {bf_hi(u[i].x), bf_hi(u[i].y), bf_hi(u[i].z), bf_hi(u[i].w)};
    const bool turn = hd < p.NQ + kv.NKV;
    if (turn) {
      const float cl[4] = {bf_lo(cs[0].x), bf_hi(cs[0].x), bf_lo(cs[0].y), bf_hi(cs[0].y)};
      const float ch[4] = {bf_lo(cs[1].x), bf_hi(cs[1].x), bf_lo(cs[1].y), bf_hi(cs[1].y)};
      const float sl[4] = {bf_lo(cs[2].x), bf_hi(cs[2].x), bf_lo(cs[2].y), bf_hi(cs[2].y)};
      const float sh[4] = {bf_lo(cs[3].x), bf_hi(cs[3].x), bf_lo(cs[3].y), bf_hi(cs[3].y)};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = lo[e], b = hi[e];
        lo[e] = a * cl[e] - b * sl[e];
        hi[e] = b * ch[e] + a * sh[e];
      }
    }
    uint32_t amax = 0;  // |x| as bits: their order is that of the numbers, NaN on top
#pragma unroll
    for (int e = 0; e < 4; ++e)
      amax = max(amax, max(__float_as_uint(lo[e]) & 0x7FFFFFFFu, __float_as_uint(hi[e]) & 0x7FFFFFFFu));
    if (kFp8) {
#pragma unroll
      for (int o = 4; o; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if (!live || hd >= nh) continue;
    if (!placed) {  // a row of no position is stored nowhere, not even its V
      atomicExch(p.error, 1);
      continue;
    }
    auto pack = [](const float(&x)[4]) {
      __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
      return make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    };
    if (hd < p.NQ) {
      uint2* q = reinterpret_cast<uint2*>(p.q_out + ((size_t)row * p.NQ + hd) * 64) + l;
      q[0] = pack(lo);
      q[8] = pack(hi);
      continue;
    }
    if (slot == -1) continue;
    if (page < 0 || page >= kv.num_pages) {
      atomicExch(p.error, 1);
      continue;
    }
    const int g = hd - p.NQ - (turn ? 0 : kv.NKV);
    const size_t r = ((size_t)page * kv.NKV + g) * kv.ps + off;
    uint8_t* pool = turn ? kv.k : kv.v;
    if (!kFp8) {
      uint2* dst = reinterpret_cast<uint2*>(pool + r * 128) + l;
      dst[0] = pack(lo);
      dst[8] = pack(hi);
      continue;
    }
    const int byte = e8m0_of(amax);
    const float f = byte == kScaleNaN ? 0.f : inv_scale(byte);
    uint32_t* dst = reinterpret_cast<uint32_t*>(pool + r * 64) + l;
    uint32_t a = 0, b = 0;
    if (byte != kScaleNaN) {
      a = e4m3x2(lo[0] * f, lo[1] * f) | (e4m3x2(lo[2] * f, lo[3] * f) << 16);
      b = e4m3x2(hi[0] * f, hi[1] * f) | (e4m3x2(hi[2] * f, hi[3] * f) << 16);
    }
    dst[0] = a;
    dst[8] = b;
    if (l == 0) (turn ? kv.k_scales : kv.v_scales)[r] = (uint8_t)byte;
  }
}

struct KVReadParams {
  KVLayer kv;
  const int* lengths;        // [batch]
  int max_len;
  __nv_bfloat16* k_out;      // [batch][NKV][max_len][64]
  __nv_bfloat16* v_out;
  int* error;
};

// One thread per 16 bytes of output (eight dims of a row), K and V both.
template <bool kFp8>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KVReadParams p) {
  pdl_trigger();
  pdl_wait();
  const KVLayer& kv = p.kv;
  const int g = blockIdx.y, b = blockIdx.z;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int pos = (int)(i >> 3), piece = (int)(i & 7);
  if (pos >= p.max_len) return;
  const size_t o = ((((size_t)b * kv.NKV + g) * p.max_len) + pos) * 8 + piece;
  uint4 kq = make_uint4(0, 0, 0, 0), vq = kq;
  if (pos < p.lengths[b]) {
    const int blk = pos / kv.ps;
    const int page = blk < kv.max_blocks ? kv.block_tables[(size_t)b * kv.max_blocks + blk] : -1;
    if (page < 0 || page >= kv.num_pages) {
      atomicExch(p.error, 1);
    } else {
      const size_t r = ((size_t)page * kv.NKV + g) * kv.ps + pos % kv.ps;
      if (!kFp8) {
        kq = reinterpret_cast<const uint4*>(kv.k)[r * 8 + piece];
        vq = reinterpret_cast<const uint4*>(kv.v)[r * 8 + piece];
      } else {
        auto decode = [](uint2 c, float s) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = e4m3x2_to_float2((uint16_t)((j < 2 ? c.x : c.y) >> (16 * (j & 1))));
            __nv_bfloat162 h = __floats2bfloat162_rn(f.x * s, f.y * s);
            w[j] = *reinterpret_cast<uint32_t*>(&h);
          }
          return make_uint4(w[0], w[1], w[2], w[3]);
        };
        kq = decode(reinterpret_cast<const uint2*>(kv.k)[r * 8 + piece], e8m0_value(kv.k_scales[r]));
        vq = decode(reinterpret_cast<const uint2*>(kv.v)[r * 8 + piece], e8m0_value(kv.v_scales[r]));
      }
    }
  }
  reinterpret_cast<uint4*>(p.k_out)[o] = kq;
  reinterpret_cast<uint4*>(p.v_out)[o] = vq;
}

}  // namespace mk
