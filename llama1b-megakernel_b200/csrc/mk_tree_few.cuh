// Attention of few drafted rows per K/V head (mk_tree.cuh has the definition, the
// parameters and the join of split ranges): decode steps and small trees.
//
// With at most 16 rows (nodes x query heads of a K/V head) a 128-row tensor tile
// would be mostly empty and its softmax would run on a quarter of the SM, while the
// work is to stream K and V once. So a tile is 8 or 16 rows (RT eights) on
// mma.sync.m16n8k16, whose B operand comes straight from registers:
//  * three consumer warps take turns at the chunks of the range (32 positions of
//    bf16, 64 of 8-bit codes: 8 KB either way), each with its own maximum, sum and O,
//    joined in shared memory at the end; a producer warp keeps six chunks in
//    flight by TMA, two for each consumer;
//  * bf16: fragments by ldmatrix from the 128-byte-swizzled rows, P bf16;
//  * 8-bit: all products in f16, where every code is exact and one conversion makes
//    two of them. A thread's K fragment is 16 consecutive codes of a position (one
//    128-bit load; the order of dims in a sum is free, so Q is laid out to match);
//    Q goes to f16 under a power of two for each row that brings its largest value
//    to 2^14: what is lost lies below 2^-38 of it. The row's K scale multiplies the
//    score. A V fragment pairs two positions of a dim. V's scales multiply P, relative
//    to the largest one that the row has seen so far (2^E; O is in units of it, and
//    rescaled when it grows; a drafted node counts for the rows that see it).
//    A row's largest P is 2^7 (2^15 before O is rescaled), so that P in f16 is rounded
//    by 2^-11 of itself down to 2^-14, 2^-21 of the largest. What is smaller loses up
//    to 2^-25, however many positions there are: 32 of them lose at most 2^-23 of a
//    row's sum of such products if that is 8 or more (kFewEnough), which is looked at
//    before the products are rounded, until it is. Where a row has less (its largest P met
//    values of little size, or one of great size came by that it does not look at) the 32
//    positions are done again with P and V as bf16 (tree_decode's way), which rounds the
//    smallest by 2^-8 as well. (64 sequences of 2,600 to 4,100 positions: 54.9 us without
//    a look, 55.8 so; one of 1,025: 5.7 and 6.0.)
//    The positions of a block of 8 are permuted between fragment columns and rows
//    in memory (few_place) so that both loads are free of bank conflicts under the
//    64-byte swizzle.
// O is rescaled when a maximum grew by more than 8 powers of two, as in mk_tree.cuh.
//
// What bounds it: memory, where sequences fill the GPU (36 of 1,000 to 2,000 positions in
// 8 bits: 19 us; 64 of 2,600 to 4,100: 56 us, 4.0 TB/s, as their 512 CTAs end one by one),
// and the latency of a CTA's few chunks where they do not (one of 1,025 bf16: 6.2 us).
// The split of an SM was measured (consumers x stages x CTAs; 64 of 2,600 to 4,100 in 8
// bits, and 32 of 2,700 to 4,100 in bf16 with 16 rows): 3 x 6 x 4 55 and 45 us, 4 x 8 x 3 80
// and 50, 4 x 4 x 4 (32 of 8-bit: 35 against 34) and 45; with 5 or 6 CTAs registers spill.
#pragma once

#include <type_traits>

#include "mk_tree.cuh"

namespace mk {

constexpr int kFewWarps = 3;
constexpr int kFewStages = 6;
// A stage is always the same warp's, who has then waited for each of its phases. With
// another number a warp may come to a stage that others filled and drained since it
// last looked; a parity then does not tell the phase it waits for from the one before it.
static_assert(kFewStages % kFewWarps == 0, "a stage belongs to one warp");
constexpr int kFewCtas = 4;           // of an SM: 16 warps of 128 registers, 12 of them consumers
constexpr int kFewStageBytes = 8192;  // K rows, then V rows
constexpr float kFewLead = 7.f;       // 8-bit: log2 of a row's largest P
constexpr float kFewEnough = 8.f;     // 8-bit: a row's sum of P times V's scale with which f16 loses nothing that shows

template <bool kFp8>
struct FewShape {
  static constexpr int kChunk = kFp8 ? 64 : 32;
  static constexpr uint32_t kScales = kFewStages * kFewStageBytes;
  static constexpr uint32_t kBars = kScales + (kFp8 ? kFewStages * 2 * kChunk : 0);
  static constexpr uint32_t kBytes = kBars + 256;
};

// The row within its 8 that fragment column c reads (8-bit): bits (c1 ^ c0, c0, c2).
__device__ __forceinline__ int few_place(int c) { return (((c >> 1) ^ c) & 1) | ((c & 1) << 1) | (c & 4); }

// Where, in 8-bit V rows, the thread of dims 8 g8 .. 8 g8 + 7 finds the position of column c.
__device__ __forceinline__ uint32_t few_v_at(int c, int g8) {
  const int r = few_place(c);
  return r * 64 + (((g8 >> 1) ^ ((r >> 1) & 3)) << 4) + (g8 & 1) * 8;
}

__device__ __forceinline__ void few_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void few_ldmatrix_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// c = a b + (first ? 0 : c)
template <bool kHalf>
__device__ __forceinline__ void few_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first = false) {
  const float z0 = first ? 0.f : c[0], z1 = first ? 0.f : c[1], z2 = first ? 0.f : c[2], z3 = first ? 0.f : c[3];
  if constexpr (kHalf) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
  }
}

// Two e4m3 codes (the low or the high half of w) as f16, exactly.
__device__ __forceinline__ uint32_t few_half2(uint32_t w, bool high) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(high ? w >> 16 : w)));
  return h;
}

// RT: eights of rows, 1 or 2
template <bool kFp8, int RT>
__global__ void __launch_bounds__((kFewWarps + 1) * 32, kFewCtas)
    tree_few_kernel(const __grid_constant__ TreeTmaParams tp) {
  using L = FewShape<kFp8>;
  constexpr int C = L::kChunk, R = 8 * RT;
  constexpr int X = RT;  // the tile's upper and lower eight rows, of 16
  const TreeParams& p = tp.p;
  const KVLayer& kv = p.kv;
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t smem[];
  const int g = blockIdx.y;
  int tile, split;
  tree_item(p, tile, split);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
  auto full = [&](int i) { return base + L::kBars + 8 * i; };
  auto empty = [&](int i) { return base + L::kBars + 64 + 8 * i; };
  volatile uint32_t* abort_word = reinterpret_cast<volatile uint32_t*>(smem + L::kBars + 128);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kFewStages; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full(i)), "r"(kFp8 ? 33 : 1) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty(i)) : "memory");
    }
    *abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int p0 = split * p.split_len;
  pdl_wait();
  const int b = tree_turn(p);
  // the producer's first page ids and the sequence's lengths are on their way together
  TreePages pages(kv, b, p0, warp == kFewWarps ? lane : 1 << 30, p.error);
  int row0, nodes, prefix;
  if (!tree_sequence(p, b, row0, nodes, prefix)) return;
  if (base & 1023) {
    atomicCAS(p.error, 0, 2);
    return;
  }
  const int trow0 = tile * R;
  const int trows = min(R, nodes * p.group - trow0);
  const int end = prefix + nodes;
  const int p1 = min(end, p0 + p.split_len);
  if (trows <= 0 || p0 >= p1) return;
  const int nchunks = (p1 - p0 + C - 1) / C;
  auto wait_all = [&](uint32_t bar, uint32_t parity) {
    return (bool)__all_sync(0xffffffffu, tree_wait(bar, parity, abort_word, p.error));
  };

  if (warp == kFewWarps) {
    // ---- producer
    const int ps = kv.ps, nbox = C / p.box, blks = C / ps, offs = C % ps;
    // the chunk's place, this lane's box's, and its four scales': lanes 0-15 K's, 16-31 V's
    TreePlace first(p0, ps), box(p0 + lane * p.box, ps), four(p0 + 4 * (lane & 15), ps);
    const uint32_t box_bytes = p.box * (kFp8 ? 64 : 128);
    const uint8_t* scale_pool = lane < 16 ? kv.k_scales : kv.v_scales;
    int issued = 0, st = 0, phase = 1;
    for (int j = 0; j < nchunks; ++j) {
      const int c0 = p0 + j * C;
      const int boxes = min(nbox, (p1 - c0 + p.box - 1) / p.box);
      pages.reach(first.blk);
      const int row = (pages.page(box.blk, lane < boxes) * kv.NKV + g) * ps + box.off;
      const bool scales = kFp8 && c0 + 4 * (lane & 15) < p1;
      const int64_t srow = kFp8 ? ((int64_t)pages.page(four.blk, scales) * kv.NKV + g) * ps + four.off : 0;
      if (j >= kFewStages && !wait_all(empty(st), phase)) break;
      const uint32_t kdst = base + st * kFewStageBytes, vdst = kdst + kFewStageBytes / 2;
      if (lane == 0)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full(st)),
                     "r"(2 * boxes * box_bytes)
                     : "memory");
      __syncwarp();
      if (lane < boxes) {
        tree_tma(kdst + lane * box_bytes, &tp.tm_k, full(st), row);
        tree_tma(vdst + lane * box_bytes, &tp.tm_v, full(st), row);
      }
      if (kFp8) {
        if (scales)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(base + L::kScales + st * 2 * C + 4 * lane),
                       "l"(scale_pool + srow)
                       : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full(st)) : "memory");
        four.advance(blks, offs, ps);
      }
      first.advance(blks, offs, ps);
      box.advance(blks, offs, ps);
      if (++st == kFewStages) {
        st = 0;
        phase ^= 1;
      }
      ++issued;
    }
    // every box issued lands before the CTA may exit (bounded)
    for (int j = max(0, issued - kFewStages); j < issued; ++j) tree_land(full(j % kFewStages), (j / kFewStages) & 1);
  } else {
    // ---- consumers. Fragment rows of thread (g8, t4): g8 and g8 + 8 of each 16.
    const int g8 = lane >> 2, t4 = lane & 3;
    const uint32_t pick0 = 0x0444u | (uint32_t)few_place(2 * t4 & 3) << 12, pick1 = 0x0444u | (uint32_t)(few_place((2 * t4 & 3) + 1) & 3) << 12;
    uint32_t qa[4][4] = {};
    float fac[2];  // scores in powers of two: times this (and, 8-bit, the K scale)
    const float c2 = p.scale * 1.4426950408889634f;
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const int r = x * 8 + g8, pr = trow0 + r;
      const bool real = r < trows;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(
          p.q + ((size_t)(row0 + (real ? pr >> p.group_log : 0)) * p.NQ + g * p.group + (pr & (p.group - 1))) * 64);
      if (!kFp8) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {  // dims 16 kk + 2 t4 (+ 1), and 8 more
          qa[kk][x] = real ? q[8 * kk + t4] : 0u;
          qa[kk][2 + x] = real ? q[8 * kk + 4 + t4] : 0u;
        }
        fac[x] = c2;
      } else {
        // dims 16 t4 + 4 kk (+ 1), and 2 more
        uint32_t w[8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = real ? q[8 * t4 + i] : 0u;
          top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest exponent becomes 14 (an infinity or NaN stays one; a row of zeros may take any factor)
        const int e = min(max((int)(top >> 7), 30), 254);  // biased
        const float f = __uint_as_float((uint32_t)(127 + 14 + 127 - e) << 23);
        fac[x] = fmaxf(c2 / f, 1.2e-38f);  // never 0: it meets masked scores of -inf
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t u = w[2 * kk + y];
            __half2 h = __floats2half2_rn(bf_lo(u) * f, bf_hi(u) * f);
            qa[kk][2 * y + x] = *reinterpret_cast<uint32_t*>(&h);
          }
        }
      }
    }
    constexpr float kLead = kFp8 ? kFewLead : 0.f;
    float m[2], l[2], o[8][4];  // m: P is 2^(score - m), the maximum's 2^kLead
    float mass[2] = {};         // 8-bit: this thread's share of a row's sum of P times V's scale, until all rows have
    bool enough = false;        // kFewEnough; it stays that unless a maximum or V's largest scale grows
    bool short_of = false;      // the last positions were not enough
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    // 8-bit: a row's unit of O is 2^(top_v - 127); before drafted positions the rows' are equal, and all_unit 1 / it
    int top_v[2] = {};
    float all_unit = e8m0_value(254);
    bool ok = true;
    // 8-bit: O in a unit 2^down as large; what falls out of fp32 is that far below a value that the row sees
    auto grow_unit = [&](int x, int down) {
      const float f = down <= 126 ? e8m0_value(127 - down) : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[i][2 * x] *= f;
        o[i][2 * x + 1] *= f;
      }
      mass[x] *= f;
      top_v[x] += down;
    };
    // this thread's places in 32 rows of a chunk
    const uint32_t k_at = kFp8 ? few_place(g8) * 64 + ((t4 ^ ((few_place(g8) >> 1) & 3)) << 4) : (lane & 7) * 128;
    const uint32_t v_at[2] = {few_v_at(2 * t4, g8), few_v_at(2 * t4 + 1, g8)};
    const int scale_at = (t4 >> 1) * 4;
    int st = warp, phase = 0;
    for (int j = warp; j < nchunks; j += kFewWarps) {
      ok = wait_all(full(st), phase);
      if (!ok) break;
      bool odd = false;  // 8-bit: the chunk has a scale byte whose float is not its power of two: 255 (NaN) or 0 (2^-127)
      if (kFp8) {
        // the scales of positions 2 lane and 2 lane + 1; what lies behind the end is nothing
        const uint8_t* sc = smem + L::kScales + st * 2 * C;
        const uint32_t k2 = reinterpret_cast<const uint16_t*>(sc)[lane], v2 = reinterpret_cast<const uint16_t*>(sc + C)[lane];
        const int v0 = v2 & 255, v1 = v2 >> 8, pos = p0 + j * C + 2 * lane;
        const bool whole = p0 + j * C + C <= prefix;
        uint32_t four = k2 | v2 << 16;
        if (!whole) four = pos + 1 < end ? four : pos < end ? (four & 0x00FF00FFu) | 0x7F007F00u : 0x7F7F7F7Fu;
        const uint32_t zero = (four - 0x01010101u) & ~four, ones = (~four - 0x01010101u) & four;  // a byte of 0, of 255
        odd = __any_sync(0xffffffffu, (zero | ones) & 0x80808080u);
        int most = max(v0, v1);  // of V's, those of committed positions that are numbers count
        if (!whole || odd)
          most = max(pos < prefix && v0 != kScaleNaN ? v0 : 0, pos + 1 < prefix && v1 != kScaleNaN ? v1 : 0);
        most = __reduce_max_sync(0xffffffffu, most);
        if (most > top_v[0]) {
#pragma unroll
          for (int x = 0; x < X; ++x) grow_unit(x, most - top_v[x]);
          all_unit = e8m0_value(254 - most);
          enough = false;
        }
      }
      // 32 positions; kPlain: all committed, every scale a number, P in f16's range (if it is
      // not: false, and nothing added)
      auto step = [&](auto plain, const int sub) {
        constexpr bool kPlain = decltype(plain)::value;
        const int c0 = p0 + j * C + sub * 32;
        const bool tail = !kPlain && c0 + 32 > prefix;
        const uint32_t kb = base + st * kFewStageBytes + sub * 32 * (kFp8 ? 64 : 128), vb = kb + kFewStageBytes / 2;
        const uint8_t* krow = smem + (kb - base);
        const uint8_t* sc = smem + L::kScales + st * 2 * C + sub * 32;  // K scales; V's are C further
        uint32_t vis[2], dead = 0;  // seen positions; positions without a finite V
        vis[0] = vis[1] = 0xffffffffu;
        if (tail) {
          const int pos = c0 + lane;
          bool bad = false;
          if (kFp8) {
            bad = sc[C + lane] == kScaleNaN;
          } else if (pos >= prefix && pos < end) {
            const uint4* v = reinterpret_cast<const uint4*>(smem + (vb - base) + lane * 128);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint4 u = v[c];
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                bad |= (w[e] & 0x7F800000u) == 0x7F800000u || (w[e] & 0x7F80u) == 0x7F80u;
            }
          }
          if (pos >= end || bad) {  // V becomes 0: a masked P of 0 must not meet a NaN
            uint4* v = reinterpret_cast<uint4*>(smem + (vb - base) + lane * (kFp8 ? 64 : 128));
#pragma unroll
            for (int c = 0; c < (kFp8 ? 4 : 8); ++c) v[c] = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          bad = bad && pos >= prefix && pos < end;
          const uint32_t poison = __ballot_sync(0xffffffffu, bad);
          dead = poison | __ballot_sync(0xffffffffu, pos >= end);
#pragma unroll
          for (int x = 0; x < X; ++x) {
            const int r = x * 8 + g8;
            vis[x] = 0;
            if (r < trows)
              vis[x] = (uint32_t)tree_bits(p.mask + (size_t)(row0 + ((trow0 + r) >> p.group_log)) * p.words, p.words,
                                               nodes, c0 - prefix);
            // a row that sees a V that is not finite has no finite result
            if (vis[x] & poison) l[x] = __uint_as_float(0x7FFFFFFFu);
          }
          __syncwarp();
        }
        // ---- scores: four blocks of 8 positions
        float s[4][4];
        float sv[4][2];  // 8-bit: V's scales of this thread's columns
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
          if (!kFp8) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              uint32_t kf[4];
              few_ldmatrix(kf, kb + k_at + nb * 1024 + (((hf * 4 + (lane >> 3)) ^ (lane & 7)) << 4));
#pragma unroll
              for (int u = 0; u < 2; ++u)
                few_mma<false>(s[nb], qa[hf * 2 + u], kf[2 * u], kf[2 * u + 1], hf == 0 && u == 0);
            }
          } else {
            const uint4 u = *reinterpret_cast<const uint4*>(krow + k_at + nb * 512);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint32_t b0 = few_half2(w[kk], false), b1 = few_half2(w[kk], true);
              few_mma<true>(s[nb], qa[kk], b0, b1, kk == 0);
            }
            // the scales of this thread's two columns, out of four neighbouring bytes
            const uint32_t ks = *reinterpret_cast<const uint32_t*>(sc + scale_at + nb * 8);
            const uint32_t vs = *reinterpret_cast<const uint32_t*>(sc + scale_at + C + nb * 8);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // the byte on top, then down by one: a float's exponent
              uint32_t kx = __byte_perm(ks, 0, e ? pick1 : pick0) >> 1, vx = __byte_perm(vs, 0, e ? pick1 : pick0) >> 1;
              if (!kPlain) {
                kx = max(kx, 0x00400000u);  // byte 0: 2^-127
                vx = max(vx, 0x00400000u);
              }
              float kf = __uint_as_float(kx), vf = __uint_as_float(vx);
              if (!kPlain && (tail || odd)) {
                if (kx == 0x7F800000u) kf = __uint_as_float(0x7FFFFFFFu);
                if (vx == 0x7F800000u) vf = __uint_as_float(0x7FFFFFFFu);
                if ((dead >> (nb * 8 + few_place(2 * t4 + e))) & 1) vf = 0.f;
              }
              sv[nb][e] = vf;
#pragma unroll
              for (int x = 0; x < X; ++x) s[nb][2 * x + e] *= kf;
            }
          }
        }
        if (tail) {
#pragma unroll
          for (int nb = 0; nb < 4; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int at = nb * 8 + (kFp8 ? few_place(2 * t4 + e) : 2 * t4 + e);
#pragma unroll
              for (int x = 0; x < X; ++x)
                if (!((vis[x] >> at) & 1)) s[nb][2 * x + e] = -INFINITY;
            }
          if (kFp8) {  // the largest scale of V that a row sees here
#pragma unroll
            for (int x = 0; x < X; ++x) {
              float t = 0.f;
#pragma unroll
              for (int nb = 0; nb < 4; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if ((vis[x] >> (nb * 8 + few_place(2 * t4 + e))) & 1) t = fmaxf(t, sv[nb][e]);  // not a NaN's
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
              const int most = (int)(__float_as_uint(t) >> 23);
              const bool more = most > top_v[x];
              if (more) grow_unit(x, most - top_v[x]);
              if (__any_sync(0xffffffffu, more)) enough = false;
            }
          }
        }
        float v_unit[2] = {all_unit, all_unit};
        if (kFp8 && tail) {
#pragma unroll
          for (int x = 0; x < X; ++x) v_unit[x] = e8m0_value(254 - top_v[x]);
        }
        // ---- maxima
        float mx[2];
        bool grow = false;
#pragma unroll
        for (int x = 0; x < X; ++x) {
          float t = -INFINITY;
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) t = tree_max3(t, s[nb][2 * x], s[nb][2 * x + 1]);
          mx[x] = t * fac[x];
          grow |= mx[x] > m[x] + (8.f + kLead);
        }
        if (__any_sync(0xffffffffu, grow)) {
          enough = false;
#pragma unroll
          for (int x = 0; x < X; ++x) {
            float t = mx[x];  // the row's four lanes agree
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            if (t > m[x] + (8.f + kLead)) {
              const float alpha = exp2_approx(m[x] - (t - kLead));  // 0 for the first maximum
              m[x] = t - kLead;
              l[x] *= alpha;
              mass[x] *= alpha;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                o[i][2 * x] *= alpha;
                o[i][2 * x + 1] *= alpha;
              }
            }
          }
        }
        // ---- probabilities, as the A fragments of P V
        uint32_t pa[2][4] = {};
        const float l_was[2] = {l[0], l[1]};
#pragma unroll
        for (int x = 0; x < X; ++x) {
          const float mu = m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) {
            float e0 = exp2_approx(fmaf(s[nb][2 * x], fac[x], -mu));
            float e1 = exp2_approx(fmaf(s[nb][2 * x + 1], fac[x], -mu));
            l[x] += e0 + e1;
            if (kFp8) {
              // V's scales in the row's unit: at most 1 where it sees the position
              float w0 = sv[nb][0] * v_unit[x], w1 = sv[nb][1] * v_unit[x];
              if (tail) {
                w0 = w0 > 1.f ? 1.f : w0;  // (a NaN stays)
                w1 = w1 > 1.f ? 1.f : w1;
              }
              s[nb][2 * x] = e0 * w0;
              s[nb][2 * x + 1] = e1 * w1;
            } else {
              __nv_bfloat162 h = __floats2bfloat162_rn(e0, e1);
              pa[nb >> 1][(nb & 1) * 2 + x] = *reinterpret_cast<uint32_t*>(&h);
            }
          }
        }
        bool wide = false;  // 8-bit: P needs bf16's range
        if (kFp8) {
          if (!enough) {
            bool little = false;
            float with[2];
#pragma unroll
            for (int x = 0; x < X; ++x) {
              with[x] = mass[x];
#pragma unroll
              for (int nb = 0; nb < 4; ++nb) with[x] += s[nb][2 * x] + s[nb][2 * x + 1];
              float w = with[x];
              w += __shfl_xor_sync(0xffffffffu, w, 1);
              w += __shfl_xor_sync(0xffffffffu, w, 2);
              little |= w < kFewEnough && m[x] > -INFINITY;
            }
            wide = __any_sync(0xffffffffu, little);
            enough = !wide;
            if (kPlain && wide) {
#pragma unroll
              for (int x = 0; x < X; ++x) l[x] = l_was[x];
              return false;
            }
#pragma unroll
            for (int x = 0; x < X; ++x) mass[x] = with[x];
          }
#pragma unroll
          for (int x = 0; x < X; ++x)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) {
              uint32_t& a = pa[nb >> 1][(nb & 1) * 2 + x];
              if (!kPlain && wide) {
                // 2^60 from V to P: P may be as small as V's scales lie apart
                __nv_bfloat162 h = __floats2bfloat162_rn(s[nb][2 * x] * 0x1p60f, s[nb][2 * x + 1] * 0x1p60f);
                a = *reinterpret_cast<uint32_t*>(&h);
              } else {
                __half2 h = __floats2half2_rn(s[nb][2 * x], s[nb][2 * x + 1]);
                a = *reinterpret_cast<uint32_t*>(&h);
              }
            }
        }
        // ---- P . V: two steps of 16 positions, eight blocks of 8 dims
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          if (!kFp8) {
#pragma unroll
            for (int dp = 0; dp < 4; ++dp) {
              uint32_t vf[4];
              const int r = ks * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), c = dp * 2 + (lane >> 4);
              few_ldmatrix_t(vf, vb + r * 128 + ((c ^ (r & 7)) << 4));
#pragma unroll
              for (int u = 0; u < 2; ++u)
                few_mma<false>(o[dp * 2 + u], pa[ks], vf[2 * u], vf[2 * u + 1]);
            }
          } else {
            uint2 v[2][2];  // [8 positions][column e]: dims 8 g8 .. 8 g8 + 7 of a position
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                v[q][e] = *reinterpret_cast<const uint2*>(krow + kFewStageBytes / 2 + v_at[e] + (ks * 16 + q * 8) * 64);
              }
            if (kPlain || !wide) {
#pragma unroll
              for (int d = 0; d < 8; d += 2) {
                uint32_t bf[2][2];  // [dim][8 positions]
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  const uint32_t lo = d < 4 ? v[q][0].x : v[q][0].y, hi = d < 4 ? v[q][1].x : v[q][1].y;
                  const uint32_t w = __byte_perm(lo, hi, (d & 2) ? 0x7362 : 0x5140);
                  bf[0][q] = few_half2(w, false);
                  bf[1][q] = few_half2(w, true);
                }
                few_mma<true>(o[d], pa[ks], bf[0][0], bf[0][1]);
                few_mma<true>(o[d + 1], pa[ks], bf[1][0], bf[1][1]);
              }
            } else {
              const __nv_bfloat162 f = tree_pow2(247 - 60);  // 2^120 of the code, 2^-60
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                uint32_t bf[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  const uint32_t lo = d < 4 ? v[q][0].x : v[q][0].y, hi = d < 4 ? v[q][1].x : v[q][1].y;
                  const uint32_t w = __byte_perm(lo, hi, (d & 3) << 4 | (4 + (d & 3)) << 12);
                  const uint32_t z = ((w >> 4) & 0x07F007F0u) | (w & 0x80008000u);
                  const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&z), f);
                  bf[q] = *reinterpret_cast<const uint32_t*>(&y);
                }
                few_mma<false>(o[d], pa[ks], bf[0], bf[1]);
              }
            }
          }
        }
        return true;
      };
#pragma unroll 1
      for (int sub = 0; sub < C / 32; ++sub) {
        const int c0 = p0 + j * C + sub * 32;
        if (c0 >= p1) break;
        // where the last one was short of mass this one is likely to be, so it is not tried in f16
        if (c0 + 32 > prefix || odd || (kFp8 && short_of) || !step(std::true_type{}, sub)) {
          step(std::false_type{}, sub);
          short_of = !enough;
        }
      }
      __syncwarp();
      if (lane == 0) tree_arrive(empty(st));
      st += kFewWarps;
      if (st >= kFewStages) {
        st -= kFewStages;
        phase ^= 1;
      }
    }

    // ---- the three warps joined; their states lie over the ring, which nobody reads any more
    float* state = reinterpret_cast<float*>(smem);  // [warp][R][kTreePartial]
    const float lead = kFp8 ? exp2f(-kLead) : 1.f;
    asm volatile("bar.sync 1, %0;" ::"n"(kFewWarps * 32) : "memory");
#pragma unroll
    for (int x = 0; x < X; ++x) {
      float t = l[x] * lead;
      t += __shfl_xor_sync(0xffffffffu, t, 1);
      t += __shfl_xor_sync(0xffffffffu, t, 2);
      const float unit = kFp8 ? e8m0_value(top_v[x]) * lead : 1.f;
      float* d = state + (warp * R + x * 8 + g8) * kTreePartial;
      if (t4 == 0) *reinterpret_cast<float2*>(d + 64) = make_float2(m[x] + kLead, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!kFp8) {  // dims 8 i + 2 t4 (+ 1)
          *reinterpret_cast<float2*>(d + 8 * i + 2 * t4) = make_float2(o[i][2 * x], o[i][2 * x + 1]);
        } else {  // in units of V's largest scale; dims 16 t4 + i and 8 more
          d[16 * t4 + i] = o[i][2 * x] * unit;
          d[16 * t4 + 8 + i] = o[i][2 * x + 1] * unit;
        }
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kFewWarps * 32) : "memory");
    float* joined = state + kFewWarps * R * kTreePartial;  // in a cluster: [R], for its other CTAs
    static_assert((kFewWarps + 1) * R * kTreePartial * 4 <= kFewStages * kFewStageBytes, "the states fit over the ring");
    const int lane16 = lane & 15;
    for (int r = 2 * warp + (lane >> 4); ok && r < trows; r += 2 * kFewWarps) {
      TreeRow t;
      t.add(kFewWarps, [&](int w, float2& ml, float4& v) {
        const float* d = state + (w * R + r) * kTreePartial;
        ml = *reinterpret_cast<const float2*>(d + 64);
        v = *reinterpret_cast<const float4*>(d + 4 * lane16);
      });
      const int pr = trow0 + r;
      if (p.splits > 1) {
        float* dst = p.cluster ? joined + r * kTreePartial
                               : p.work + ((((size_t)b * kv.NKV + g) * p.splits + split) * p.max_nodes * p.group + pr) * kTreePartial;
        if (lane16 == 0) *reinterpret_cast<float2*>(dst + 64) = make_float2(t.m, t.l);
        *reinterpret_cast<float4*>(dst + 4 * lane16) = t.o;
      } else {
        t.write(p, row0 + (pr >> p.group_log), g * p.group + (pr & (p.group - 1)), lane16);
      }
    }
  }
  if (p.cluster) {
    tree_cluster_sync();
    tree_join(p, base + kFewWarps * R * kTreePartial * 4, (end + p.split_len - 1) / p.split_len, split, warp, kFewWarps + 1, lane,
              row0, trow0, trows, g);
  }
}

}  // namespace mk
