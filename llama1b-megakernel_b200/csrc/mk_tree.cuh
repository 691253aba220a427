// Attention of drafted tokens over a paged cache, on the tcgen05 tensor cores.
//
// Sequence b has prefix_b committed positions in its pages and, behind them, n_b
// drafted nodes whose K/V rows sit at positions prefix_b + j. Node i sees every
// committed position and those nodes j whose bit (i, j) is set (itself and its
// ancestors in a tree; j <= i for a chunk of a prompt):
//   s_j = scale q_i . k_j,  p_j = exp(s_j - m),  o = sum p_j v_j / sum p_j,
//   lse = m + log sum p_j,  m >= max_j s_j - 8 log 2,
// per query head, the sums in fp32. A row that sees nothing gets o = 0 and
// lse = -inf.
//
// The query heads of a K/V head share its rows, so the nodes of a sequence and
// those heads (row = node * group + head) are the rows of one matrix product, in
// tiles of 128. A CTA takes a tile, a K/V head and a range of positions, 128 at a
// time (a block):
//  * a producer warp brings the block's K and V rows in by TMA (boxes of the
//    largest power of two, at most 128, that divides the page size, so a box never
//    leaves its page) into a ring of stages;
//  * a warpgroup makes the block fit for the tensor cores. bf16: it only acts on
//    blocks that reach past the committed positions: V rows behind the last node
//    become zeros, and so do drafted V rows that hold an infinity or NaN (0 * inf
//    in P V would reach rows that do not see them), which are noted in a bit mask.
//    8-bit: it turns codes into bf16 rows of the value code * 2^e, exactly (see
//    tree_decode), and treats the last block's V in the same way;
//  * one thread issues S = Q K^T (M 128, N 64, 64 dims) for half a block and O += P V
//    (N 64, 64 positions) with P read from TMEM and V taken MN-major as it lies;
//  * two warpgroups do the softmax, one the first halves of the blocks and one the
//    second, each with its own S, maximum, sum and O, which are joined at the end: a
//    row's thread spends as long on waits, loads and bookkeeping as on its 64
//    exponentials, so four warps (two CTAs) on each scheduler keep the special
//    function unit busy where two did not (4 sequences of 256 nodes at 16,000: 235 us
//    with one softmax warpgroup, 211 with two). A thread
//    has a row (TMEM lane): the 64 scores, the exponentials, P as bf16 pairs over S.
//    O is only rescaled when a row's maximum has grown by more than 8 powers of two
//    since it was last set: until then p is at most 256, which costs bf16 and fp32
//    nothing.
// P is rounded to bf16 (relative 2^-8 at most, unbiased, as V is no more precise
// itself); its sum is taken before the rounding. The ranges of a sequence that is
// split into at most eight are one thread-block cluster, whose CTAs leave (m, l, O)
// in shared memory and join them there, a share of the rows each (tree_join); more
// ranges go through the workspace and tree_merge_kernel.
//
// What bounds it: a lone CTA takes 5.1 us and 1.1 us a block, the latency of the chain S,
// softmax, P V; two on an SM 1.8 us a block each, 16,384 exponentials at 16 a cycle being
// 0.55 us of it apiece. 4 sequences of 256 nodes behind 11,000 to 16,000 positions: 181 to
// 197 us (two GPUs), 610 to 660 TFLOP/s; 32 of 64 nodes over 5,200 to 8,200 8-bit positions: 205 us, 543 TFLOP/s, bound by
// instructions (a block warp issues 425 for a block's conversion beside the softmax's
// 271 a half block).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "mk_device.cuh"
#include "mk_kv8.cuh"

namespace mk {

constexpr int kTreeMaxNodes = 256;
constexpr int kTreeRows = 128;     // rows of a tile (the MMA's M)
constexpr int kTreeBlock = 128;    // positions of a block
constexpr int kTreeHalf = 64;      // of a step of the softmax
constexpr int kTreeThreads = 448;  // 2 x 4 softmax warps, 4 block warps, producer, issuer
constexpr int kTreePartial = 68;   // o[64], m, l, two to align
constexpr int kTreeCluster = 8;    // ranges that may join in a cluster: the portable size
constexpr uint32_t kTreeTmem = 256;  // columns: S (and P over it) 2 x 64, O 2 x 64
constexpr uint32_t kTreeTileBytes = kTreeBlock * 128;  // a bf16 K or V block (and the Q tile)
constexpr uint32_t kTreeRawBytes = kTreeBlock * 64;    // an 8-bit one

template <bool kFp8>
struct TreeSmem {
  static constexpr int kStages = kFp8 ? 2 : 3;   // blocks in flight from memory
  static constexpr int kReady = kFp8 ? 2 : 3;    // blocks ready for the tensor cores
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kTiles = kTreeTileBytes;                        // kReady x (K, V) bf16
  static constexpr uint32_t kRaw = kTiles + kReady * 2 * kTreeTileBytes;    // 8-bit: kStages x (K, V)
  static constexpr uint32_t kScales = kRaw + (kFp8 ? kStages * 2 * kTreeRawBytes : 0);  // kStages x 256
  static constexpr uint32_t kBars = kScales + (kFp8 ? kStages * 2 * kTreeBlock : 0);
  static constexpr uint32_t kBytes = kBars + 256;   // the (m, l) of the second softmax lie over Q at the end
};

struct TreeParams {
  const __nv_bfloat16* q;           // [rows][NQ][64]
  KVLayer kv;
  const int* cu_nodes;              // [batch + 1]
  const unsigned long long* mask;   // [rows][words]
  const int* prefix;                // [batch]
  int rows, words, max_nodes, max_len, NQ;
  int group, group_log;             // query heads of a K/V head: 1, 2, 4 or 8
  int box;                          // rows of a TMA box
  int tiles, splits, split_len;     // split_len: a multiple of kTreeBlock
  int cluster;                      // the ranges of a tile are a cluster (else: partials in work)
  int sorted;                       // long sequences first (tree_turn): 1 + log2 of a bucket's positions; 0: as they come
  float scale;
  float* work;                      // [batch][NKV][splits][max_nodes * group][kTreePartial]
  __nv_bfloat16* out;               // [rows][NQ][64]
  float* lse;                       // [rows][NQ] or null
  int* error;
};

struct alignas(64) TreeTmaParams {
  CUtensorMap tm_k;  // the pool as rows of 64 values
  CUtensorMap tm_v;
  TreeParams p;
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

__device__ __forceinline__ uint32_t tree_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}

// Wait with a limit: 2 s and a thousand looks, so that neither a pause of the whole
// GPU nor a timer that steps back is taken for a wait that ran out. One that did reports error 2 and raises the
// CTA's abort word, on which every other wait of the CTA gives up. The waiting is
// kept out of the roles' loops, which have to stay in the instruction cache.
__device__ __noinline__ bool tree_wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* abort_word, int* error) {
  uint64_t t0 = 0;
  for (uint32_t looks = 0;; ++looks) {
    // asleep until the phase ends, 1 ms at most: warps that poll take issue slots from the softmax
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2, 1000000;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if (*abort_word) return false;
    const uint64_t now = global_ns();
    if (!t0) {
      t0 = now;
    } else if (looks >= 1000 && (int64_t)(now - t0) > 2000000000ll) {
      *abort_word = 1;
      atomicCAS(error, 0, 2);
      return false;
    }
  }
}

__device__ __forceinline__ bool tree_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_word, int* error) {
  return tree_try(bar, parity) || tree_wait_slow(bar, parity, abort_word, error);
}

// Until a phase that nothing holds up any more has ended: copies and MMAs under way finish
// before the CTA gives up its memory, also where its other waits have run out. 4 s and a
// thousand looks, as above.
__device__ __noinline__ void tree_land(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = global_ns();
  for (uint32_t looks = 0; !tree_try(bar, parity); ++looks)
    if (looks >= 1000 && (int64_t)(global_ns() - t0) > 4000000000ll) return;
}

// The pages of a range as a producer warp walks through it: 32 entries of the block
// table in a register of each lane and the next 32 on their way, so that no copy
// waits for a load, and no division a position (with both, an iteration of the
// producer took 2,100 cycles, and the copies were what the kernel waited for).
struct TreePages {
  const int* table;
  int count, ps, num_pages, base, cur, nxt, lane;
  int* error;
  __device__ __forceinline__ int window(int w) const { return lane < count - w ? table[w + lane] : 0; }
  // sequence b from position p0 on; its length need not be known yet
  __device__ __forceinline__ TreePages(const KVLayer& kv, int b, int p0, int lane_, int* error_)
      : table(kv.block_tables + (size_t)b * kv.max_blocks), count(kv.max_blocks), ps(kv.ps), num_pages(kv.num_pages),
        base(p0 / kv.ps), lane(lane_), error(error_) {
    cur = window(base);
    nxt = window(base + 32);
  }
  // The page of block blk (at most 63 past the window's first), all lanes together;
  // an id outside the pool is reported and taken as page 0.
  __device__ __forceinline__ int page(int blk, bool used) const {
    const int i = blk - base;
    const int a = __shfl_sync(0xffffffffu, cur, i & 31), b = __shfl_sync(0xffffffffu, nxt, i & 31);
    int id = i < 32 ? a : b;
    if (used && (id < 0 || id >= num_pages)) {
      atomicExch(error, 1);
      id = 0;
    }
    return id;
  }
  // The walk has come to block blk.
  __device__ __forceinline__ void reach(int blk) {
    if (blk - base >= 32) {
      base += 32;
      cur = nxt;
      nxt = window(base + 32);
    }
  }
};

// A place in the sequence: block and offset, moved on by a fixed number of positions.
struct TreePlace {
  int blk, off;
  __device__ __forceinline__ TreePlace(int pos, int ps) : blk(pos / ps), off(pos % ps) {}
  __device__ __forceinline__ void advance(int blks, int offs, int ps) {
    blk += blks;
    off += offs;
    if (off >= ps) {
      off -= ps;
      ++blk;
    }
  }
};

__device__ __forceinline__ void tree_tma(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(tm), "r"(bar), "r"(0), "r"(row)
      : "memory");
}

__device__ __forceinline__ void tree_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The issuing warp runs converged and lets elect.sync pick the thread: descriptors
// and addresses stay uniform over the warp. (Inside `if (lane == 0)` every MMA cost
// about 100 cycles of moves into uniform registers, and the four of a product more
// than the softmax of a half block.)
__device__ __forceinline__ void tree_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}

// D = A B, four steps of 16 along K, A and B K-major in shared memory (a step is 32 bytes).
__device__ __forceinline__ void tree_mma_scores(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred q, no, yes;\n\t"
      ".reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 no, 0, 0;\n\t"
      "setp.eq.b32 yes, 0, 0;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, no;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, yes;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, yes;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, yes;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc)
      : "memory");
}

// D (+)= A B, four steps of 16 along K, A in TMEM (a step is 8 columns), B MN-major
// in shared memory (a step is 16 rows of 128 bytes).
__device__ __forceinline__ void tree_mma_values(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred q, first, yes;\n\t"
      ".reg .b64 b1, b2, b3;\n\t"
      ".reg .b32 a1, a2, a3;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 first, %4, 0;\n\t"
      "setp.eq.b32 yes, 0, 0;\n\t"
      "add.s32 a1, %1, 8;\n\tadd.s32 a2, %1, 16;\n\tadd.s32 a3, %1, 24;\n\t"
      "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, first;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, yes;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, yes;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, yes;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}

// A 128-byte-swizzled operand of 128-byte rows, groups of 8 rows 1024 bytes apart:
// K-major for Q and K (the rows are M or N), MN-major for V (the rows are K).
__device__ __forceinline__ uint64_t tree_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// fp32 accumulator, bf16 operands, M 128, N n; trans_b: B is MN-major.
__device__ __forceinline__ constexpr uint32_t tree_idesc(int n, bool trans_b) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((trans_b ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTreeRows >> 4) << 24);
}

// 32 columns of the thread's TMEM lane.
__device__ __forceinline__ void tree_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float tree_max3(float a, float b, float c) {  // NaN is nobody's largest
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of two numbers on the FMA pipe, for some of a row's: the special function unit
// (16 exponentials a cycle) is what bounds the softmax of bf16 rows. x = n + f, |f| <= 1/2, and a polynomial for 2^f (least largest relative error, fitted by
// reweighted least squares: 2^-22.1 in fp32, as good as ex2.approx); n goes into the
// exponent by a multiplication, which keeps a NaN. Below 2^-126.5 the result is 0 (an
// exponent field of 0 for n = -127), as a value of 3e38 may go with it. 4 sequences of 256 nodes at 16,000: none 199 us, 2 of 16
// 184, 3 of 16 181, 4 of 16 183, 5 of 16 195; with 8-bit rows, whose conversion takes the issue slots,
// 32 x 64 nodes: none 223 us, 2 of 16 235.
__device__ __forceinline__ float2 tree_exp2(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));  // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
  auto both = [](float c) { return make_float2(c, c); };
  const float2 t = add2(x, both(12583039.f));  // 1.5 * 2^23 + 127: n, biased, in the low bits
  const float2 f = fma2(add2(t, both(-12583039.f)), both(-1.f), x);
  float2 q = fma2(f, both(0.0013276466634124517f), both(0.009675540961325169f));
  q = fma2(q, f, both(0.05550713464617729f));
  q = fma2(q, f, both(0.24022120237350464f));
  q = fma2(q, f, both(0.6931469440460205f));
  q = fma2(q, f, both(1.0000001192092896f));
  return mul2(q, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}

__device__ __forceinline__ void tree_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tree_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// Four e4m3 codes as bf16: {d0, d2} and {d1, d3}. A code s eeee mmm moved into
// bf16's place for (exponent, mantissa) is its value times 2^(7 - 127), its
// subnormals becoming bf16's, so one exact multiplication by 2^120 and the row's
// scale (`f`, in both halves) gives the value.
__device__ __forceinline__ uint2 tree_decode(uint32_t w, __nv_bfloat162 f) {
  uint32_t a = ((w << 4) & 0x07F007F0u) | ((w << 8) & 0x80008000u);
  uint32_t b = ((w >> 4) & 0x07F007F0u) | (w & 0x80008000u);
  __nv_bfloat162 x = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), f);
  __nv_bfloat162 y = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&b), f);
  return make_uint2(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y));
}

__device__ __forceinline__ __nv_bfloat162 tree_pow2(int biased) {  // 2^(biased - 127) twice
  const uint32_t w = (uint32_t)biased << 7;
  const uint32_t ww = w | (w << 16);
  return *reinterpret_cast<const __nv_bfloat162*>(&ww);
}

__device__ __forceinline__ __nv_bfloat162 tree_nan2() {
  const uint32_t w = 0x7FC07FC0u;
  return *reinterpret_cast<const __nv_bfloat162*>(&w);
}

// 64 bits of row `mask` from bit j0 on (j0 may be negative: committed positions, all seen).
__device__ __noinline__ unsigned long long tree_bits(const unsigned long long* mask, int words, int nodes, int j0) {
  auto word = [&](int w) -> unsigned long long {
    if (w < 0) return ~0ull;
    if (w >= words || 64 * w >= nodes) return 0;
    const int left = nodes - 64 * w;
    return mask[w] & (left >= 64 ? ~0ull : (1ull << left) - 1);
  };
  const int w = j0 >> 6, sh = j0 & 63;
  const unsigned long long lo = word(w);
  return sh ? (lo >> sh) | (word(w + 1) << (64 - sh)) : lo;
}

// The CTA's row tile and range.
__device__ __forceinline__ void tree_item(const TreeParams& p, int& tile, int& split) {
  if (p.cluster) {  // a tile's ranges side by side
    split = blockIdx.x % p.splits;
    tile = blockIdx.x / p.splits;
  } else {          // the tiles that read the same positions side by side
    tile = blockIdx.x % p.tiles;
    split = blockIdx.x / p.tiles;
  }
}

// The CTA's sequence: as they come, or the longer ones first, by buckets of their
// committed positions (at most 32 buckets; within one as they come). Every warp finds out
// by itself: lane k counts bucket 31 - k, a scan gives the bucket of this CTA's turn, and
// the turn within it is a set bit of the ballots.
__device__ __forceinline__ int tree_turn(const TreeParams& p) {
  const int turn = blockIdx.z;
  if (!p.sorted) return turn;
  const int lane = threadIdx.x & 31, batch = p.kv.batch;
  // the place of sequence b's bucket in the order, 32 for none
  auto bucket = [&](int b) { return b < batch ? 31 - min(max(p.prefix[b], 0) >> (p.sorted - 1), 31) : 32; };
  int count = 0;
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const int k = bucket(b0 + lane);
    uint32_t same = __ballot_sync(0xffffffffu, k < 32);  // the lanes whose k is this lane's number
#pragma unroll
    for (int bit = 0; bit < 5; ++bit) {
      const uint32_t set = __ballot_sync(0xffffffffu, (k >> bit) & 1);
      same &= (lane >> bit) & 1 ? set : ~set;
    }
    count += __popc(same);
  }
  int upto = count;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  const int mine = __ffs(__ballot_sync(0xffffffffu, upto > turn)) - 1;
  int left = turn - __shfl_sync(0xffffffffu, upto - count, mine);
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const bool in = bucket(b0 + lane) == mine;
    const uint32_t there = __ballot_sync(0xffffffffu, in);
    const uint32_t hit = __ballot_sync(0xffffffffu, in && __popc(there & ((1u << lane) - 1)) == left);
    if (hit) return b0 + __ffs(hit) - 1;
    left -= __popc(there);
  }
  return 0;  // not reached: the buckets hold `batch` sequences
}

// lse of a row out of its maximum, in powers of two, and sum (not 0); lg2.approx is
// within 2^-22 of 1 or of the logarithm.
__device__ __forceinline__ float tree_lse(float m, float sum) {
  float lg;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(sum));
  return ((m == -INFINITY ? 0.f : m) + lg) * 0.6931471805599453f;
}
__device__ __forceinline__ float tree_inverse(float sum) {  // within an ulp
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(sum));
  return y;
}

// A row's partials joined, four dims a lane (16 lanes a row), four partials at a time so
// that all their loads are on their way before the first is used. (One lane group at a
// time, in a loop of dependent loads, with divisions: 1,400 cycles a row and warp.)
struct TreeRow {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  // load(q, ml, v): partial q's (m, l) and this lane's dims
  template <typename Load>
  __device__ __forceinline__ void add(int n, Load load) {
    for (int q0 = 0; q0 < n; q0 += 4) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        ml[q] = make_float2(-INFINITY, 0.f);
        v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (q0 + q < n) load(q0 + q, ml[q], v[q]);
      }
      const float top = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
      const float mu = top == -INFINITY ? 0.f : top, was = exp2_approx(m - mu);
      m = top;
      l *= was;
      o = make_float4(o.x * was, o.y * was, o.z * was, o.w * was);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float f = exp2_approx(ml[q].x - mu);
        l = fmaf(ml[q].y, f, l);
        o = make_float4(fmaf(v[q].x, f, o.x), fmaf(v[q].y, f, o.y), fmaf(v[q].z, f, o.z), fmaf(v[q].w, f, o.w));
      }
    }
  }
  __device__ __forceinline__ void write(const TreeParams& p, int row, int head, int lane16) const {
    const bool any = l != 0.f;  // NaN counts as something
    const float f = any ? tree_inverse(l) : 0.f;
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(any ? o.x * f : 0.f, any ? o.y * f : 0.f),
                           __floats2bfloat162_rn(any ? o.z * f : 0.f, any ? o.w * f : 0.f)};
    *reinterpret_cast<uint2*>(p.out + ((size_t)row * p.NQ + head) * 64 + 4 * lane16) =
        make_uint2(*reinterpret_cast<uint32_t*>(&h[0]), *reinterpret_cast<uint32_t*>(&h[1]));
    if (p.lse && lane16 == 0) p.lse[(size_t)row * p.NQ + head] = any ? tree_lse(m, l) : -INFINITY;
  }
};

__device__ __forceinline__ void tree_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Join the ranges of a cluster, after tree_cluster_sync: every CTA with a range has its
// partials [rows][kTreePartial] at shared address `part` (the same in each) and writes a
// share of the rows, its first `warps` warps two at a time. All threads of these CTAs
// pass the barriers; a CTA without a range has left, as they wait for threads that have
// not exited only (kept to the end, such CTAs took the slots of others: 17.4 us for 8
// sequences of 25 nodes behind 0 to 1,111 positions, 15.5 so).
__device__ __forceinline__ void tree_join(const TreeParams& p, uint32_t part, int ranges, int split, int warp, int warps,
                                          int lane, int row0, int trow0, int trows, int g) {
  const int lane16 = lane & 15;
  for (int r = warp < warps ? 2 * (split * warps + warp) + (lane >> 4) : trows; r < trows; r += 2 * ranges * warps) {
    TreeRow t;
    t.add(ranges, [&](int q, float2& ml, float4& v) {
      uint32_t a;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(part + r * kTreePartial * 4), "r"(q));
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(a + 256));
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                   : "r"(a + 16 * lane16));
    });
    const int pr = trow0 + r;
    t.write(p, row0 + (pr >> p.group_log), g * p.group + (pr & (p.group - 1)), lane16);
  }
  tree_cluster_sync();  // nobody leaves while another may still read its partials
}

template <bool kFp8>
__global__ void __launch_bounds__(kTreeThreads, 2) tree_attn_kernel(const __grid_constant__ TreeTmaParams tp) {
  using L = TreeSmem<kFp8>;
  const TreeParams& p = tp.p;
  const KVLayer& kv = p.kv;
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t smem[];
  const int g = blockIdx.y;
  int tile, split;
  tree_item(p, tile, split);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
  // barriers: full[3], empty[3], ready[3], free[3], -, s[2], p[2], o; then words
  const uint32_t bars = base + L::kBars;
  auto full = [&](int i) { return bars + 8 * i; };
  auto empty = [&](int i) { return bars + 24 + 8 * i; };
  auto ready = [&](int i) { return bars + 48 + 8 * i; };
  auto free_ = [&](int i) { return bars + 72 + 8 * i; };
  const uint32_t b_o = bars + 136;                             // all O are complete
  // of the first and second halves of the blocks, a phase per block
  auto b_s = [&](int half) { return bars + 104 + 8 * half; };  // S is in TMEM (and O has the block before)
  auto b_p = [&](int half) { return bars + 120 + 8 * half; };  // P is in TMEM
  volatile uint32_t* words = reinterpret_cast<volatile uint32_t*>(smem + L::kBars + 144);
  volatile uint32_t* abort_word = words;      // words[1]: TMEM base
  volatile uint32_t* bad = words + 4;         // [kReady][4] drafted positions whose V is not finite

  auto init = [](uint32_t bar, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory");
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) {
      init(full(i), kFp8 ? 33 : 1);   // the expected bytes; each producer lane's scale bytes
      init(empty(i), kFp8 ? 4 : 1);   // the block warps have read the codes; P V has read the rows
      init(ready(i), 4);
      init(free_(i), 1);
    }
    init(b_s(0), 1);
    init(b_s(1), 1);
    init(b_o, 1);
    *abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();  // the producer and the block warps need no other
  const int p0 = split * p.split_len;
  pdl_wait();
  const int b = tree_turn(p);
  // the producer's first page ids and the sequence's lengths are on their way together
  TreePages pages(kv, b, p0, warp == 12 ? lane : 1 << 30, p.error);
  int row0, nodes, prefix;
  if (!tree_sequence(p, b, row0, nodes, prefix)) return;
  if (base & 1023) {  // the swizzled layouts count on it
    atomicCAS(p.error, 0, 2);
    return;
  }
  const int trow0 = tile * kTreeRows;  // first row (node * group + head) of the tile
  const int trows = min(kTreeRows, nodes * p.group - trow0);
  const int end = prefix + nodes;
  const int p1 = min(end, p0 + p.split_len);
  if (trows <= 0 || p0 >= p1) return;
  if (warp == 13) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::kBars + 148),
                 "r"(kTreeTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int nblocks = (p1 - p0 + kTreeBlock - 1) / kTreeBlock;
  const int halves = (p1 - p0 + kTreeHalf - 1) / kTreeHalf;
  const int active = (trows + 31) >> 5;  // softmax warps with a row
  if (threadIdx.x == 0) {
    init(b_p(0), active);
    init(b_p(1), active);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // while the first copies are under way, the softmax warps bring Q in, 16 rows each
  // and eight lanes a row (a row a lane is 32 cache lines a load: 1,000 cycles more)
  if (warp < 8) {
    uint4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = trow0 + warp * 16 + i * 4 + (lane >> 3);
      u[i] = make_uint4(0, 0, 0, 0);
      if (at < trow0 + trows)
        u[i] = reinterpret_cast<const uint4*>(
            p.q + ((size_t)(row0 + (at >> p.group_log)) * p.NQ + g * p.group + (at & (p.group - 1))) * 64)[lane & 7];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = warp * 16 + i * 4 + (lane >> 3);
      if (kFp8)  // the order of dims that tree_decode leaves: 0, 2, 1, 3
        u[i] = make_uint4(__byte_perm(u[i].x, u[i].y, 0x5410), __byte_perm(u[i].x, u[i].y, 0x7632),
                          __byte_perm(u[i].z, u[i].w, 0x5410), __byte_perm(u[i].z, u[i].w, 0x7632));
      *reinterpret_cast<uint4*>(smem + L::kQ + at * 128 + (((lane & 7) ^ (at & 7)) << 4)) = u[i];
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp < 8 || warp == 13) {  // Q, TMEM and the barriers of P are there
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("bar.sync 2, 288;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  const uint32_t tmem = words[1];
  // of the first and second halves of the blocks
  auto t_s = [&](int half) { return tmem + 64 * half; };  // P lies over the first 32 columns of S
  auto t_o = [&](int half) { return tmem + 128 + 64 * half; };
  auto slot_at = [&](int slot) { return base + L::kTiles + slot * 2 * kTreeTileBytes; };
  // the whole warp: the same answer in every lane, and all of them there again
  auto wait_all = [&](uint32_t bar, uint32_t parity) {
    return (bool)__all_sync(0xffffffffu, tree_wait(bar, parity, abort_word, p.error));
  };

  if (warp == 12) {
    // ---- producer
    const int ps = kv.ps, nbox = kTreeBlock / p.box, blks = kTreeBlock / ps, offs = kTreeBlock % ps;
    TreePlace first(p0, ps), box(p0 + lane * p.box, ps), four(p0 + 4 * lane, ps);  // the block's, this lane's box's, its four scales'
    const uint32_t box_bytes = p.box * (kFp8 ? 64 : 128);
    int issued = 0, st = 0, phase = 1;
    for (int j = 0; j < nblocks; ++j) {
      const int c0 = p0 + j * kTreeBlock;
      const int boxes = min(nbox, (p1 - c0 + p.box - 1) / p.box);
      pages.reach(first.blk);
      const int row = (pages.page(box.blk, lane < boxes) * kv.NKV + g) * ps + box.off;
      const bool scales = kFp8 && c0 + 4 * lane < p1;  // the page size is a multiple of 8: four scale bytes lie together
      const int64_t srow = kFp8 ? ((int64_t)pages.page(four.blk, scales) * kv.NKV + g) * ps + four.off : 0;
      if (j >= L::kStages && !wait_all(empty(st), phase)) break;
      const uint32_t kdst = base + (kFp8 ? L::kRaw + st * 2 * kTreeRawBytes : L::kTiles + st * 2 * kTreeTileBytes);
      const uint32_t vdst = kdst + (kFp8 ? kTreeRawBytes : kTreeTileBytes);
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
        if (scales) {
          const uint32_t sdst = base + L::kScales + st * 2 * kTreeBlock + 4 * lane;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sdst), "l"(kv.k_scales + srow) : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sdst + kTreeBlock), "l"(kv.v_scales + srow)
                       : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full(st)) : "memory");
        four.advance(blks, offs, ps);
      }
      first.advance(blks, offs, ps);
      box.advance(blks, offs, ps);
      if (++st == L::kStages) {
        st = 0;
        phase ^= 1;
      }
      ++issued;
    }
    // every box issued lands before the CTA may exit (bounded)
    for (int j = max(0, issued - L::kStages); j < issued; ++j) tree_land(full(j % L::kStages), (j / L::kStages) & 1);
  } else if (warp == 13) {
    // ---- issuer, the whole warp converged
    constexpr uint32_t id_s = tree_idesc(kTreeHalf, false), id_o = tree_idesc(64, true);
    const uint64_t dq = tree_desc(base + L::kQ);
    int slot = 0, next = 0, next_phase = 0;  // the block's slot; the next one's, and its phase
    auto scores = [&](int half) {
      if (!half && !wait_all(ready(next), next_phase)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      tree_mma_scores(t_s(half), dq, tree_desc(slot_at(next) + half * (kTreeHalf * 128)), id_s);
      tree_commit(b_s(half));
      return true;
    };
    bool ok = scores(0) && (halves < 2 || scores(1));
    for (int j = 0; j < nblocks && ok; ++j) {
      if (++next == L::kReady) {
        next = 0;
        next_phase ^= 1;
      }
      for (int half = 0; half < 2; ++half) {
        const int h = 2 * j + half;
        if (h >= halves) break;
        ok = wait_all(b_p(half), j & 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tree_mma_values(t_o(half), t_s(half), tree_desc(slot_at(slot) + kTreeTileBytes + half * (kTreeHalf * 128)), id_o,
                        j > 0 ? 1u : 0u);
        if (half) tree_commit(kFp8 ? free_(slot) : empty(slot));
        // the next S over the P just used: MMAs of one thread run in order
        if (h + 2 < halves) ok = scores(half);
        if (!ok) break;
      }
      slot = next;
    }
    // what was issued finishes before the results are read and TMEM is released
    tree_commit(b_o);
    if (!wait_all(b_o, 0)) tree_land(b_o, 0);
  } else if (warp >= 8) {
    // ---- block warps, one thread per position. They pass every block, also those that
    // need nothing: a wait for a phase means something only to who has waited for the last
    const int r = threadIdx.x - 256;
    static_assert(L::kStages == L::kReady, "one slot counter for both rings");
    int rd = 0, phase = 0;
    for (int j = 0; j < nblocks; ++j) {
      const int st = rd, c0 = p0 + j * kTreeBlock, pos = c0 + r;
      const bool tail = c0 + kTreeBlock > prefix;
      const bool drafted = pos >= prefix && pos < end;
      uint8_t* vrow = smem + L::kTiles + rd * 2 * kTreeTileBytes + kTreeTileBytes + r * 128;
      bool not_finite = false;
      if (!wait_all(full(st), phase)) break;
      if (kFp8) {
        if (j >= L::kReady && !wait_all(free_(rd), phase ^ 1)) break;
        const uint8_t* sc = smem + L::kScales + st * 2 * kTreeBlock;
        const int ks = sc[r];
        int vs = sc[kTreeBlock + r];
        if (pos >= end) vs = -1;  // nothing there: V is 0
        if (drafted && vs == kScaleNaN) {
          not_finite = true;
          vs = -1;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // K, V
          const int byte = x ? vs : ks;
          // 2^120 * 2^(byte - 127); above bf16's range in two factors
          const __nv_bfloat162 f = byte < 0 ? tree_pow2(0) : byte == kScaleNaN ? tree_nan2() : tree_pow2(min(byte + 120, 254));
          const __nv_bfloat162 f2 = byte + 120 > 254 && byte != kScaleNaN ? tree_pow2(byte + 120 - 254 + 127) : tree_pow2(127);
          const bool two = __any_sync(0xffffffffu, byte + 120 > 254 && byte != kScaleNaN);
          const uint8_t* src = smem + L::kRaw + st * 2 * kTreeRawBytes + x * kTreeRawBytes + r * 64;
          uint8_t* dst = smem + L::kTiles + rd * 2 * kTreeTileBytes + x * kTreeTileBytes + r * 128;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            // the codes came in with the 64-byte swizzle, the rows go out with the 128-byte one
            const uint4 u = *reinterpret_cast<const uint4*>(src + ((c ^ ((r >> 1) & 3)) << 4));
            uint2 w[4] = {tree_decode(u.x, f), tree_decode(u.y, f), tree_decode(u.z, f), tree_decode(u.w, f)};
            if (two) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                __nv_bfloat162 a = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&w[e].x), f2);
                __nv_bfloat162 d = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&w[e].y), f2);
                w[e] = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&d));
              }
            }
            *reinterpret_cast<uint4*>(dst + (((2 * c) ^ (r & 7)) << 4)) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
            *reinterpret_cast<uint4*>(dst + (((2 * c + 1) ^ (r & 7)) << 4)) = make_uint4(w[2].x, w[2].y, w[3].x, w[3].y);
          }
        }
      } else if (tail) {
        if (drafted) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint4 u = reinterpret_cast<const uint4*>(vrow)[c];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              not_finite |= (w[e] & 0x7F800000u) == 0x7F800000u || (w[e] & 0x7F80u) == 0x7F80u;
          }
        }
        if (pos >= end || not_finite) {
#pragma unroll
          for (int c = 0; c < 8; ++c) reinterpret_cast<uint4*>(vrow)[c] = make_uint4(0, 0, 0, 0);
        }
      }
      if (tail) {
        const uint32_t w = __ballot_sync(0xffffffffu, not_finite);
        if (lane == 0) bad[rd * 4 + warp - 8] = w;
      }
      if (kFp8 || tail) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (kFp8) tree_arrive(empty(st));
        tree_arrive(ready(rd));
      }
      if (++rd == L::kReady) {
        rd = 0;
        phase ^= 1;
      }
    }
  } else if ((warp & 3) < active) {
    // ---- softmax, one thread per row; warps 0-3 the first halves, 4-7 the second
    const int half = warp >> 2, r = threadIdx.x & 127;
    const int row = row0 + (r < trows ? (trow0 + r) >> p.group_log : 0);
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = t_s(half) + tl, o_at = t_o(half) + tl;
    const float c2 = p.scale * 1.4426950408889634f;  // scores in powers of two
    float m = -INFINITY, l = 0.f;  // m: the reference maximum, in powers of two
    const int mine = (halves + 1 - half) >> 1;
    bool ok = true;
    // one half block; kTail: it reaches past the committed positions
    auto step = [&](auto kind, const int j) {
      constexpr bool kTail = decltype(kind)::value, kPoly = !kFp8 && !kTail;
      unsigned long long vis = ~0ull;
      if constexpr (kTail) {
        const int rd = j % L::kReady;
        vis = tree_bits(p.mask + (size_t)row * p.words, p.words, nodes, p0 + j * kTreeBlock + half * kTreeHalf - prefix);
        if (!wait_all(ready(rd), (j / L::kReady) & 1)) return false;
        // a row that sees a V that is not finite has no finite result
        if (vis & (bad[rd * 4 + 2 * half] | (unsigned long long)bad[rd * 4 + 2 * half + 1] << 32))
          l = __uint_as_float(0x7FFFFFFFu);
      }
      if (!wait_all(b_s(half), j & 1)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (j == 0) {  // the first maximum
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t raw[32];
          tree_ld32(s_at + 32 * c, raw);
          const uint32_t v = (uint32_t)(vis >> (32 * c));
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            if (kTail) {
              if (!(v & (1u << i))) raw[i] = 0xFF800000u;  // -inf
              if (!(v & (2u << i))) raw[i + 1] = 0xFF800000u;
            }
            top[(i >> 1) & 1] = tree_max3(top[(i >> 1) & 1], __uint_as_float(raw[i]), __uint_as_float(raw[i + 1]));
          }
        }
        m = fmaxf(top[0], top[1]) * c2;
      }
      // the probabilities under the maximum so far; where a row's has grown by more
      // than 8 powers of two (or only now has one), once more under the new one
      uint32_t w[2][16];
      float2 s0, s1;
#pragma unroll 1
      for (int attempt = 0;; ++attempt) {
        const float mu = m == -INFINITY ? 0.f : m;
        const float2 scale2 = make_float2(c2, c2), shift2 = make_float2(-mu, -mu);
        float top[2] = {-INFINITY, -INFINITY};
        s0 = s1 = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t raw[32];
          tree_ld32(s_at + 32 * c, raw);
          if constexpr (kTail) {
            const uint32_t v = (uint32_t)(vis >> (32 * c));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(v & (1u << i))) raw[i] = 0xFF800000u;  // -inf
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 x = make_float2(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
            x = fma2(x, scale2, shift2);
            top[i & 1] = tree_max3(top[i & 1], x.x, x.y);
            if (kPoly && i % 5 == 3)
              x = tree_exp2(x);
            else
              x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
            if (i & 1) {
              s1 = add2(s1, x);
            } else {
              s0 = add2(s0, x);
            }
            __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
            w[c][i] = *reinterpret_cast<uint32_t*>(&h);
          }
        }
        const float mx = fmaxf(top[0], top[1]);
        const bool grow = mx > 8.f || m == -INFINITY;
        if (attempt || __builtin_expect(!__any_sync(0xffffffffu, grow), 1)) break;
        const float to = grow ? mx + mu : m;
        const float alpha = grow ? exp2_approx(m - to) : 1.f;  // 0 for the first maximum
        if (to != -INFINITY) l *= alpha;
        m = to;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[16];
            tree_ld16(o_at + 16 * c, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * (m == -INFINITY ? 1.f : alpha));
            tree_st16(o_at + 16 * c, o);
          }
        }
      }
      l += (s0.x + s0.y) + (s1.x + s1.y);
      tree_st16(s_at, w[0]);  // P over S
      tree_st16(s_at + 16, w[1]);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) tree_arrive(b_p(half));
      return true;
    };
    const int plain = min(mine, max(prefix - p0 - half * kTreeHalf + kTreeHalf, 0) / kTreeBlock);
    int j = 0;
#pragma unroll 1
    for (; j < plain && ok; ++j) ok = step(std::false_type{}, j);
#pragma unroll 1
    for (; j < mine && ok; ++j) ok = step(std::true_type{}, j);
    // ---- the two softmaxes joined, (m, l) by way of shared memory; each writes half the dims
    if (ok) ok = wait_all(b_o, 0);  // no MMA reads Q any more
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float2* ml = reinterpret_cast<float2*>(smem + L::kQ);
    ml[threadIdx.x] = make_float2(m, l);
    asm volatile("bar.sync 1, %0;" ::"r"(64 * active) : "memory");
    if (ok) {
      const bool two = halves > 1;
      const float2 x0 = ml[r], x1 = two ? ml[128 + r] : make_float2(-INFINITY, 0.f);
      const float top = fmaxf(x0.x, x1.x), mu = top == -INFINITY ? 0.f : top;
      const float a0 = exp2_approx(x0.x - mu), a1 = exp2_approx(x1.x - mu);
      const float sum = fmaf(x1.y, a1, x0.y * a0);
      const bool whole = p.splits == 1, any = sum != 0.f;  // NaN counts as something
      const float inv = !whole ? 1.f : any ? tree_inverse(sum) : 0.f, f0 = a0 * inv, f1 = a1 * inv;
      // the row's result or partial goes over the blocks, which no copy and no MMA needs any
      // more, and leaves from there with neighbouring lanes on neighbouring addresses
      uint8_t* tiles = smem + L::kTiles;
      float* part = reinterpret_cast<float*>(tiles) + r * kTreePartial;
      if (!half) {
        if (!whole)
          *reinterpret_cast<float2*>(part + 64) = make_float2(top, sum);
        else if (p.lse && r < trows)
          p.lse[(size_t)row * p.NQ + g * p.group + ((trow0 + r) & (p.group - 1))] = any ? tree_lse(mu, sum) : -INFINITY;
      }
#pragma unroll 1
      for (int c = 2 * half; c < 2 * half + 2; ++c) {
        uint32_t w[16], w1[16];
        float o[16];
        tree_ld16(t_o(0) + tl + 16 * c, w);
        if (two) tree_ld16(t_o(1) + tl + 16 * c, w1);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = __uint_as_float(w[i]) * f0;
          o[kFp8 && (i & 3) % 3 ? (i ^ 3) : i] = two ? fmaf(__uint_as_float(w1[i]), f1, x) : x;
        }
        if (whole) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              __nv_bfloat162 h = __floats2bfloat162_rn(o[8 * q + 2 * e], o[8 * q + 2 * e + 1]);
              v[e] = any ? *reinterpret_cast<uint32_t*>(&h) : 0u;
            }
            *reinterpret_cast<uint4*>(tiles + r * 128 + (((2 * c + q) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            reinterpret_cast<float4*>(part + 16 * c)[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if (p.cluster)
    tree_cluster_sync();
  else
    __syncthreads();
  if (warp == 13) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTreeTmem) : "memory");
  }
  if (p.cluster) {
    tree_join(p, base + L::kTiles, (end + p.split_len - 1) / p.split_len, split, warp, kTreeThreads / 32, lane, row0, trow0,
              trows, g);
  } else if (p.splits > 1) {
    float4* dst = reinterpret_cast<float4*>(
        p.work + ((((size_t)b * kv.NKV + g) * p.splits + split) * p.max_nodes * p.group + trow0) * kTreePartial);
    for (int i = threadIdx.x; i < trows * (kTreePartial / 4); i += kTreeThreads)
      dst[i] = reinterpret_cast<const float4*>(smem + L::kTiles)[i];
  } else {
    for (int i = threadIdx.x; i < trows * 8; i += kTreeThreads) {
      const int r = i >> 3, pr = trow0 + r;
      reinterpret_cast<uint4*>(p.out + ((size_t)(row0 + (pr >> p.group_log)) * p.NQ + g * p.group + (pr & (p.group - 1))) *
                                           64)[i & 7] =
          *reinterpret_cast<const uint4*>(smem + L::kTiles + r * 128 + (((i & 7) ^ (r & 7)) << 4));
    }
  }
}

// The splits' partials joined, in split order: a warp takes kMergeRows pairs of rows
// (node, query head).
constexpr int kMergeRows = 2;
__global__ void __launch_bounds__(256) tree_merge_kernel(const __grid_constant__ TreeParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane16 = threadIdx.x & 15, g = blockIdx.y, b = blockIdx.z;
  int row0, nodes, prefix;
  if (!tree_sequence(p, b, row0, nodes, prefix)) return;
  const int splits = (prefix + nodes + p.split_len - 1) / p.split_len;
  const size_t stride = (size_t)p.max_nodes * p.group * kTreePartial;
  const float* work = p.work + ((size_t)b * p.kv.NKV + g) * p.splits * stride;
  for (int i = 0; i < kMergeRows; ++i) {
    const int pr = (blockIdx.x * kMergeRows + i) * 16 + (threadIdx.x >> 4);
    if (pr >= nodes * p.group) return;
    TreeRow t;
    t.add(splits, [&](int q, float2& ml, float4& v) {
      const float* src = work + q * stride + (size_t)pr * kTreePartial;
      ml = *reinterpret_cast<const float2*>(src + 64);
      v = *reinterpret_cast<const float4*>(src + 4 * lane16);
    });
    t.write(p, row0 + (pr >> p.group_log), g * p.group + (pr & (p.group - 1)), lane16);
  }
}

}  // namespace mk
