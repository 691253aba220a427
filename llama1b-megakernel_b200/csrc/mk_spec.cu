// mk_spec.cu — C ABI (include/mk.h) of the speculative-decoding operators:
// cache rows written and read back (mk_kv8.cuh), attention of drafted tokens
// (mk_tree.cuh), log probabilities of tokens (mk_logprobs.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/mk.h"
#include "mk_host.cuh"
#include "mk_kv8.cuh"
#include "mk_logprobs.cuh"
#include "mk_tree.cuh"
#include "mk_tree_few.cuh"

using namespace mk::host;

namespace {

int check_layer(const MkKVLayer* kv, int32_t batch, mk::KVLayer* out) {
  if (!kv || !kv->k_pages || !kv->v_pages || !kv->block_tables) return fail(MK_EINVAL, "NULL argument");
  if (kv->format != MK_KV_BF16 && kv->format != MK_KV_E4M3) return fail(MK_EINVAL, "cache format %d", kv->format);
  if (kv->format == MK_KV_E4M3 && (!kv->k_scales || !kv->v_scales))
    return fail(MK_EINVAL, "an 8-bit cache needs k_scales and v_scales");
  if (kv->page_size < 8 || kv->page_size % 8 || kv->num_pages < 1 || kv->num_kv_heads < 1 ||
      kv->num_kv_heads > 65535 || kv->max_blocks < 1 ||
      (long long)kv->page_size * kv->max_blocks > 0x7fffffffLL)
    return fail(MK_EINVAL, "cache geometry (page_size %d, num_pages %d, num_kv_heads %d, max_blocks %d)",
                kv->page_size, kv->num_pages, kv->num_kv_heads, kv->max_blocks);
  if (!aligned16(kv->k_pages) || !aligned16(kv->v_pages))
    return fail(MK_EINVAL, "the page pools must be 16-byte aligned");
  // four scale bytes are copied at a time; a layer's begin at a multiple of its pages, heads and page size
  if (kv->format == MK_KV_E4M3 && ((reinterpret_cast<uintptr_t>(kv->k_scales) | reinterpret_cast<uintptr_t>(kv->v_scales)) & 3))
    return fail(MK_EINVAL, "k_scales and v_scales must be 4-byte aligned");
  if (batch < 1 || batch > 65535) return fail(MK_EINVAL, "batch %d outside [1, 65535]", batch);
  out->k = static_cast<uint8_t*>(kv->k_pages);
  out->v = static_cast<uint8_t*>(kv->v_pages);
  out->k_scales = static_cast<uint8_t*>(kv->k_scales);
  out->v_scales = static_cast<uint8_t*>(kv->v_scales);
  out->block_tables = kv->block_tables;
  out->ps = kv->page_size;
  out->num_pages = kv->num_pages;
  out->NKV = kv->num_kv_heads;
  out->max_blocks = kv->max_blocks;
  out->batch = batch;
  return MK_OK;
}

// Which kernel a call takes and how the positions of a sequence are split over its
// CTAs. Up to kTreeFewRows rows (nodes x query heads of a K/V head) go to the
// mma.sync kernel, in one tile of 8 or 16; more to the tcgen05 kernel in tiles of 128.
// (16 rows at 32 x 4096: 44.8 us against 45.0 of bf16, 40 against 56 of 8-bit rows; 20
// to 32 rows in a small tile of 32: 64 to 66 against 45, 57 to 59 against 56.)
//
// The cut with the least estimated time is taken, in tenths of a microsecond, fitted to
// launches of 1 to 50 sequences: a CTA costs a fixed part (first bytes, the store) and
// its share of 128 positions, more when the SM has another one; the launch costs as many
// waves of that as it fills; ranges that join cost a little in a cluster (up to eight
// ranges) and a launch and a trip through the workspace otherwise. 10 sequences of 25
// nodes behind 2,000 to 4,000 positions: 38 us whole, 34 in two, 27 in three, 29 in four.
//
// Where an SM gets a second CTA (of few rows: where not all fit at once) the longer
// sequences go first, so that short ones share SMs and fill the last wave: 28 sequences of
// 25 nodes behind 2,000 to 4,000 positions 50 us as they come, 40 so; 12 of 64 nodes behind
// 4,000 to 8,000 83 and 61; 32 of 64 over 5,200 to 8,200 8-bit positions 223 and 205. It
// costs a CTA half a microsecond, more with many sequences, which even out by themselves
// (200 of 25 nodes: 80 and 88): up to kTreeSort sequences.
//
// No cut is finer than it takes to fill the slots once. What the estimate promises
// beyond that, ragged lengths eat, as the hardware hands out whole CTAs more evenly than
// the waves here (20 such sequences: 40 us whole, 36 in two, 45 in three), and row tiles
// that share positions drift apart (4 sequences of 256 nodes at 16,000: 182 us whole, 205
// in two).
constexpr int kTreeFewRows = 16;
constexpr int kTreeMaxLen = 1 << 30;  // positions are ints that a range's and a block's length are added to
constexpr int kTreeSort = 128;
using mk::kTreeCluster;
struct TreePlan {
  int few;  // eights of rows in a tile of the mma.sync kernel (1, 2), 0: tcgen05
  int tiles, splits, len;
  bool sorted;  // the longer sequences first
  bool cluster() const { return splits > 1 && splits <= kTreeCluster; }
};
TreePlan tree_plan(int batch, int num_kv_heads, int rows, int max_len) {
  TreePlan t{};
  t.few = rows <= 8 ? 1 : rows <= kTreeFewRows ? 2 : 0;
  const int tile_rows = t.few ? 8 * t.few : mk::kTreeRows;
  t.tiles = (rows + tile_rows - 1) / tile_rows;
  const int unit = mk::kTreeBlock, units = (max_len + unit - 1) / unit;
  const long long ctas = (long long)batch * num_kv_heads * t.tiles, sms = device_sms();
  const long long slots = (t.few ? mk::kFewCtas : 2) * sms;
  long long best = -1;
  for (int want = 1, last = 0; want <= units && ctas * last < slots;) {
    const int per = (units + want - 1) / want, splits = (units + per - 1) / per;
    last = splits;
    want = per > 1 ? (units + per - 2) / (per - 1) : units + 1;  // the next that shortens the ranges
    const long long n = ctas * splits;
    auto wave = [&](long long k) -> long long {
      return k == 0 ? 0 : t.few ? 26 + 15 * per : k <= sms ? 51 + 11 * per : 65 + 18 * per;
    };
    const int join = splits == 1 ? 0 : splits <= kTreeCluster ? (t.few ? 9 : 16) : (t.few ? 25 : 50) + 2 * splits;
    const long long cost = n / slots * wave(slots) + wave(n % slots) + join;
    if (best < 0 || cost < best) {
      best = cost;
      t.splits = splits;
      t.len = per * unit;
      t.sorted = batch > 1 && batch <= kTreeSort && n > (t.few ? slots : sms);
    }
  }
  return t;
}

int64_t tree_workspace(const TreePlan& t, int batch, int num_kv_heads, int rows) {
  if (t.splits == 1 || t.cluster()) return 0;
  return (int64_t)batch * num_kv_heads * t.splits * rows * mk::kTreePartial * 4;
}

// A page pool as rows of 64 values, boxes of `box` whole rows: bf16 rows with the
// 128-byte swizzle that the tensor cores read, codes with the 64-byte one.
int encode_rows(CUtensorMap* out, const void* pool, long long rows, int box, bool fp8) {
  if (!fp8) return encode_sw128(out, pool, rows, 64, box);
  EncodeTiledFn enc = nullptr;
  if (int rc = encode_tiled_fn(&enc)) return rc;
  cuuint64_t dims[2] = {64, (cuuint64_t)rows};
  cuuint64_t strides[1] = {64};
  cuuint32_t boxes[2] = {64, (cuuint32_t)box};
  cuuint32_t es[2] = {1, 1};
  CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, boxes, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MK_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return MK_OK;
}

// The kernel's shared-memory limit, once per device.
template <typename K>
cudaError_t allow_smem(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && done[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done[dev] = true;
  return e;
}

// With programmatic stream serialization, and the ranges of a tile as a cluster where they are one.
template <typename K>
cudaError_t launch_ranges(K kernel, const mk::TreeTmaParams& tp, dim3 grid, int threads, int smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = tp.p.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tp.p.cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, tp);
}

template <bool kFp8, int RT>
cudaError_t launch_few(const mk::TreeTmaParams& tp, dim3 grid, cudaStream_t st) {
  static bool done[64];
  constexpr int smem = mk::FewShape<kFp8>::kBytes;
  if (cudaError_t e = allow_smem(mk::tree_few_kernel<kFp8, RT>, smem, done)) return e;
  return launch_ranges(mk::tree_few_kernel<kFp8, RT>, tp, grid, (mk::kFewWarps + 1) * 32, smem, st);
}

template <bool kFp8>
cudaError_t launch_tree(const mk::TreeTmaParams& tp, int few, dim3 grid, cudaStream_t st) {
  if (few == 1) return launch_few<kFp8, 1>(tp, grid, st);
  if (few == 2) return launch_few<kFp8, 2>(tp, grid, st);
  static bool done[64];
  constexpr int smem = mk::TreeSmem<kFp8>::kBytes;
  if (cudaError_t e = allow_smem(mk::tree_attn_kernel<kFp8>, smem, done)) return e;
  return launch_ranges(mk::tree_attn_kernel<kFp8>, tp, grid, mk::kTreeThreads, smem, st);
}

// How a row is cut: chunks of 16 logits a thread or of one vector, and slices of
// whole chunks. A CTA beside k - 1 others on its SM (three fit, of the small chunks
// four) takes about, in hundredths of a microsecond, 300 + 200 k, 60 for each ranking
// after the first (they come after 2, 4, 8 ... chunks), and 55 + 10 k a chunk of 16 (a
// smaller one costs more than its share): latency more than work, so a second CTA costs
// little. The cut with the least is taken. 128,256 bf16 logits, five alternatives: one
// row 10 us in 16 slices, 27 whole; 120 rows 20 in three, 24 in two, 31 whole; 200 rows
// 25 in two, 34 whole, 36 in three; 300 rows 36 whole, 42 in two. The slices of a row are a
// cluster; more than the portable eight only for a few rows, which cannot fill the GPU
// otherwise.
constexpr int kLpMaxVocab = 1 << 30;
struct LpCut {
  int per, slices, len;
};
LpCut lp_cut(int rows, int vocab, int vector) {
  const int sms = device_sms(), most = rows <= 8 ? mk::kLpMaxSlices : 8;
  LpCut best{};
  long long least = -1;
  for (int per : {16, vector}) {
    const int n = (int)(((long long)vocab + mk::kLpThreads * per - 1) / (mk::kLpThreads * per));
    for (int want = 1; want <= std::min(n, most); ++want) {
      const int e = (n + want - 1) / want, k = (n + e - 1) / e;
      int ranks = 0, fit = per == 16 ? 3 : 4;
      while ((1 << ranks) < e) ++ranks;
      auto wave = [&](long long on) -> long long {
        return on == 0 ? 0 : 300 + 200 * on + 60 * ranks + e * (per == 16 ? 16 : per + 2) * (55 + 10 * on) / 16;
      };
      // clusters do not fill the last slots (148 rows in three: 32 us, in two 24)
      const long long ctas = (long long)rows * k, on = (ctas + (k > 1 ? ctas / 32 : 0) + sms - 1) / sms;
      const long long cost = on / fit * wave(fit) + wave(on % fit);
      if (least < 0 || cost < least) {
        least = cost;
        best = {per, k, e * mk::kLpThreads * per};
      }
    }
  }
  return best;
}

template <typename T, int E, bool kVec>
cudaError_t launch_logprobs_k(const mk::LogprobsParams& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.slices, p.rows);
  cfg.blockDim = dim3(mk::kLpThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.slices;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.slices > 1 ? 2 : 1;
  if (p.slices > 8) {
    static bool done[64];
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    if (dev >= 64 || !done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(mk::logprobs_kernel<T, E, kVec>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
      if (dev < 64) done[dev] = true;
    }
  }
  return cudaLaunchKernelEx(&cfg, mk::logprobs_kernel<T, E, kVec>, p);
}

template <typename T>
cudaError_t launch_logprobs(const mk::LogprobsParams& p, int per, bool vec, cudaStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  if (per == N) return vec ? launch_logprobs_k<T, N, true>(p, st) : launch_logprobs_k<T, N, false>(p, st);
  return vec ? launch_logprobs_k<T, 16, true>(p, st) : launch_logprobs_k<T, 16, false>(p, st);
}

}  // namespace

extern "C" {

int mk_kv_write(const MkKVLayer* kv, int32_t batch, const void* qkv, const void* rope_cos,
                const void* rope_sin, int32_t rope_len, const int32_t* seqs, const int32_t* slots,
                const int32_t* positions, int32_t rows, int32_t num_q_heads, void* q_out,
                int32_t* error, void* stream) {
  mk::KVWriteParams p{};
  if (int rc = check_layer(kv, batch, &p.kv)) return rc;
  if (rows < 0 || num_q_heads < 1 || num_q_heads > 65535 || rope_len < 1)
    return fail(MK_EINVAL, "rows %d, num_q_heads %d, rope_len %d", rows, num_q_heads, rope_len);
  if (rows == 0) return MK_OK;  // arrays of nothing may be NULL
  if (!qkv || !rope_cos || !rope_sin || !seqs || !slots || !positions || !q_out || !error)
    return fail(MK_EINVAL, "NULL argument");
  if (!aligned16(qkv) || !aligned16(rope_cos) || !aligned16(rope_sin) || !aligned16(q_out))
    return fail(MK_EINVAL, "qkv, the RoPE tables and q_out must be 16-byte aligned");
  p.qkv = static_cast<const uint8_t*>(qkv);
  p.cos_t = static_cast<const __nv_bfloat16*>(rope_cos);
  p.sin_t = static_cast<const __nv_bfloat16*>(rope_sin);
  p.seqs = seqs;
  p.slots = slots;
  p.positions = positions;
  p.rows = rows;
  p.NQ = num_q_heads;
  p.rope_len = rope_len;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.error = error;
  const int64_t pairs = (int64_t)rows * ((num_q_heads + 2 * kv->num_kv_heads + 1) / 2);
  const int64_t ctas = (pairs + 31) / 32;
  if (ctas > 0x7ffffffLL) return fail(MK_EINVAL, "%d rows of %d query heads", rows, num_q_heads);
  MK_CUDA(launch_pdl(kv->format == MK_KV_E4M3 ? mk::kv_write_kernel<true> : mk::kv_write_kernel<false>,
                     dim3((unsigned)ctas), dim3(256), 0, static_cast<cudaStream_t>(stream), p));
  return MK_OK;
}

int mk_kv_read(const MkKVLayer* kv, const int32_t* lengths, int32_t batch, int32_t max_len,
               void* k_out, void* v_out, int32_t* error, void* stream) {
  mk::KVReadParams p{};
  if (int rc = check_layer(kv, batch, &p.kv)) return rc;
  if (max_len < 0 || max_len > (long long)kv->page_size * kv->max_blocks)
    return fail(MK_EINVAL, "max_len %d outside [0, page_size * max_blocks]", max_len);
  if (max_len == 0) return MK_OK;
  if (!lengths || !k_out || !v_out || !error) return fail(MK_EINVAL, "NULL argument");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(MK_EINVAL, "k_out and v_out must be 16-byte aligned");
  p.lengths = lengths;
  p.max_len = max_len;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.error = error;
  MK_CUDA(launch_pdl(kv->format == MK_KV_E4M3 ? mk::kv_read_kernel<true> : mk::kv_read_kernel<false>,
                     dim3((unsigned)(((int64_t)max_len * 8 + 255) / 256), kv->num_kv_heads, batch),
                     dim3(256), 0, static_cast<cudaStream_t>(stream), p));
  return MK_OK;
}

int64_t mk_tree_attention_workspace(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                    int32_t max_nodes, int32_t max_len) {
  if (batch < 1 || batch > 65535 || num_kv_heads < 1 || num_q_heads < num_kv_heads || max_nodes < 1 ||
      max_nodes > mk::kTreeMaxNodes || max_len < 1 || max_len > kTreeMaxLen)
    return 0;
  const int group = num_q_heads / num_kv_heads;
  if (group > 8) return 0;
  return tree_workspace(tree_plan(batch, num_kv_heads, max_nodes * group, max_len), batch, num_kv_heads, max_nodes * group);
}

int mk_tree_attention(const void* q, const MkKVLayer* kv, const int32_t* cu_nodes,
                      const uint64_t* mask, const int32_t* prefix_lens, int32_t batch, int32_t rows,
                      int32_t max_nodes, int32_t max_len, int32_t num_q_heads, float scale,
                      void* workspace, int64_t workspace_bytes, void* out, float* lse,
                      int32_t* error, void* stream) {
  mk::TreeTmaParams tp{};
  mk::TreeParams& p = tp.p;
  if (int rc = check_layer(kv, batch, &p.kv)) return rc;
  const int nkv = kv->num_kv_heads;
  const int group = num_q_heads / nkv;
  if (num_q_heads < 1 || num_q_heads % nkv || (group != 1 && group != 2 && group != 4 && group != 8))
    return fail(MK_EINVAL, "num_q_heads %d must be 1, 2, 4 or 8 times num_kv_heads %d", num_q_heads, nkv);
  if (max_nodes < 1 || max_nodes > mk::kTreeMaxNodes)
    return fail(MK_EINVAL, "max_nodes %d outside [1, %d]", max_nodes, mk::kTreeMaxNodes);
  if (rows < 0 || max_len < 1 || max_len > kTreeMaxLen || max_len > (long long)kv->page_size * kv->max_blocks)
    return fail(MK_EINVAL, "rows %d, max_len %d (at most %d; page_size %d, max_blocks %d)", rows, max_len, kTreeMaxLen,
                kv->page_size, kv->max_blocks);
  if (!(scale > 0.f) || !(scale < 3.0e38f)) return fail(MK_EINVAL, "scale %g must be positive and finite", (double)scale);
  if (rows == 0) return MK_OK;
  if (!q || !cu_nodes || !mask || !prefix_lens || !out || !error) return fail(MK_EINVAL, "NULL argument");
  if (!aligned16(q) || !aligned16(out)) return fail(MK_EINVAL, "q and out must be 16-byte aligned");
  const long long pool_rows = (long long)kv->num_pages * nkv * kv->page_size;
  if (pool_rows > 0x7fffffffLL) return fail(MK_EINVAL, "KV pool of %lld rows", pool_rows);
  const TreePlan plan = tree_plan(batch, nkv, max_nodes * group, max_len);
  const int64_t need = tree_workspace(plan, batch, nkv, max_nodes * group);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(MK_EINVAL, "workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  if (need > 0 && !aligned16(workspace)) return fail(MK_EINVAL, "workspace must be 16-byte aligned");
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.cu_nodes = cu_nodes;
  p.mask = reinterpret_cast<const unsigned long long*>(mask);
  p.prefix = prefix_lens;
  p.rows = rows;
  p.words = (max_nodes + 63) / 64;
  p.max_nodes = max_nodes;
  p.max_len = max_len;
  p.NQ = num_q_heads;
  p.group = group;
  p.group_log = group == 8 ? 3 : group >> 1;
  p.scale = scale;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.error = error;
  p.tiles = plan.tiles;
  p.splits = plan.splits;
  p.split_len = plan.len;
  p.cluster = plan.cluster();
  if (plan.sorted)
    for (p.sorted = 1; max_len >> (p.sorted - 1) > 31;) ++p.sorted;
  p.work = static_cast<float*>(workspace);
  const bool fp8 = kv->format == MK_KV_E4M3;
  p.box = !plan.few ? mk::kTreeBlock : fp8 ? mk::FewShape<true>::kChunk : mk::FewShape<false>::kChunk;
  while (kv->page_size % p.box) p.box /= 2;
  if (int rc = encode_rows(&tp.tm_k, kv->k_pages, pool_rows, p.box, fp8)) return rc;
  if (int rc = encode_rows(&tp.tm_v, kv->v_pages, pool_rows, p.box, fp8)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(p.tiles * p.splits, nkv, batch);
  MK_CUDA(fp8 ? launch_tree<true>(tp, plan.few, grid, st) : launch_tree<false>(tp, plan.few, grid, st));
  if (p.splits > 1 && !p.cluster)
    MK_CUDA(launch_pdl(mk::tree_merge_kernel, dim3((max_nodes * group + 16 * mk::kMergeRows - 1) / (16 * mk::kMergeRows), nkv, batch), dim3(256), 0, st, p));
  return MK_OK;
}

int64_t mk_token_logprobs_workspace(int32_t rows, int32_t vocab, int32_t top) {
  (void)rows;
  (void)vocab;
  (void)top;
  return 0;  // a row's slices meet in distributed shared memory
}

int mk_token_logprobs(const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t ld,
                      const int32_t* targets, int32_t num_targets, int32_t top, void* workspace,
                      int64_t workspace_bytes, float* logprobs, float* entropy, int32_t* top_ids,
                      float* top_logprobs, int32_t* error, void* stream) {
  if (dtype != MK_F32 && dtype != MK_BF16) return fail(MK_EINVAL, "logits type %d", dtype);
  if (rows < 0 || vocab < 1 || vocab > kLpMaxVocab || ld < vocab) return fail(MK_EINVAL, "rows %d, vocab %d, ld %lld", rows, vocab, (long long)ld);
  if (num_targets < 0) return fail(MK_EINVAL, "num_targets %d", num_targets);
  if (top < 0 || top > mk::kLogprobsMaxTop || top > vocab)
    return fail(MK_EINVAL, "top %d must be in [0, min(%d, vocab)]", top, mk::kLogprobsMaxTop);
  if (rows == 0) return MK_OK;
  if (!logits || !entropy || !error) return fail(MK_EINVAL, "NULL argument");
  if (num_targets && (!targets || !logprobs)) return fail(MK_EINVAL, "num_targets %d needs targets and logprobs", num_targets);
  if (top && (!top_ids || !top_logprobs)) return fail(MK_EINVAL, "top %d needs top_ids and top_logprobs", top);
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == MK_F32 ? 4 : 2)) return fail(MK_EINVAL, "logits are not aligned to their type");
  (void)workspace;
  (void)workspace_bytes;
  mk::LogprobsParams p{};
  p.logits = logits;
  p.ld = ld;
  p.rows = rows;
  p.V = vocab;
  p.num_targets = num_targets;
  p.top = top;
  p.targets = targets;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  p.error = error;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int size = dtype == MK_F32 ? 4 : 2;
  const LpCut cut = lp_cut(rows, vocab, 16 / size);
  p.slices = cut.slices;
  p.slice_len = cut.len;
  const bool vec = aligned16(logits) && (rows == 1 || (ld * size) % 16 == 0);
  // rows go in launches of at most 65,535 (the grid's second dimension)
  for (int r0 = 0; r0 < rows; r0 += 65535) {
    mk::LogprobsParams q = p;
    const int64_t n = std::min(rows - r0, 65535);
    q.logits = static_cast<const uint8_t*>(logits) + (int64_t)r0 * ld * size;
    q.rows = (int)n;
    q.targets += (int64_t)r0 * num_targets;
    q.logprobs += (int64_t)r0 * num_targets;
    q.entropy += r0;
    q.top_ids += (int64_t)r0 * top;
    q.top_logprobs += (int64_t)r0 * top;
    MK_CUDA(dtype == MK_F32 ? launch_logprobs<float>(q, cut.per, vec, st) : launch_logprobs<__nv_bfloat16>(q, cut.per, vec, st));
  }
  return MK_OK;
}

}  // extern "C"
