// paged_api.cuh -- C entry points of the paged 4-bit K/V cache, of the
// attention over it and of packed prompt attention (included by b2q_api.cu).
// None of them allocates, synchronises or keeps state: the caller owns the
// pool, the workspace and the outputs, so calls on different streams do not
// meet, and every call can be captured into a graph.
#pragma once

#include <atomic>

#include "internal.h"
#include "attn_paged.cuh"
#include "attn_prompt.cuh"

namespace b2q {

// Makes the engine's device current and the caller's again at the end.
struct DeviceGuard {
  int prev = -1;
  cudaError_t err;
  explicit DeviceGuard(int dev) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != dev) err = cudaSetDevice(dev);
    else if (err == cudaSuccess) prev = -1;
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

static int el_type(int ggml_type) {
  return ggml_type == B2Q_F32 ? kElF32 : ggml_type == B2Q_F16 ? kElF16 : ggml_type == B2Q_BF16 ? kElBF16 : -1;
}
static int el_size(int el) { return el == kElF32 ? 4 : 2; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static b2q_status check_heads(const char* what, int n_heads, int n_kv_heads, int head_dim) {
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads > 1024)
    return set_error(B2Q_EINVAL, "%s: %d query heads over %d K/V heads", what, n_heads, n_kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return set_error(B2Q_EUNSUP, "%s: head_dim %d (64 and 128 are supported)", what, head_dim);
  return B2Q_OK;
}

static b2q_status check_kv_config(const char* what, const b2q_kv_config* c) {
  if (!c) return set_error(B2Q_EINVAL, "%s: NULL configuration", what);
  b2q_status s = check_heads(what, c->n_heads, c->n_kv_heads, c->head_dim);
  if (s != B2Q_OK) return s;
  if (c->kv_type != B2Q_Q4_0)
    return set_error(B2Q_EUNSUP, "%s: cache type %d (B2Q_Q4_0 is supported)", what, c->kv_type);
  if (c->page_tokens < kKvBlk || c->page_tokens % kKvBlk || c->page_tokens > 4096)
    return set_error(B2Q_EINVAL, "%s: %d tokens a page (a multiple of 16, at most 4096)", what, c->page_tokens);
  if (c->n_pages <= 0 || c->max_pages <= 0 || (int64_t)c->max_pages * c->page_tokens > (1 << 30))
    return set_error(B2Q_EINVAL, "%s: bad pool (%d pages, at most %d a sequence)", what, c->n_pages, c->max_pages);
  return B2Q_OK;
}

static b2q_status check_kv_batch(const char* what, const b2q_kv_batch* b) {
  if (!b) return set_error(B2Q_EINVAL, "%s: NULL batch", what);
  if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_new < 0 || b->n_seqs > 65535)
    return set_error(B2Q_EINVAL, "%s: bad batch (%d sequences, %d tokens, at most %d new)", what, b->n_seqs, b->n_tokens,
                     b->max_new);
  if (!b->q_start || !b->kv_len || !b->page_table) return set_error(B2Q_EINVAL, "%s: NULL array in the batch", what);
  return B2Q_OK;
}

// A strided [tokens][heads * D] operand: 16-byte aligned rows that do not overlap.
static b2q_status check_rows(const char* what, const char* name, const void* p, int64_t stride, int64_t width, int el) {
  if (!p) return set_error(B2Q_EINVAL, "%s: %s is NULL", what, name);
  if (!aligned16(p) || (stride * el_size(el)) % 16)
    return set_error(B2Q_EINVAL, "%s: the rows of %s must start on 16-byte boundaries", what, name);
  if (stride < width || stride > ((int64_t)1 << 31))
    return set_error(B2Q_EINVAL, "%s: %s has %lld elements between rows of %lld", what, name, (long long)stride,
                     (long long)width);
  return B2Q_OK;
}

static KvBatch make_batch(const b2q_kv_config& c, const b2q_kv_batch& b) {
  KvBatch k;
  k.n_seqs = b.n_seqs;
  k.n_tokens = b.n_tokens;
  k.KV = c.n_kv_heads;
  k.D = c.head_dim;
  k.page_tokens = c.page_tokens;
  k.n_pages = c.n_pages;
  k.max_pages = c.max_pages;
  k.q_start = b.q_start;
  k.kv_len = b.kv_len;
  k.page_table = b.page_table;
  return k;
}

// A launch that may start while the one before it on the stream drains; the
// kernels wait for that one (pdl_wait) before they touch memory.
static cudaLaunchConfig_t dependent_launch(unsigned grid, unsigned block, size_t smem, cudaStream_t st,
                                           cudaLaunchAttribute (&attr)[1]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// f(integral_constant...) for the element types' and the head width's instances
template <typename F>
static void by_type(int el, F f) {
  if (el == kElF32) f(std::integral_constant<int, kElF32>());
  else if (el == kElF16) f(std::integral_constant<int, kElF16>());
  else f(std::integral_constant<int, kElBF16>());
}
template <typename F>
static void by_dim(int D, F f) {
  if (D == 64) f(std::integral_constant<int, 64>());
  else f(std::integral_constant<int, 128>());
}

// Lets a kernel take `bytes` of shared memory on the current device; asked
// once per kernel and device (`done`: bits of the first 64).
template <typename K>
static cudaError_t allow_smem(K* kern, int bytes, int device, std::atomic<uint64_t>& done) {
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return err;
}

// CTAs of the paged attention: one per SM.
static int paged_ctas(const b2q_engine* e) { return std::max(1, std::min(e->num_sms, kPgMaxCtas)); }
static size_t paged_desc_bytes(int ctas) { return ((size_t)ctas * 2 * sizeof(PgDesc) + 255) / 256 * 256; }

template <int D, int NG, bool QSPLIT, bool PSPLIT>
static cudaError_t launch_paged(const PagedArgs& a, int ctas, int device, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  cudaError_t err = allow_smem(attn_paged_kernel<D, NG, QSPLIT, PSPLIT>, pg_ring_bytes(D, NG), device, done);
  if (err != cudaSuccess) return err;
  cudaLaunchAttribute attr[1], both[2];
  cudaLaunchConfig_t cfg = dependent_launch((unsigned)ctas, pg_warps(NG) * 32, pg_ring_bytes(D, NG), st, attr);
  if (a.whole > 1) {
    both[0] = attr[0];
    both[1].id = cudaLaunchAttributeClusterDimension;
    both[1].val.clusterDim.x = (unsigned)a.whole;
    both[1].val.clusterDim.y = both[1].val.clusterDim.z = 1;
    cfg.attrs = both;
    cfg.numAttrs = 2;
  }
  err = cudaLaunchKernelEx(&cfg, attn_paged_kernel<D, NG, QSPLIT, PSPLIT>, a);
  if (err != cudaSuccess || a.whole) return err;
  cfg.blockDim = dim3(kPgJoinThreads);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attn_paged_join_kernel<D, NG>, a);
}

// Tensor maps of the prompt attention: boxes with rows of 64 elements (128
// bytes, 128-byte swizzle).  Queries as (dim, head of the group, K/V head,
// token), a box of tpt tokens with gp heads each; keys and values as (dim, K/V
// head, token), a box of 128 tokens.  Rows past the end read as zeros.
static bool prompt_map(CUtensorMap* m, int type, int rank, const void* p, const cuuint64_t* dims, const cuuint64_t* strides,
                       const cuuint32_t* box) {
  const TmapEncodeFn enc = tmap_encoder();
  const cuuint32_t one[4] = {1u, 1u, 1u, 1u};
  return enc != nullptr &&
         enc(m, type == kElF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank,
             const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static bool prompt_map_q(CUtensorMap* m, const PromptArgs& a, int D, int type) {
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.G, (cuuint64_t)a.KV, (cuuint64_t)a.n_q};
  const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)a.G * D * 2, (cuuint64_t)a.q_stride * 2};
  const cuuint32_t box[4] = {64u, (cuuint32_t)a.gp, 1u, (cuuint32_t)a.tpt};
  return prompt_map(m, type, 4, a.q, dims, strides, box);
}
static bool prompt_map_kv(CUtensorMap* m, const void* p, int64_t stride, int rows, int KV, int D, int type) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)KV, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)kPrN};
  return prompt_map(m, type, 3, p, dims, strides, box);
}
template <int D, int TYPE, bool HALVES>
static cudaError_t launch_prompt(const PromptArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                                 unsigned grid, int device, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  cudaError_t err = allow_smem(attn_prompt_kernel<D, TYPE, HALVES>, pr_smem_bytes(D), device, done);
  if (err != cudaSuccess) return err;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = dependent_launch(grid, kPrThreads, pr_smem_bytes(D), st, attr);
  return cudaLaunchKernelEx(&cfg, attn_prompt_kernel<D, TYPE, HALVES>, a, mq, mk, mv);
}

}  // namespace b2q

extern "C" {

size_t b2q_kv_page_bytes(const b2q_kv_config* cfg) {
  if (check_kv_config("b2q_kv_page_bytes", cfg) != B2Q_OK) return 0;
  return (size_t)cfg->n_kv_heads * (cfg->page_tokens / kKvBlk) * kv_blk_bytes(cfg->head_dim);
}

b2q_status b2q_kv_append_dev(b2q_engine* e, const b2q_kv_config* cfg, const b2q_kv_batch* batch, const b2q_rope* rope,
                             int x_type, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                             int64_t v_stride, void* pages, void* q_out, int q_out_type, void* stream) {
  static const char* const what = "b2q_kv_append_dev";
  if (!e) return set_error(B2Q_EINVAL, "%s: NULL engine", what);
  b2q_status s = check_kv_config(what, cfg);
  if (s == B2Q_OK) s = check_kv_batch(what, batch);
  if (s != B2Q_OK) return s;
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return B2Q_OK;  // (empty tensors have NULL addresses)
  const int xt = el_type(x_type), D = cfg->head_dim;
  const int ot = q ? el_type(q_out_type) : (int)kElF32;
  if (xt < 0 || ot < 0) return set_error(B2Q_EUNSUP, "%s: element type %d", what, xt < 0 ? x_type : q_out_type);
  s = check_rows(what, "k", k, k_stride, (int64_t)cfg->n_kv_heads * D, xt);
  if (s == B2Q_OK) s = check_rows(what, "v", v, v_stride, (int64_t)cfg->n_kv_heads * D, xt);
  if (s == B2Q_OK && q) s = check_rows(what, "q", q, q_stride, (int64_t)cfg->n_heads * D, xt);
  if (s == B2Q_OK && q) s = check_rows(what, "q_out", q_out, (int64_t)cfg->n_heads * D, (int64_t)cfg->n_heads * D, ot);
  if (s != B2Q_OK) return s;
  if (!pages || !aligned16(pages)) return set_error(B2Q_EINVAL, "%s: pages must be a 16-byte aligned pointer", what);
  if (rope && rope->rot_dim) {
    if (rope->rot_dim < 0 || rope->rot_dim > D || rope->rot_dim % 8 || rope->n_pos <= 0)
      return set_error(B2Q_EINVAL, "%s: rotation of %d dims (a multiple of 8, at most %d) over %d positions", what,
                       rope->rot_dim, D, rope->n_pos);
    if (!rope->cos || !rope->sin || !aligned16(rope->cos) || !aligned16(rope->sin))
      return set_error(B2Q_EINVAL, "%s: the rotation tables must be 16-byte aligned pointers", what);
  }
  DeviceGuard dev(e->device);
  if (dev.err != cudaSuccess) return cuda_error(dev.err, what);
  AppendArgs a;
  a.b = make_batch(*cfg, *batch);
  a.H = cfg->n_heads;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.rot_dim = rope ? rope->rot_dim : 0;
  a.n_pos = rope ? rope->n_pos : 0;
  a.cos = rope ? rope->cos : nullptr;
  a.sin = rope ? rope->sin : nullptr;
  a.pages = static_cast<uint8_t*>(pages);
  a.q_out = q_out;
  cudaLaunchAttribute attr[1];
  // a token to a CTA while that fills the GPU once, then four
  const int tok = a.b.n_tokens <= 4 * e->num_sms ? 1 : 4;
  const cudaLaunchConfig_t lc =
      dependent_launch((unsigned)((a.b.n_tokens + tok - 1) / tok), kAppendThreads, 0, stream ? (cudaStream_t)stream : e->stream, attr);
  cudaError_t err = cudaSuccess;
  by_dim(D, [&](auto d) {
    by_type(xt, [&](auto x) {
      by_type(ot, [&](auto o) {
        err = tok == 1 ? cudaLaunchKernelEx(&lc, kv_append_kernel<d(), x(), o(), 1>, a)
                       : cudaLaunchKernelEx(&lc, kv_append_kernel<d(), x(), o(), 4>, a);
      });
    });
  });
  launch_counted(e, 1);
  return err == cudaSuccess ? B2Q_OK : cuda_error(err, what);
}

b2q_status b2q_kv_gather_dev(b2q_engine* e, const b2q_kv_config* cfg, const b2q_kv_batch* batch, const void* pages,
                             void* k_out, void* v_out, int out_type, void* stream) {
  static const char* const what = "b2q_kv_gather_dev";
  if (!e) return set_error(B2Q_EINVAL, "%s: NULL engine", what);
  b2q_status s = check_kv_config(what, cfg);
  if (s == B2Q_OK) s = check_kv_batch(what, batch);
  if (s != B2Q_OK) return s;
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return B2Q_OK;  // (empty tensors have NULL addresses)
  const int ot = el_type(out_type);
  if (ot < 0) return set_error(B2Q_EUNSUP, "%s: element type %d", what, out_type);
  if (!k_out && !v_out) return set_error(B2Q_EINVAL, "%s: neither k_out nor v_out", what);
  if (!pages || !aligned16(pages) || !aligned16(k_out) || !aligned16(v_out))
    return set_error(B2Q_EINVAL, "%s: pages, k_out and v_out must be 16-byte aligned", what);
  DeviceGuard dev(e->device);
  if (dev.err != cudaSuccess) return cuda_error(dev.err, what);
  GatherArgs a;
  a.b = make_batch(*cfg, *batch);
  a.pages = static_cast<const uint8_t*>(pages);
  a.k_out = k_out;
  a.v_out = v_out;
  cudaLaunchAttribute attr[1];
  // heads apart while that brings CTAs to fill the GPU eight times; a CTA keeps two
  // heads (a turn for each of its warps).  64 rows of 8 heads: 3 us, by whole rows 12.
  const int gx = (a.b.n_tokens + kGatherRows - 1) / kGatherRows;
  a.heads = std::max(2, (int)std::min<int64_t>(a.b.KV, ((int64_t)gx * a.b.KV + 8 * e->num_sms - 1) / (8 * e->num_sms)));
  cudaLaunchConfig_t lc = dependent_launch((unsigned)gx, 256, 0, stream ? (cudaStream_t)stream : e->stream, attr);
  lc.gridDim.y = (unsigned)((a.b.KV + a.heads - 1) / a.heads);
  cudaError_t err = cudaSuccess;
  by_dim(cfg->head_dim, [&](auto d) {
    by_type(ot, [&](auto o) { err = cudaLaunchKernelEx(&lc, kv_gather_kernel<d(), o()>, a); });
  });
  launch_counted(e, 1);
  return err == cudaSuccess ? B2Q_OK : cuda_error(err, what);
}

size_t b2q_attn_paged_work_bytes(const b2q_engine* e, const b2q_kv_config* cfg, const b2q_kv_batch* batch) {
  static const char* const what = "b2q_attn_paged_work_bytes";
  if (!e) set_error(B2Q_EINVAL, "%s: NULL engine", what);
  if (!e || check_kv_config(what, cfg) != B2Q_OK || check_kv_batch(what, batch) != B2Q_OK) return 0;
  // descriptors and pieces of the items cut between CTAs (16 rows: either tiling)
  const size_t ctas = paged_ctas(e), D = cfg->head_dim;
  return paged_desc_bytes(ctas) + ctas * 2 * pg_part_floats(D, 2) * sizeof(float) +
         ctas * std::max(pg_warps(1) * pg_piece_floats(D, 1), pg_warps(2) * pg_piece_floats(D, 2)) * sizeof(float);
}

b2q_status b2q_attn_paged_dev(b2q_engine* e, const b2q_kv_config* cfg, const b2q_kv_batch* batch, const void* q, int q_type,
                              int64_t q_stride, const void* pages, float scale, void* out, int out_type, void* work,
                              size_t work_bytes, void* stream) {
  static const char* const what = "b2q_attn_paged_dev";
  if (!e) return set_error(B2Q_EINVAL, "%s: NULL engine", what);
  b2q_status s = check_kv_config(what, cfg);
  if (s == B2Q_OK) s = check_kv_batch(what, batch);
  if (s != B2Q_OK) return s;
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return B2Q_OK;  // (empty tensors have NULL addresses)
  const int qt = el_type(q_type), ot = el_type(out_type), D = cfg->head_dim;
  if (qt < 0 || ot < 0) return set_error(B2Q_EUNSUP, "%s: element type %d", what, qt < 0 ? q_type : out_type);
  s = check_rows(what, "q", q, q_stride, (int64_t)cfg->n_heads * D, qt);
  if (s == B2Q_OK) s = check_rows(what, "out", out, (int64_t)cfg->n_heads * D, (int64_t)cfg->n_heads * D, ot);
  if (s != B2Q_OK) return s;
  if (!pages || !aligned16(pages)) return set_error(B2Q_EINVAL, "%s: pages must be a 16-byte aligned pointer", what);
  if ((int64_t)batch->n_tokens * cfg->n_heads > (1 << 30))
    return set_error(B2Q_EINVAL, "%s: %d tokens of %d heads in one call", what, batch->n_tokens, cfg->n_heads);
  if (!(scale > 0.0f && scale <= 1e30f)) return set_error(B2Q_EINVAL, "%s: scale must be positive and at most 1e30", what);
  const size_t need = b2q_attn_paged_work_bytes(e, cfg, batch);
  if (!work || !aligned16(work) || work_bytes < need)
    return set_error(B2Q_EINVAL, "%s: a workspace of %zu bytes is needed (%zu given)", what, need, work_bytes);
  DeviceGuard dev(e->device);
  if (dev.err != cudaSuccess) return cuda_error(dev.err, what);
  PagedArgs a;
  a.b = make_batch(*cfg, *batch);
  a.H = cfg->n_heads;
  a.G = cfg->n_heads / cfg->n_kv_heads;
  a.q = q;
  a.q_type = qt;
  a.q_stride = q_stride;
  a.pages = static_cast<const uint8_t*>(pages);
  a.scale = scale;
  a.out = out;
  a.out_type = ot;
  cudaStream_t st = stream ? (cudaStream_t)stream : e->stream;
  a.dG = fast_div(a.G);
  a.dKV = fast_div(a.b.KV);
  a.dPage = fast_div(a.b.page_tokens);
  // all sequences as long as their pages allow, in units of 2^coarse blocks
  const int64_t blocks = ((int64_t)a.b.max_pages * a.b.page_tokens + kKvBlk - 1) / kKvBlk;
  const int64_t items = ((int64_t)a.b.n_tokens * a.G / 8 + 2 * (int64_t)a.b.n_seqs) * a.b.KV;
  a.coarse = 0;
  while (a.coarse < 26 && items * (((blocks - 1) >> a.coarse) + 1 + kPgSetup) > INT32_MAX) ++a.coarse;
  if (items * (((blocks - 1) >> a.coarse) + 1 + kPgSetup) > INT32_MAX)
    return set_error(B2Q_EINVAL, "%s: %d tokens of %d heads in one call", what, a.b.n_tokens, a.H);
  const int ctas = paged_ctas(e);
  a.desc = static_cast<PgDesc*>(work);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + paged_desc_bytes(ctas));
  a.part0 = a.part + (size_t)ctas * 2 * pg_part_floats(D, 2);
  // 16 rows to an item where the queries are 16-bit (f32 ones take the matrix
  // tile's other 8 rows for their second part) and more than 8 rows share a K/V head
  const bool wide = qt != kElF32 && (int64_t)batch->max_new * a.G > 8;
  // the probabilities' second part where the output shows it
  const bool split = ot == kElF32;
  // Few items that the page table keeps short: a cluster of CTAs to each, the more
  // the better down to half a block of keys a warp, and no second launch.  Device
  // times so / by the line, 8 K/V heads: one sequence of 100 tokens 7.8 / 8.9 us, 585
  // 9.5 / 12.2, 2048 11.7 / 13.4; four of 1024 11.7 / 13.8, of 2048 (2.7 blocks a
  // warp, without this limit) 16.1 / 14.6: the line leaves no SM without work.
  // (sequences with rows: k at most, so row blocks: (rows + k (R - 1)) / R at most)
  const int warps = pg_warps(wide ? 2 : 1), R = pg_rows(wide ? 2 : 1);
  const int64_t k = std::min(a.b.n_seqs, a.b.n_tokens);
  const int64_t few = std::min(((int64_t)a.b.n_tokens * a.G + k * (R - 1)) / R, (int64_t)a.b.n_tokens * ((a.G + R - 1) / R)) * a.b.KV;
  // (the larger a cluster the fewer SMs a GPU full of them reaches: 16 of eight CTAs took
  // two rounds, two sequences of 585 tokens 16.7 us; in clusters of four 10.6)
  int cluster = 1;
  if (blocks > warps)
    while (cluster < kPgMaxCluster && 2 * cluster * few <= (cluster == 1 ? ctas : cluster == 2 ? ctas * 7 / 8 : ctas * 2 / 3) &&
           2 * blocks > cluster * warps)
      cluster *= 2;
  a.whole = cluster * few <= ctas && blocks <= 2 * cluster * warps ? cluster : 0;
  const int grid = a.whole ? (int)(few * cluster) : ctas;
  cudaError_t err = cudaSuccess;
  by_dim(D, [&](auto d) {
    if (wide) err = split ? launch_paged<d(), 2, false, true>(a, grid, e->device, st) : launch_paged<d(), 2, false, false>(a, grid, e->device, st);
    else if (qt == kElF32) err = split ? launch_paged<d(), 1, true, true>(a, grid, e->device, st) : launch_paged<d(), 1, true, false>(a, grid, e->device, st);
    else err = split ? launch_paged<d(), 1, false, true>(a, grid, e->device, st) : launch_paged<d(), 1, false, false>(a, grid, e->device, st);
  });
  launch_counted(e, a.whole ? 1 : 2);
  return err == cudaSuccess ? B2Q_OK : cuda_error(err, what);
}

b2q_status b2q_attn_prompt_dev(b2q_engine* e, const b2q_prompt* p, const void* q, int64_t q_stride, const void* k,
                               int64_t k_stride, const void* v, int64_t v_stride, float scale, void* out, void* stream) {
  static const char* const what = "b2q_attn_prompt_dev";
  if (!e || !p) return set_error(B2Q_EINVAL, "%s: NULL argument", what);
  b2q_status s = check_heads(what, p->n_heads, p->n_kv_heads, p->head_dim);
  if (s != B2Q_OK) return s;
  const int t = el_type(p->type), D = p->head_dim;
  if (t != kElF16 && t != kElBF16) return set_error(B2Q_EUNSUP, "%s: element type %d (F16 and BF16 are supported)", what, p->type);
  if (p->n_seqs < 0 || p->n_q < 0 || p->n_kv < 0 || p->max_new < 0 || p->n_seqs > 65535)
    return set_error(B2Q_EINVAL, "%s: bad batch (%d sequences, %d queries, %d keys)", what, p->n_seqs, p->n_q, p->n_kv);
  if (!p->q_start || !p->kv_start) return set_error(B2Q_EINVAL, "%s: NULL offsets", what);
  if (p->n_q == 0 || p->n_seqs == 0) return B2Q_OK;  // (empty tensors have NULL addresses)
  s = check_rows(what, "q", q, q_stride, (int64_t)p->n_heads * D, t);
  if (s == B2Q_OK) s = check_rows(what, "out", out, (int64_t)p->n_heads * D, (int64_t)p->n_heads * D, t);
  if (s == B2Q_OK && p->n_kv) s = check_rows(what, "k", k, k_stride, (int64_t)p->n_kv_heads * D, t);
  if (s == B2Q_OK && p->n_kv) s = check_rows(what, "v", v, v_stride, (int64_t)p->n_kv_heads * D, t);
  if (s != B2Q_OK) return s;
  if (!(scale > 0.0f && scale <= 1e30f)) return set_error(B2Q_EINVAL, "%s: scale must be positive and at most 1e30", what);
  DeviceGuard dev(e->device);
  if (dev.err != cudaSuccess) return cuda_error(dev.err, what);
  PromptArgs a;
  a.H = p->n_heads;
  a.KV = p->n_kv_heads;
  a.n_seqs = p->n_seqs;
  a.n_q = p->n_q;
  a.n_kv = p->n_kv;
  a.q_start = p->q_start;
  a.kv_start = p->kv_start;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.scale = scale;
  a.out = out;
  a.G = a.H / a.KV;
  a.gp = std::min(a.G, 64);
  a.chunks = (a.G + a.gp - 1) / a.gp;
  a.tpt = kPrM / a.gp;
  CUtensorMap mq, mk, mv;
  bool maps = prompt_map_q(&mq, a, D, t);
  if (a.n_kv == 0) mk = mv = mq;  // (no tile is loaded, but the kernel prefetches all three)
  else maps = maps && prompt_map_kv(&mk, a.k, a.k_stride, a.n_kv, a.KV, D, t) && prompt_map_kv(&mv, a.v, a.v_stride, a.n_kv, a.KV, D, t);
  if (!maps)
    return set_error(B2Q_ECUDA, "%s: cuTensorMapEncodeTiled failed", what);
  // two row tiles to an item; one, in halves, where those are no more than the SMs
  // (16 tokens behind 2048: 22 us, 32 with room for a second row tile; with more items
  // than SMs two rounds of half the length gain nothing and load the keys twice)
  const int64_t hc = (int64_t)a.KV * a.chunks;
  a.nq = ((int64_t)(a.n_q / a.tpt) + a.n_seqs) * hc <= e->num_sms ? 1 : 2;
  const int64_t slots = (int64_t)(a.n_q / (a.nq * a.tpt)) + a.n_seqs;
  if (slots * hc > INT32_MAX - 4096) return set_error(B2Q_EINVAL, "%s: %d queries of %d heads in one call", what, a.n_q, a.H);
  a.slots = (int)slots;
  a.items = (int)(slots * hc);
  a.d_hc = fast_div((int)hc);
  a.d_chunks = fast_div(a.chunks);
  a.d_gp = fast_div(a.gp);
  a.d_bt = fast_div(a.nq * a.tpt);
  const unsigned grid = (unsigned)std::min<int64_t>(a.items, e->num_sms);
  cudaStream_t st = stream ? (cudaStream_t)stream : e->stream;
  cudaError_t err = cudaSuccess;
  by_dim(D, [&](auto d) {
    if (a.nq == 1)
      err = t == kElF16 ? launch_prompt<d(), kElF16, true>(a, mq, mk, mv, grid, e->device, st)
                        : launch_prompt<d(), kElBF16, true>(a, mq, mk, mv, grid, e->device, st);
    else
      err = t == kElF16 ? launch_prompt<d(), kElF16, false>(a, mq, mk, mv, grid, e->device, st)
                        : launch_prompt<d(), kElBF16, false>(a, mq, mk, mv, grid, e->device, st);
  });
  launch_counted(e, 1);
  return err == cudaSuccess ? B2Q_OK : cuda_error(err, what);
}

}  // extern "C"
