// attn_paged.cuh -- attention of the newest tokens of many sequences over
// their keys and values in the paged 4-bit cache (kv_page.cuh):
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - max),  j <= position.
#pragma once

#include "kv_page.cuh"

namespace b2q {

struct PagedArgs {
  KvBatch b;
  int H;
  const void* q;
  int64_t q_stride;
  const uint8_t* pages;
  float scale;
  void* out;
};

// One warp per query row (token, head), one key at a time.
template <int D, int QT, int OT>
__global__ void __launch_bounds__(128) attn_paged_kernel(const __grid_constant__ PagedArgs a) {
  typedef typename Elem<QT>::type Q;
  typedef typename Elem<OT>::type O;
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(row / a.H), h = (int)(row % a.H), kvh = h / (a.H / a.b.KV);
  if (t >= a.b.n_tokens) return;
  int seq, pos;
  if (!kv_row_of(a.b, t, seq, pos)) return;
  const int cap = a.b.max_pages * a.b.page_tokens;
  if (pos < 0 || pos >= cap) kv_batch_error();
  pos = min(pos, cap - 1);
  float q[E], o[E], m = -INFINITY, sum = 0.0f;
  const Q* qr = reinterpret_cast<const Q*>(a.q) + (int64_t)t * a.q_stride + h * D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = el_f(qr[lane + 32 * e]) * a.scale;
    o[e] = 0.0f;
  }
  const int bpp = a.b.page_tokens / kKvBlk;
  for (int j0 = 0; j0 <= pos; j0 += kKvBlk) {
    int64_t blk = kv_block_of(a.b, seq, j0);
    if (blk < 0) continue;
    const uint8_t* bp = a.pages + (blk + (int64_t)kvh * bpp) * kv_blk_bytes(D);
    for (int j = j0; j <= min(pos, j0 + kKvBlk - 1); ++j) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], kv_key_at(bp, D, j - j0, lane + 32 * e), s);
      s = warp_sum(s);
      const float nm = fmaxf(m, s), al = expf(m - nm), p = expf(s - nm);
      m = nm;
      sum = sum * al + p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(p, kv_value_at(bp, D, j - j0, lane + 32 * e), o[e] * al);
    }
  }
  O* orow = reinterpret_cast<O*>(a.out) + ((int64_t)t * a.H + h) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) orow[lane + 32 * e] = el_from<O>(sum == 0.0f ? 0.0f : o[e] / sum);
}

}  // namespace b2q
