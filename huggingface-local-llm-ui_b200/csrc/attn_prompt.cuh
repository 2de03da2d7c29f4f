// attn_prompt.cuh -- causal attention over packed prompts of different
// lengths, grouped heads, f16 or bf16:  query i of a sequence with n queries
// and l keys attends the keys j <= i + l - n.
#pragma once

#include "kv_page.cuh"

namespace b2q {

struct PromptArgs {
  int H, KV, n_seqs, n_q, n_kv;
  const int32_t *q_start, *kv_start;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  float scale;
  void* out;
};

// Sequence of packed query row t: its queries [qa, qe), keys [ka, ke).
// False behind the last sequence, and (with the error word) for offsets
// that make no sense.
__device__ __forceinline__ bool prompt_seq_of(const PromptArgs& a, int t, int& qa, int& qe, int& ka, int& ke) {
  int lo = 0, hi = a.n_seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.q_start[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= a.n_seqs) return false;
  qa = a.q_start[lo];
  qe = a.q_start[lo + 1];
  ka = a.kv_start[lo];
  ke = a.kv_start[lo + 1];
  if (qa < 0 || t < qa || t >= qe || qe > a.n_q || ka < 0 || ke < ka || ke > a.n_kv) {
    kv_batch_error();
    return false;
  }
  return true;
}

// One warp per query row (token, head), one key at a time.
template <int D, int T>
__global__ void __launch_bounds__(128) attn_prompt_kernel(const __grid_constant__ PromptArgs a) {
  typedef typename Elem<T>::type E_t;
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(row / a.H), h = (int)(row % a.H), kvh = h / (a.H / a.KV);
  if (t >= a.n_q) return;
  int qa, qe, ka, ke;
  if (!prompt_seq_of(a, t, qa, qe, ka, ke)) return;
  const int last = t - qa + (ke - ka) - (qe - qa);  // the row's last key
  float q[E], o[E], m = -INFINITY, sum = 0.0f;
  const E_t* qr = reinterpret_cast<const E_t*>(a.q) + (int64_t)t * a.q_stride + h * D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = el_f(qr[lane + 32 * e]) * a.scale;
    o[e] = 0.0f;
  }
  for (int j = 0; j <= last; ++j) {
    const E_t* kr = reinterpret_cast<const E_t*>(a.k) + (int64_t)(ka + j) * a.k_stride + kvh * D;
    const E_t* vr = reinterpret_cast<const E_t*>(a.v) + (int64_t)(ka + j) * a.v_stride + kvh * D;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], el_f(kr[lane + 32 * e]), s);
    s = warp_sum(s);
    const float nm = fmaxf(m, s), al = expf(m - nm), p = expf(s - nm);
    m = nm;
    sum = sum * al + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(p, el_f(vr[lane + 32 * e]), o[e] * al);
  }
  E_t* orow = reinterpret_cast<E_t*>(a.out) + ((int64_t)t * a.H + h) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) orow[lane + 32 * e] = el_from<E_t>(sum == 0.0f ? 0.0f : o[e] / sum);
}

}  // namespace b2q
