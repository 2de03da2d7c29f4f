// attn_prompt.cuh -- causal attention over packed prompts of different
// lengths, grouped heads, f16 or bf16:  query i of a sequence with n queries
// and l keys attends the keys j <= i + l - n.
//
// S = Q K^T and O += P V run on the 5th-generation tensor cores with their
// accumulators in TMEM.  A CTA takes two tiles of 128 query rows; a row is a
// (token, head) pair, the G heads of a K/V head side by side, so that a
// short prompt fills a tile and each K/V tile is fetched once for all of them.
// Over the key tiles (128 keys, K and V by TMA into a ring of 32 KB stages at
// D = 128) the two row tiles take turns: while one's scores go through the
// softmax the matrix unit works on the other's.
//   warps 0-3, 4-7  softmax of row tile 0 / 1: a thread owns a row, reads its
//                   128 scores out of TMEM, and writes the probabilities over
//                   them in the 16-bit type, where the P V product reads them;
//   warp 8          TMA;   warp 9  issues the matrix instructions;
//   warps 10, 11    look over the value tiles that some row sees only in part.
// The running maximum moves only when a row's grows by more than 2^8: until
// then probabilities up to 2^15 serve as well (they start at 2^7 for the largest,
// out of f16's subnormals), and the output in TMEM needs no rescaling.  When it
// does move, the softmax threads rescale the output themselves: the scores'
// completion covers the P V product issued before them.
// Values that no row may see reach no result: rows behind a sequence's end are
// zeroed in shared memory (0 * NaN is NaN), and where a tile with the causal
// edge holds an infinity or a NaN the CTA computes its rows again one key at a time.
#pragma once

#include <cuda.h>

#include "gemm_tc.cuh"
#include "kv_page.cuh"

namespace b2q {

struct PromptArgs {
  int H, KV, n_seqs, n_q, n_kv;
  const int32_t *q_start, *kv_start;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  float scale;
  void* out;
  // tiling: heads of a row tile side by side (at most G), chunks of them, tokens of a tile
  int G, gp, chunks, tpt;
};

constexpr int kPrThreads = 384, kPrM = 128, kPrN = 128;
__host__ __device__ constexpr int pr_tile_bytes(int D) { return 128 * D * 2; }  // of queries, keys or values
__host__ __device__ constexpr int pr_stages(int D) { return D == 128 ? 5 : 8; }
__host__ __device__ constexpr int pr_smem_bytes(int D) { return (2 + pr_stages(D)) * pr_tile_bytes(D) + 1024; }

// The offsets of one sequence, checked: queries [qa, qe), keys [ka, ke).
__device__ __forceinline__ bool prompt_seq(const PromptArgs& a, int s, int& qa, int& qe, int& ka, int& ke) {
  qa = a.q_start[s];
  qe = a.q_start[s + 1];
  ka = a.kv_start[s];
  ke = a.kv_start[s + 1];
  if (qe == qa) return false;
  if (qa < 0 || qe < qa || qe > a.n_q || ka < 0 || ke < ka || ke > a.n_kv) {
    if (qe > qa) kv_batch_error();
    return false;
  }
  return true;
}

// One row (a token's head) by a warp, one key at a time, from global memory.
template <int D, typename T>
__device__ __noinline__ void prompt_row_slow(const PromptArgs& a, int tok, int h, int ka, int last) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, kvh = h / a.G;
  float q[E], o[E], m = -INFINITY, sum = 0.0f;
  const T* qr = reinterpret_cast<const T*>(a.q) + (int64_t)tok * a.q_stride + h * D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = el_f(qr[lane + 32 * e]) * a.scale;
    o[e] = 0.0f;
  }
  for (int j = 0; j <= last; ++j) {
    const T* kr = reinterpret_cast<const T*>(a.k) + (int64_t)(ka + j) * a.k_stride + kvh * D;
    const T* vr = reinterpret_cast<const T*>(a.v) + (int64_t)(ka + j) * a.v_stride + kvh * D;
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
  T* orow = reinterpret_cast<T*>(a.out) + ((int64_t)tok * a.H + h) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) orow[lane + 32 * e] = el_from<T>(sum == 0.0f ? 0.0f : o[e] / sum);
}

// ---- tensor copies, matrix and TMEM instructions ----
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// Operand descriptors of tiles with rows of 64 elements (128 bytes, 128-byte
// swizzle, groups of 8 rows every 1024 bytes).  K-major (queries, keys): the
// products run along the row; a k16 step is 32 bytes further.  MN-major
// (values): the products run over the rows, a k16 step is 16 rows further, and
// the next 64 columns lie `lbo` bytes behind.
__device__ __forceinline__ uint64_t pr_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
__host__ __device__ constexpr uint32_t pr_idesc(bool bf16, int N, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(kPrM >> 4) << 24);
}
__device__ __forceinline__ void pr_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pr_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pr_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 32 columns of the warp's 32 TMEM lanes: a thread's row
__device__ __forceinline__ void pr_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void pr_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void pr_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pr_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float pr_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kPrLag = 8.0f;    // (log2) growth of a row's maximum that is let pass
constexpr float kPrShift = 7.0f;  // (log2) the largest probability at a fresh maximum

template <int D, int TYPE>
__global__ void __launch_bounds__(kPrThreads, 1) attn_prompt_kernel(const __grid_constant__ PromptArgs a,
                                                                    const __grid_constant__ CUtensorMap mq,
                                                                    const __grid_constant__ CUtensorMap mk,
                                                                    const __grid_constant__ CUtensorMap mv) {
  typedef typename Elem<TYPE>::type T;
  constexpr int NS = pr_stages(D), TB = pr_tile_bytes(D), CB = 128 * 128;  // bytes of a 64-column chunk of a tile
  constexpr int NC = D / 64;
  constexpr bool BF = TYPE == kElBF16;
  extern __shared__ uint8_t pr_smem[];
  __shared__ uint64_t q_full[2], full[NS], empty[NS], v_land[NS], s_full[2], p_full[2], o_full[2], v_ok[NS];
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail_, s_poison_;
  volatile int *s_fail = &s_fail_, *s_poison = &s_poison_;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pr_smem) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = base;
  uint8_t* ring = base + 2 * TB;

  pdl_wait();
  pdl_launch_dependents();

  // ---- which rows: blocks of 2 tpt tokens; sequence s owns the slots from
  // q_start[s] / (2 tpt) + s on (increasing in s, and enough for its blocks) ----
  const int bt = 2 * a.tpt, hc = a.KV * a.chunks;
  const int slots = a.n_q / bt + a.n_seqs;
  const int slot = slots - 1 - (int)(blockIdx.x / hc);  // late blocks, which see the most keys, first
  const int kvh = (int)(blockIdx.x % hc) / a.chunks, hoff = ((int)(blockIdx.x % hc) % a.chunks) * a.gp;
  int lo = 0, hi = a.n_seqs - 1;  // the last s with q_start[s] / bt + s <= slot
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.q_start[mid] / bt + mid <= slot) lo = mid;
    else hi = mid - 1;
  }
  int qa, qe, ka, ke;
  if (!prompt_seq(a, lo, qa, qe, ka, ke)) return;
  const int blk = slot - (qa / bt + lo), n = qe - qa, l = ke - ka;
  const long long tok0l = (long long)blk * bt;  // first token of the block within the sequence
  if (blk < 0 || tok0l >= n) return;
  const int tok0 = (int)tok0l;
  const int diff = l - n;  // token i attends the keys up to i + diff
  const int tok_last = min(n, tok0 + bt) - 1;
  const int kmax = max(0, tok_last + diff + 1);  // keys of the block's last token
  const int nt = (kmax + kPrN - 1) / kPrN;
  const int first_lim = tok0 + diff;
  const int kt_edge = first_lim < 0 ? 0 : (first_lim + 1) / kPrN;  // the first tile that not every row sees whole

  // Value tiles from kt_edge on land on barriers of their own, which the lookers
  // follow without the uses of the ring before them; their stage's full
  // barrier is passed at once.  v_land and v_ok are per stage, so that neither can
  // run a phase ahead of whom it wakes.  Phase of use x: the earlier ones of its stage.
  auto land_phase = [&](int x) { return (uint32_t)((x - (2 * kt_edge + 1)) / (NS & 1 ? 2 * NS : NS)) & 1u; };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&v_land[i], 1);
      mbar_init(&v_ok[i], 2);
    }
    *s_fail = 0;
    *s_poison = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;  // columns: S0, S1 (128 each), O0, O1

  float sum = 0.0f;  // softmax threads: their row's
  if (warp < 8) {
    // ---- softmax of row tile i ----
    const int i = warp >> 2, r = threadIdx.x & 127;
    const int tok = tok0 + i * a.tpt + r / a.gp;
    const int lim = min(tok + diff, kmax - 1);
    const int edge = tok0 + i * a.tpt + diff;  // the tile's first token's last key
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_base + i * 128, to = tmem + lane_base + 256 + i * D;
    const float c = a.scale * 1.4426950408889634f;
    float ref = -INFINITY;  // (scores times c)
    for (int j = 0; j < nt; ++j) {
      if (!__all_sync(B2Q_FULL, mbar_wait_bounded(&s_full[i], j & 1)) || *s_fail) {
        *s_fail = 1;
        break;
      }
      tc_fence_after();
      uint32_t s[128];
      pr_ld32(ts, s);
      pr_ld32(ts + 32, s + 32);
      pr_ld32(ts + 64, s + 64);
      pr_ld32(ts + 96, s + 96);
      pr_wait_ld();
      if (j * kPrN + kPrN - 1 > edge) {
        const int lc = lim - j * kPrN;  // the row's last column
#pragma unroll
        for (int x = 0; x < 128; ++x)
          if (x > lc) s[x] = 0xff800000u;
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int x = 0; x < 128; ++x) m4[x & 3] = fmaxf(m4[x & 3], __uint_as_float(s[x]));
      const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * c;
      const bool move = m > ref + kPrLag;  // (from -inf: any finite maximum)
      if (__any_sync(B2Q_FULL, move)) {
        const float al = move ? (ref == -INFINITY ? 0.0f : pr_exp2(ref - m)) : 1.0f;
        if (move) ref = m;
        sum *= al;
        if (j > 0) {
#pragma unroll
          for (int x = 0; x < D; x += 32) {
            uint32_t o[32];
            pr_ld32(to + x, o);
            pr_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * al);
            pr_st32(to + x, o);
          }
          pr_wait_st();
        }
      }
      const float off = ref == -INFINITY ? 0.0f : kPrShift - ref;
      float t4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t p[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          const float e0 = pr_exp2(fmaf(__uint_as_float(s[64 * h + 2 * x]), c, off));
          const float e1 = pr_exp2(fmaf(__uint_as_float(s[64 * h + 2 * x + 1]), c, off));
          t4[x & 1] += e0;
          t4[2 + (x & 1)] += e1;
          p[x] = el_pack2<T>(e0, e1);
        }
        pr_st32(ts + 32 * h, p);
      }
      sum += (t4[0] + t4[1]) + (t4[2] + t4[3]);
      pr_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i]);
    }
  } else if (warp == 8) {
    // ---- TMA: Q0, K0, Q1, V0, K1, V1, ... ----
    if (lane == 0) {
      const uint32_t qbytes = (uint32_t)(a.tpt * a.gp * 128 * NC);
      int issued = 0;
      auto load_q = [&](int i) {
        mbar_arrive_expect_tx(&q_full[i], qbytes);
        for (int cnk = 0; cnk < NC; ++cnk)
          tma_load_4d(qs + i * TB + cnk * CB, &mq, cnk * 64, hoff, kvh, qa + tok0 + i * a.tpt, &q_full[i]);
      };
      bool ok = true;
      if (nt > 0) load_q(0);
      for (int x = 0; x < 2 * nt; ++x) {
        const int st = x % NS;
        if (x >= NS && !mbar_wait_bounded(&empty[st], ((x / NS) - 1) & 1)) {
          ok = false;
          break;
        }
        if (*s_fail) {
          ok = false;
          break;
        }
        const bool look = (x & 1) && (x >> 1) >= kt_edge;
        uint64_t* bar = look ? &v_land[st] : &full[st];
        mbar_arrive_expect_tx(bar, (uint32_t)TB);
        for (int cnk = 0; cnk < NC; ++cnk)
          tma_load_3d(ring + st * TB + cnk * CB, (x & 1) ? &mv : &mk, cnk * 64, kvh, ka + (x >> 1) * kPrN, bar);
        if (look) mbar_arrive(&full[st]);
        ++issued;
        if (x == 0) load_q(1);
      }
      // copies in flight land before the CTA may end
      if (!ok) *s_fail = 1;
      if (nt > 0) mbar_wait_bounded(&q_full[0], 0);
      if (issued > 0) mbar_wait_bounded(&q_full[1], 0);
      for (int x = max(0, issued - NS); x < issued; ++x) {
        if ((x & 1) && (x >> 1) >= kt_edge) mbar_wait_bounded(&v_land[x % NS], land_phase(x));
        else mbar_wait_bounded(&full[x % NS], (x / NS) & 1);
      }
    }
  } else if (warp == 9) {
    // ---- matrix instructions ----
    if (lane == 0 && nt > 0) {
      constexpr uint32_t id_s = pr_idesc(BF, kPrN, false), id_o = pr_idesc(BF, D, true);
      bool ok = true;
      auto scores = [&](int i, int st) {  // S_i = Q_i K^T
        const uint32_t q0 = smem_u32(qs + i * TB), k0 = smem_u32(ring + st * TB);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = (k >> 2) * CB + (k & 3) * 32;
          pr_mma_ss(tmem + i * 128, pr_desc(q0 + o, 16), pr_desc(k0 + o, 16), id_s, k > 0);
        }
        pr_commit(&s_full[i]);
      };
      ok = mbar_wait_bounded(&q_full[0], 0) && mbar_wait_bounded(&full[0], 0);
      if (ok) {
        tc_fence_after();
        scores(0, 0);
        ok = mbar_wait_bounded(&q_full[1], 0);
        if (ok) {
          scores(1, 0);
          pr_commit(&empty[0]);
        }
      }
      for (int j = 0; ok && j < nt; ++j) {
        const int xv = 2 * j + 1, xk = 2 * j + 2, sv = xv % NS, sk = xk % NS;
        const bool more = j + 1 < nt;
        ok = mbar_wait_bounded(&full[sv], (xv / NS) & 1);
        if (ok && j >= kt_edge) ok = mbar_wait_bounded(&v_ok[sv], land_phase(xv));
        if (ok && more) ok = mbar_wait_bounded(&full[sk], (xk / NS) & 1);
        for (int i = 0; ok && i < 2; ++i) {
          ok = mbar_wait_bounded(&p_full[i], j & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t v0 = smem_u32(ring + sv * TB);
#pragma unroll
          for (int k = 0; k < kPrN / 16; ++k)
            pr_mma_ts(tmem + 256 + i * D, tmem + i * 128 + k * 8, pr_desc(v0 + k * 2048, CB), id_o, j > 0 || k > 0);
          if (more) scores(i, sk);
          else pr_commit(&o_full[i]);
        }
        if (ok) {
          pr_commit(&empty[sv]);
          if (more) pr_commit(&empty[sk]);
        }
      }
      if (!ok) {
        *s_fail = 1;
        pr_commit(&o_full[0]);  // (whatever was issued completes before the TMEM is freed)
        pr_commit(&o_full[1]);
      }
    }
  } else {
    // ---- value tiles that some row sees only in part ----
    const int w = threadIdx.x - 320;  // 0..63: rows w and w + 64
    for (int j = kt_edge; j < nt; ++j) {
      const int x = 2 * j + 1;
      if (!__all_sync(B2Q_FULL, mbar_wait_bounded(&v_land[x % NS], land_phase(x))) || *s_fail) {
        *s_fail = 1;
        break;
      }
      uint8_t* vt = ring + (x % NS) * TB;
      bool bad = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = w + 64 * h;
        if (j * kPrN + row >= l) {  // behind the sequence
          for (int y = 0; y < 8 * NC; ++y)
            *reinterpret_cast<uint4*>(vt + (y >> 3) * CB + row * 128 + ((y ^ row) & 7) * 16) = make_uint4(0, 0, 0, 0);
        } else {
          // an infinity or NaN has all exponent bits set
          constexpr uint32_t em = BF ? 0x7f80u : 0x7c00u;
          for (int y = 0; y < 8 * NC; ++y) {
            const uint4 v = *reinterpret_cast<const uint4*>(vt + (y >> 3) * CB + row * 128 + ((y ^ row) & 7) * 16);
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int z = 0; z < 4; ++z) bad = bad || (u[z] & em) == em || (u[z] & (em << 16)) == (em << 16);
          }
        }
      }
      if (__any_sync(B2Q_FULL, bad)) *s_poison = 1;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_ok[x % NS]);
    }
  }

  __syncwarp();

  // ---- epilogue ----
  if (warp < 8) {
    const int i = warp >> 2;
    if (nt > 0 && !__all_sync(B2Q_FULL, mbar_wait_bounded(&o_full[i], 0))) *s_fail = 1;
    tc_fence_after();
  }
  __syncthreads();
  if (warp < 8 && !*s_fail) {
    const int i = warp >> 2, r = threadIdx.x & 127;
    const int tr = r / a.gp, hg = hoff + r - tr * a.gp, tok = tok0 + i * a.tpt + tr;
    const bool live = tr < a.tpt && tok < n && hg < a.G;
    const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 256 + i * D;
    if (*s_poison) {
      for (int y = 0; y < 32; ++y) {
        if (!__shfl_sync(B2Q_FULL, (int)live, y)) continue;
        const int tk = __shfl_sync(B2Q_FULL, tok, y), hh = __shfl_sync(B2Q_FULL, hg, y);
        prompt_row_slow<D, T>(a, qa + tk, kvh * a.G + hh, ka, tk + diff);
      }
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      T* orow = reinterpret_cast<T*>(a.out) + ((int64_t)(qa + tok) * a.H + kvh * a.G + hg) * D;
#pragma unroll
      for (int x = 0; x < D; x += 32) {
        uint32_t o[32];
        if (nt > 0) {
          pr_ld32(to + x, o);
          pr_wait_ld();
        }
        uint32_t p[16];
#pragma unroll
        for (int y = 0; y < 16; ++y)
          p[y] = nt > 0 ? el_pack2<T>(__uint_as_float(o[2 * y]) * inv, __uint_as_float(o[2 * y + 1]) * inv) : 0u;
        if (live) {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            reinterpret_cast<uint4*>(orow + x)[y] = make_uint4(p[4 * y], p[4 * y + 1], p[4 * y + 2], p[4 * y + 3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace b2q
