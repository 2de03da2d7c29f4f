// attn_prompt.cuh -- causal attention over packed prompts of different
// lengths, grouped heads, f16 or bf16:  query i of a sequence with n queries
// and l keys attends the keys j <= i + l - n.
//
// S = Q K^T and O += P V run on the 5th-generation tensor cores with their
// accumulators in TMEM.  An item is two tiles of 128 query rows of a K/V head; a
// row is a (token, head) pair, the G heads of a K/V head side by side, so that a
// short prompt fills a tile and each K/V tile is fetched once for all of them.
// Over the key tiles (128 keys, K and V by TMA into a ring of 32 KB stages at D =
// 128) the two row tiles take turns: while one's scores go through the softmax the
// matrix unit works on the other's.  Where that leaves SMs without an item, an
// item is one row tile, and the CTA's halves take its key tiles in turn, each with a
// running softmax and an output of its own, joined at the end (HALVES).  One CTA
// an SM goes from item to item, the next item's loads and first scores under the
// last one's epilogue.
//   warps 0-3, 4-7  softmax of row tile 0 / 1, or of even / odd key tiles: a
//                   thread owns a row, reads its 128 scores out of TMEM, and
//                   writes the probabilities over them in the 16-bit type, where
//                   the P V product reads them;
//   warp 8          TMA;   warp 9  issues the matrix instructions;
//   warps 10, 11    look over the value tiles that some row sees only in part.
// What bounds it: the matrix unit (16 instructions of 64 cycles for each row tile
// and 128 keys, more like 90 with the softmax's TMEM traffic beside them) and, close
// behind, a softmax of 1640 cycles that has to be done when the other row tile's
// products are.  Measured at 8192 tokens of 64 heads, 900 us (1.22 PFLOP/s): keeping
// the issuing warp converged, with one elected thread, 981 -> 910 us (a branch on the
// lane moved every descriptor between register files); the next item's geometry
// under the last product and stores of 64 consecutive bytes, 910 -> 893 (16 ragged
// prompts 172 -> 157); the look at an edge tile as a sum of 0 * value, which the last
// product of every item waits for, 512 tokens 12.9 -> 11.7, the ragged prompts 159 ->
// 155.  That is a burst; where the power cap holds the clock at 1.6 to 1.7 GHz it takes
// 1050 to 1090.  16 tokens behind 2048, 32 heads over 8: 22 us in halves, 32.5 without
// (512 tokens behind 2048: 27 and 39).  Tried on the 984 us form: a
// quarter of the exponentials by a polynomial on the FMA units, 1040; two threads to
// a row, 1027; key tiles of 64 with two score buffers, 1270 (a score product of 64
// keys takes as long as one of 128: its A operand's trip from shared memory).
// The running maximum moves only when a row's grows by more than 2^8: until
// then probabilities up to 2^15 serve as well (they start at 2^7 for the largest,
// out of f16's subnormals), and the output in TMEM needs no rescaling.  When it
// does move, the softmax threads rescale the output themselves: the scores'
// completion covers the P V product issued before them.
// Values that a row must not see reach no result (0 * NaN is NaN): in the tiles with the
// causal edge the rows behind a sequence's end, infinities and NaN are zeroed in shared
// memory; the rows that do see one of those get it at their end (prompt_show_bad).
#pragma once

#include <cuda.h>

#include <climits>

#include "attn_paged.cuh"
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
  // items: slots of nq * tpt tokens (nq row tiles) x K/V heads and chunks, late slots first
  int nq, slots, items;
  FastDiv d_hc, d_chunks, d_gp, d_bt;
};

constexpr int kPrThreads = 384, kPrM = 128, kPrN = 128;
__host__ __device__ constexpr int pr_tile_bytes(int D) { return 128 * D * 2; }  // of queries, keys or values
__host__ __device__ constexpr int pr_stages(int D) { return D == 128 ? 5 : 8; }
__host__ __device__ constexpr int pr_smem_bytes(int D) { return (2 + pr_stages(D)) * pr_tile_bytes(D) + 1024; }

// Values that are not finite among the keys k0 .. k1 - 1 of the key tiles that not every
// row sees whole (there the products took them as zeros): each shows in the rows of the
// warp that see its key.  The lane's row is `row` (elements from the start of out, < 0:
// none), its last key `lim`; columns x0 .. x1 - 1 of the head.  A lane looks over the
// columns lane + 32 e: what matters of one is its first key with +inf and its first with
// -inf, NaN counting as both, so that the cost is that of reading the tiles once.
template <int D, typename T>
__device__ __noinline__ void prompt_show_bad(const PromptArgs& a, int ka, int kvh, int k0, int k1, int64_t row, int lim, int x0, int x1) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  int up[E], down[E];
#pragma unroll
  for (int e = 0; e < E; ++e) up[e] = down[e] = INT_MAX;
  const T* v = reinterpret_cast<const T*>(a.v) + kvh * D + lane;
#pragma unroll 4
  for (int j = k0; j < k1; ++j) {
    const T* vr = v + (int64_t)(ka + j) * a.v_stride;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float f = el_f(vr[32 * e]);
      if (!(f < INFINITY)) up[e] = min(up[e], j);
      if (!(f > -INFINITY)) down[e] = min(down[e], j);
    }
  }
  __syncwarp();  // the rows' stores come first
  for (int y = 0; y < 32; ++y) {
    const int64_t r = __shfl_sync(B2Q_FULL, row, y);
    const int l = __shfl_sync(B2Q_FULL, lim, y);
    if (r < 0) continue;
    T* o = reinterpret_cast<T*>(a.out) + r + lane;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool u = up[e] <= l, d = down[e] <= l;
      if ((u || d) && lane + 32 * e >= x0 && lane + 32 * e < x1) {
        const float was = el_f(o[32 * e]);  // (+inf and -inf: NaN; NaN stays)
        o[32 * e] = el_from<T>(was + (u ? d ? INFINITY - INFINITY : INFINITY : -INFINITY));
      }
    }
  }
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
// True in one thread of the (converged) warp, the same every time.
__device__ __forceinline__ bool pr_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
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

__device__ __forceinline__ float pr_max3(float a, float b, float c) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// a * b + c of pairs of 16-bit numbers
template <bool BF>
__device__ __forceinline__ uint32_t pr_fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  if (BF) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// A lane gives `b` (`odd`: `a`) and takes what its partner gives in the place.
__device__ __forceinline__ void pr_swap(bool odd, int mask, uint4& a, uint4& b) {
  uint32_t *x = &a.x, *y = &b.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t got = __shfl_xor_sync(B2Q_FULL, odd ? x[i] : y[i], mask);
    (odd ? x[i] : y[i]) = got;
  }
}

constexpr float kPrLag = 8.0f;    // (log2) growth of a row's maximum that is let pass
constexpr float kPrShift = 7.0f;  // (log2) the largest probability at a fresh maximum

// Two f32 in a register pair.
typedef unsigned long long f2;
__device__ __forceinline__ f2 f2_of(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f2 f2_of(uint32_t a, uint32_t b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void f2_to(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// One item's geometry.
struct PrItem {
  int qa, ka, n, l;  // of the sequence: first query and key row, queries, keys
  int tok0;          // first token of the item within the sequence
  int nq;            // row tiles with tokens
  int nt, kt_edge;   // key tiles, the first of them that not every row sees whole
  int kvh, hoff;     // K/V head, first head of the group
};

constexpr int kPrSeqs = 192;  // sequences whose offsets are copied to shared memory

template <int D, int TYPE, bool HALVES>
__global__ void __launch_bounds__(kPrThreads, 1) attn_prompt_kernel(const __grid_constant__ PromptArgs a,
                                                                    const __grid_constant__ CUtensorMap mq,
                                                                    const __grid_constant__ CUtensorMap mk,
                                                                    const __grid_constant__ CUtensorMap mv) {
  typedef typename Elem<TYPE>::type T;
  constexpr int NS = pr_stages(D), TB = pr_tile_bytes(D), CB = 128 * 128;  // bytes of a 64-column chunk of a tile
  constexpr int NC = D / 64;
  constexpr bool BF = TYPE == kElBF16;
  extern __shared__ uint8_t pr_smem[];
  __shared__ uint64_t q_full[2], q_empty[2], full[NS], empty[NS], v_land[NS], v_ok[NS], s_full[2], p_full[2], o_full[2], x_full, done;
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail_, s_poison_[16], s_q[kPrSeqs + 1], s_k[kPrSeqs + 1];
  volatile int *s_fail = &s_fail_, *s_poison = s_poison_;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pr_smem) + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = base;
  uint8_t* ring = base + 2 * TB;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
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
    mbar_init(&x_full, 8);
    mbar_init(&done, 1);
    *s_fail = 0;
    for (int i = 0; i < 16; ++i) s_poison[i] = 0;
    fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  const bool cached = a.n_seqs <= kPrSeqs;
  if (cached)
    for (int i = threadIdx.x; i <= a.n_seqs; i += kPrThreads) {
      s_q[i] = a.q_start[i];
      s_k[i] = a.kv_start[i];
    }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;  // columns: S0, S1 (128 each), O0, O1

  // ---- items: slots of bt tokens, of which sequence s owns those from
  // q_start[s] / bt + s on (increasing in s, and enough for it).  CTA b takes b,
  // then goes back and forth: late slots, which see the most keys, come first,
  // and what one round gives a CTA too much the next takes from it ----
  constexpr int NQ = HALVES ? 1 : 2, step = HALVES ? 2 : 1;  // row tiles of an item; from a half's key tile to its next
  const int bt = NQ * a.tpt;
  auto item = [&](int round, PrItem& it) {  // false: nothing to do
    const int x = round * (int)gridDim.x + ((round & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
    if (x >= a.items) return false;
    const int sr = fdiv(x, a.d_hc), hx = x - sr * a.d_hc.d, slot = a.slots - 1 - sr;
    it.kvh = fdiv(hx, a.d_chunks);
    it.hoff = (hx - it.kvh * a.chunks) * a.gp;
    int lo = 0, hi = a.n_seqs - 1;  // the last s with q_start[s] / bt + s <= slot
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      const int qm = cached ? s_q[mid] : a.q_start[mid];
      if (qm < 0 || fdiv(qm, a.d_bt) + mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    const int qa = cached ? s_q[lo] : a.q_start[lo], qe = cached ? s_q[lo + 1] : a.q_start[lo + 1];
    const int ka = cached ? s_k[lo] : a.kv_start[lo], ke = cached ? s_k[lo + 1] : a.kv_start[lo + 1];
    if (qe == qa) return false;
    if (qa < 0 || qe < qa || qe > a.n_q || ka < 0 || ke < ka || ke > a.n_kv) {
      if (qe > qa) kv_batch_error();
      return false;
    }
    const int blk = slot - (fdiv(qa, a.d_bt) + lo);
    const long long tok0 = (long long)blk * bt;
    if (blk < 0 || tok0 >= qe - qa) return false;
    it.qa = qa;
    it.ka = ka;
    it.n = qe - qa;
    it.l = ke - ka;
    it.tok0 = (int)tok0;
    it.nq = !HALVES && it.tok0 + a.tpt < it.n ? 2 : 1;
    const int diff = it.l - it.n;  // token i attends the keys up to i + diff
    const int kmax = max(0, min(it.n, it.tok0 + bt) + diff);
    it.nt = (kmax + kPrN - 1) / kPrN;
    const int lim = it.tok0 + diff;
    it.kt_edge = lim < 0 ? 0 : (lim + 1) / kPrN;
    return true;
  };
  // (in halves there are no more items than CTAs)
  const int rounds = HALVES ? 1 : (a.items + (int)gridDim.x - 1) / (int)gridDim.x;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- softmax of row tile i, or of every second key tile ----
    const int i = warp >> 2, ir = HALVES ? 0 : i, r = threadIdx.x & 127;
    float2* s_stat = reinterpret_cast<float2*>(qs + TB);  // [2][128] (halves: no second query tile): reference, sum
    const int tr = fdiv(r, a.d_gp), hr = r - tr * a.gp;  // the row's token and head within the tile
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_base + i * 128, to = tmem + lane_base + 256 + i * D;
    const float c = a.scale * 1.4426950408889634f;
    const f2 c2 = f2_of(c, c);
    uint32_t s_ph = 0, o_ph = 0;
    int count = 0;  // items with key tiles and this row tile
    bool ok = true;
    int round = -1;
    auto next_item = [&](PrItem& it) {  // the next item with this row tile
      while (++round < rounds) {
        if (!item(round, it)) continue;
        if (ir >= it.nq) continue;
        if (it.nt > 0) ++count;
        return true;
      }
      return false;
    };
    PrItem it;
    bool more = next_item(it);
    while (ok && more) {
      const int mine = count;  // (the item's)
      const int diff = it.l - it.n, tok = it.tok0 + ir * a.tpt + tr, h = it.hoff + hr;
      const bool live = tr < a.tpt && tok < it.n && h < a.G;
      const int lim = min(tok + diff, it.l - 1);          // the row's last key
      const int edge = it.tok0 + ir * a.tpt + diff;       // the tile's first token's
      float ref = -INFINITY, sum = 0.0f;                  // (scores times c)
      for (int j = HALVES ? i : 0; j < it.nt; j += step) {
        ok = __all_sync(B2Q_FULL, mbar_wait_bounded(&s_full[i], s_ph)) && !*s_fail;
        if (!ok) break;
        s_ph ^= 1;
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
        for (int x = 0; x < 128; x += 8)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            m4[y] = pr_max3(m4[y], __uint_as_float(s[x + 2 * y]), __uint_as_float(s[x + 2 * y + 1]));
        const float m = pr_max3(pr_max3(m4[0], m4[1], m4[2]), m4[3], m4[3]) * c;
        if (!(m < INFINITY)) sum = __uint_as_float(0x7fffffffu);  // a score that is NaN or +inf: so is the row
        const bool move = m > ref + kPrLag;  // (from -inf: any finite maximum)
        if (__any_sync(B2Q_FULL, move)) {
          const float al = move ? (ref == -INFINITY ? 0.0f : pr_exp2(ref - m)) : 1.0f;
          if (move) ref = m;
          sum *= al;
          if (j >= step) {
#pragma unroll 1
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
        const f2 off2 = f2_of(off, off);
        f2 t0 = f2_of(0.0f, 0.0f), t1 = t0;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t p[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const f2 y = f2_fma(f2_of(s[64 * hh + 2 * x], s[64 * hh + 2 * x + 1]), c2, off2);
            float e0, e1;
            f2_to(y, e0, e1);
            e0 = pr_exp2(e0);
            e1 = pr_exp2(e1);
            if (x & 1) t1 = f2_add(t1, f2_of(e0, e1));
            else t0 = f2_add(t0, f2_of(e0, e1));
            p[x] = el_pack2<T>(e0, e1);
          }
          pr_st32(ts + 32 * hh, p);
        }
        float u0, u1;
        f2_to(f2_add(t0, t1), u0, u1);
        sum += u0 + u1;
        pr_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[i]);
      }
      if (!ok) break;
      // ---- epilogue: the next item's geometry under the last product ----
      PrItem nx;
      more = next_item(nx);
      float w0 = 1.0f, w1 = 0.0f;  // weights of the halves' outputs
      if (it.nt > 0) {
        // (in halves both outputs; a second one where there are two key tiles)
        ok = __all_sync(B2Q_FULL, mbar_wait_bounded(&o_full[ir], o_ph)) && !*s_fail;
        o_ph ^= 1;
        if (HALVES && ok && it.nt > 1) ok = __all_sync(B2Q_FULL, mbar_wait_bounded(&o_full[1], 0)) && !*s_fail;
        if (!ok) break;
        tc_fence_after();
        if (HALVES) {
          s_stat[128 * i + r] = make_float2(ref, sum);
          __syncwarp();
          if (lane == 0) mbar_arrive(&x_full);
          ok = __all_sync(B2Q_FULL, mbar_wait_bounded(&x_full, 0)) && !*s_fail;
          if (!ok) break;
          const float2 st0 = s_stat[r], st1 = s_stat[128 + r];
          const float top = fmaxf(st0.x, st1.x);
          w0 = st0.x == -INFINITY ? 0.0f : pr_exp2(st0.x - top);
          w1 = st1.x == -INFINITY ? 0.0f : pr_exp2(st1.x - top);
          sum = w0 * st0.y + w1 * st1.y;
        }
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      // four lanes exchange 16-byte pieces, so that each store writes 64
      // consecutive bytes of a row: lane y of the four piece y of all four rows
      const long long at = live ? ((long long)(it.qa + tok) * a.H + it.kvh * a.G + h) * D : -1;
      long long rows[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) rows[k] = __shfl_sync(B2Q_FULL, at, (lane & 28) + k);
      const bool b0 = lane & 1, b1 = lane & 2;
      const int xa = HALVES ? i * (D / 2) : 0, xe = HALVES ? xa + D / 2 : D;
#pragma unroll 1
      for (int x = xa; x < xe; x += 32) {
        uint4 v[4];
        if (it.nt > 0) {
          uint32_t o[32];
          pr_ld32((HALVES ? tmem + lane_base + 256 : to) + x, o);
          pr_wait_ld();
          if (HALVES) {
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * w0);
            if (it.nt > 1) {
              uint32_t o1[32];
              pr_ld32(tmem + lane_base + 256 + D + x, o1);
              pr_wait_ld();
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(fmaf(__uint_as_float(o1[y]), w1, __uint_as_float(o[y])));
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              w[y] = el_pack2<T>(__uint_as_float(o[8 * k + 2 * y]) * inv, __uint_as_float(o[8 * k + 2 * y + 1]) * inv);
            v[k] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = make_uint4(0u, 0u, 0u, 0u);
        }
        pr_swap(b0, 1, v[0], v[1]);
        pr_swap(b0, 1, v[2], v[3]);
        pr_swap(b1, 2, v[0], v[2]);
        pr_swap(b1, 2, v[1], v[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (rows[k] >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + rows[k] + x + (lane & 3) * 8) = v[k];
      }
      tc_fence_before();  // (the output's reads come before the next item's first product)
      if (it.nt > 0 && s_poison[8 * ir + (mine & 7)] == mine)
        prompt_show_bad<D, T>(a, it.ka, it.kvh, it.kt_edge * kPrN, min(it.l, it.nt * kPrN), at, lim, xa, xe);
      it = nx;
    }
    if (!ok) *s_fail = 1;
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      // ---- TMA: Q0, K0, Q1, V0, K1, V1, ...; in halves Q0, K0, K1, V0, K2, V1, ... ----
      if (lane == 0) {
        const uint32_t qbytes = (uint32_t)(a.tpt * a.gp * 128 * NC);
        uint32_t ph = 0, land = 0, q_ph = 0;        // phases: of the ring, bits per stage, bits per row tile
        uint32_t used = 0, looks = 0;               // for the end: stages loaded, by which barrier
        int st = 0, qn = 0;
        bool ok = true;
        for (int round = 0; ok && round < rounds; ++round) {
          PrItem it;
          if (!item(round, it) || it.nt == 0) continue;
          auto load_q = [&](int i) {
            if (!mbar_wait_bounded(&q_empty[i], ((q_ph >> i) & 1) ^ 1)) return false;
            q_ph ^= 1u << i;
            qn |= 1 << i;
            mbar_arrive_expect_tx(&q_full[i], qbytes);
            for (int cnk = 0; cnk < NC; ++cnk)
              tma_load_4d(qs + i * TB + cnk * CB, &mq, cnk * 64, it.hoff, it.kvh, it.qa + it.tok0 + i * a.tpt, &q_full[i]);
            return true;
          };
          ok = load_q(0);
          for (int x = 0; ok && x < 2 * it.nt; ++x) {
            ok = mbar_wait_bounded(&empty[st], ph ^ 1) && !*s_fail;
            if (!ok) break;
            // Value tiles from kt_edge on land on barriers of their own, which the
            // lookers follow without the uses of the ring before them; their stage's
            // full barrier is passed at once.  v_land and v_ok are per stage, so that
            // neither can run a phase ahead of whom it wakes.
            const bool value = !HALVES ? x & 1 : x == 2 * it.nt - 1 || (x > 0 && (x & 1) == 0);
            const int tile = !HALVES ? x >> 1 : x == 2 * it.nt - 1 ? it.nt - 1 : (x & 1) ? (x + 1) >> 1 : max(0, (x >> 1) - 1);
            const bool look = value && tile >= it.kt_edge;
            uint64_t* bar = look ? &v_land[st] : &full[st];
            mbar_arrive_expect_tx(bar, (uint32_t)TB);
            for (int cnk = 0; cnk < NC; ++cnk)
              tma_load_3d(ring + st * TB + cnk * CB, value ? &mv : &mk, cnk * 64, it.kvh, it.ka + tile * kPrN, bar);
            if (look) {
              mbar_arrive(&full[st]);
              land ^= 1u << st;
            }
            used |= 1u << st;
            looks = look ? looks | 1u << st : looks & ~(1u << st);
            if (++st == NS) {
              st = 0;
              ph ^= 1;
            }
            if (x == 0 && it.nq == 2) ok = load_q(1);
          }
        }
        if (!ok) *s_fail = 1;
        // copies in flight land before the CTA may end, whichever warp gave up
        for (int i = 0; i < 2; ++i)
          if (qn >> i & 1) mbar_drain(&q_full[i], ((q_ph >> i) & 1) ^ 1);
        for (int x = 0; x < NS; ++x) {
          if (!(used >> x & 1)) continue;
          if (looks >> x & 1) mbar_drain(&v_land[x], ((land >> x) & 1) ^ 1);
          else mbar_drain(&full[x], x < st ? ph : ph ^ 1);
        }
      }
    } else if (warp == 9) {
      // ---- matrix instructions: the whole warp keeps step, one thread issues ----
      constexpr uint32_t id_s = pr_idesc(BF, kPrN, false), id_o = pr_idesc(BF, D, true);
      const uint64_t q_desc = pr_desc(smem_u32(qs), 16), k_desc = pr_desc(smem_u32(ring), 16), v_desc = pr_desc(smem_u32(ring), CB);
      uint32_t ph = 0, land = 0, q_ph = 0, p_ph = 0;
      int st = 0;
      bool ok = true;
      auto next = [&]() {
        if (++st == NS) {
          st = 0;
          ph ^= 1;
        }
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(B2Q_FULL, mbar_wait_bounded(bar, parity)) != 0; };
      auto scores = [&](int i, int ks) {  // S_i = Q_i K^T
        const uint64_t q = q_desc + (uint32_t)((HALVES ? 0 : i) * (TB >> 4)), kd = k_desc + (uint32_t)(ks * (TB >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = ((k >> 2) * CB + (k & 3) * 32) >> 4;
          pr_mma_ss(tmem + i * 128, q + o, kd + o, id_s, k > 0);
        }
        pr_commit(&s_full[i]);
      };
      for (int round = 0; ok && round < rounds; ++round) {
        PrItem it;
        if (!item(round, it) || it.nt == 0) continue;
        // the first scores: of both row tiles with the first keys, or of the one
        // with the first two
        const int ns = HALVES ? min(2, it.nt) : it.nq;
        for (int i = 0; ok && i < ns; ++i) {
          if (i == 0 || HALVES) ok = wait(&full[st], ph);
          if (ok && (i == 0 || !HALVES)) {
            ok = wait(&q_full[i], (q_ph >> i) & 1);
            q_ph ^= 1u << i;
          }
          if (!ok) break;
          tc_fence_after();
          const bool last = HALVES || i + 1 == ns;  // the keys' last use
          if (pr_elect()) {
            scores(i, st);
            if (it.nt == (HALVES ? i + 1 : 1)) pr_commit(&q_empty[HALVES ? 0 : i]);
            if (last) pr_commit(&empty[st]);
          }
          if (last) next();
        }
        for (int j = 0; ok && j < it.nt; ++j) {
          const bool more = j + step < it.nt;
          const int sv = st;
          ok = wait(&full[sv], ph);
          if (ok && j >= it.kt_edge) {
            ok = wait(&v_ok[sv], (land >> sv) & 1);
            land ^= 1u << sv;
          }
          next();
          const int sk = st;
          if (ok && more) {
            ok = wait(&full[sk], ph);
            next();
          }
          const int ie = HALVES ? (j & 1) + 1 : it.nq;
          for (int i = HALVES ? j & 1 : 0; ok && i < ie; ++i) {
            ok = wait(&p_full[i], (p_ph >> i) & 1) && !*s_fail;
            if (!ok) break;
            p_ph ^= 1u << i;
            tc_fence_after();
            if (pr_elect()) {
              const uint64_t v = v_desc + (uint32_t)(sv * (TB >> 4));  // O_i (+)= P_i V
#pragma unroll
              for (int k = 0; k < kPrN / 16; ++k)
                pr_mma_ts(tmem + 256 + i * D, tmem + i * 128 + k * 8, v + ((k * 2048) >> 4), id_o, j >= step || k > 0);
              if (more) scores(i, sk);
              else pr_commit(&o_full[i]);
              if (j + 1 + step == it.nt) pr_commit(&q_empty[HALVES ? 0 : i]);
            }
          }
          if (ok && pr_elect()) {
            pr_commit(&empty[sv]);
            if (more) pr_commit(&empty[sk]);
          }
        }
      }
      if (!ok) *s_fail = 1;
      // whatever was issued completes before the TMEM is freed, whichever warp gave up
      __syncwarp();
      if (pr_elect()) pr_commit(&done);
      mbar_drain(&done, 0);
    } else {
      // ---- value tiles that some row sees only in part ----
      const int w = threadIdx.x - 320;  // 0..63: rows w and w + 64
      uint32_t land = 0;
      // The item's first stage; items with key tiles of either row tile, in eight places for
      // each: the ring ends a few items ahead of a row tile's own next one, but row tile 0
      // may go through any number of items that have no second one while that one ends.
      int x0 = 0, count[2] = {0, 0};
      bool ok = true;
      for (int round = 0; ok && round < rounds; ++round) {
        PrItem it;
        if (!item(round, it) || it.nt == 0) continue;
        ++count[0];
        count[1] += it.nq == 2;
        for (int j = it.kt_edge; j < it.nt; ++j) {
          const int st = (x0 + (HALVES && j + 1 < it.nt ? 2 * j + 2 : 2 * j + 1)) % NS;
          ok = __all_sync(B2Q_FULL, mbar_wait_bounded(&v_land[st], (land >> st) & 1)) && !*s_fail;
          if (!ok) break;
          land ^= 1u << st;
          uint8_t* vt = ring + st * TB;
          uint32_t nan = 0;  // (pairs) the sum of 0 * value: NaN if one is not finite
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const int row = w + 64 * hh;
            if (j * kPrN + row >= it.l) {  // behind the sequence
              for (int y = 0; y < 8 * NC; ++y)
                *reinterpret_cast<uint4*>(vt + (y >> 3) * CB + row * 128 + ((y ^ row) & 7) * 16) = make_uint4(0, 0, 0, 0);
            } else {
#pragma unroll
              for (int y = 0; y < 8 * NC; ++y) {
                const uint4 v = *reinterpret_cast<const uint4*>(vt + (y >> 3) * CB + row * 128 + ((y ^ row) & 7) * 16);
                nan = pr_fma2<BF>(v.x, 0u, pr_fma2<BF>(v.y, 0u, pr_fma2<BF>(v.z, 0u, pr_fma2<BF>(v.w, 0u, nan))));
              }
            }
          }
          if (__any_sync(B2Q_FULL, (nan & 0x7fff7fffu) != 0)) {
            s_poison[count[0] & 7] = count[0];
            if (it.nq == 2) s_poison[8 + (count[1] & 7)] = count[1];
            constexpr uint32_t em = BF ? 0x7f80u : 0x7c00u;  // an infinity or NaN has all exponent bits set
#pragma unroll 1
            for (int x = 0; x < 2 * 32 * NC; ++x) {  // two values of row w or w + 64 (in whatever order)
              uint32_t* u = reinterpret_cast<uint32_t*>(vt + (x >> 6) * CB + (w + 64 * (x >> 5 & 1)) * 128) + (x & 31);
              *u &= ((*u & em) == em ? 0u : 0xffffu) | ((*u & (em << 16)) == (em << 16) ? 0u : 0xffff0000u);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ok[st]);
        }
        x0 = (x0 + 2 * it.nt) % NS;
      }
      if (!ok) *s_fail = 1;
    }
  }
  kv_check_offsets(a.q_start, a.n_seqs, s_q[0], s_q + 1, cached);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace b2q
