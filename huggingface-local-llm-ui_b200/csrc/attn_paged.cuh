// attn_paged.cuh -- attention of the newest tokens of many sequences over
// their keys and values in the paged 4-bit cache (kv_page.cuh):
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - max),  j <= position.
//
// The cache is read once, 18 * D bytes for 16 keys and values of a head, and
// that stream is the floor.  What bounds the kernel is the instructions beside it
// (some 530 a warp for 16 keys and 16 rows, half of them unpacking), issued on 43 to
// 51 % of the cycles: two or three warps a scheduler is what the registers of the
// outputs allow.  One sequence of 131072 keys, 32 heads over 8: 65 us (2.3 TB/s of
// cache); 64 ragged sequences up to 8192 keys: 95 us; 16 sequences with five drafted
// tokens of 64 heads over 8: 61 us; 585 keys: 9.5 us under a page table with room for
// as many, 12.2 under one with room for 8192, most of it latency.
//
// Items.  The query rows (token, head) of one sequence that share a K/V head
// are cut into blocks of 8 * NG rows; (sequence, row block, K/V head) is an
// item, its keys are cut into tiles of 64.  All items' blocks of 16 keys in one line are
// divided evenly over the CTAs and within a CTA over its warps, whatever the
// lengths (the lengths stay on the device, so a captured call follows them).
// A warp works alone on its tiles: a private ring of bulk copies (221 KB per
// SM over twelve warps at D = 128), a running softmax, no barrier in the loop.  Items that end
// inside a warp's share are written at once; the pieces of cut items are joined by
// their CTA, and those of items cut between CTAs, through the workspace, by
// attn_paged_join_kernel, each in order: the same bits every time.  Few items that
// the page table keeps short take a cluster of CTAs each instead, which joins its
// pieces itself (PagedArgs::whole).
//
// Products, on the warp-level tensor cores (mma.m16n8k16, f16 in, f32 out),
// with the codes as exact small integers and the f16 scales applied in f32:
//   S: A = queries (f32 queries as f16 hi rows 0-7 and lo rows 8-15 of one
//      tile, ~2^-22; 16-bit queries exactly down to 2^-27 of the row's largest; rows
//      scaled by a power of two),
//      B = key codes; the sum over each 32 dims is multiplied by the key's scale;
//   O: A = value codes (16 dims x 16 keys), B = p_j * scale_j (f16 hi, and lo
//      where the output is f32), one B for each 32 dims.
// (Codes left where they lie, as f16 subnormals, would halve the unpacking, but
// the matrix unit aligns products by their nominal exponents: 2^-17 is lost.)
// A row's softmax reference follows the largest p_j * scale_j of the keys that the row
// sees (the largest scale of a key's blocks of dims) in steps of 2^8, so that it lies
// between 2^6 and 2^15: a product keeps its bits down to 2^-31 of that one (f16's
// smallest step is 2^-24), and outputs are seldom rescaled.
#pragma once

#include <type_traits>

#include "kv_page.cuh"

namespace b2q {

constexpr int kPgTile = 64, kPgBlks = kPgTile / kKvBlk;  // keys of a tile, blocks of them
// warps of a CTA: what the registers of the tiling allow
__host__ __device__ constexpr int pg_warps(int NG) { return NG == 1 ? 12 : 8; }
template <int NG>
struct PgThreads {
  static constexpr int value = 32 * pg_warps(NG);
};
constexpr int kPgChunk = 32;                    // sequences of one partial sum of the plan
constexpr int kPgMaxChunks = 65536 / kPgChunk;  // (n_seqs <= 65535)
__host__ __device__ constexpr int pg_stage_bytes(int D) { return kPgBlks * kv_blk_bytes(D); }
__host__ __device__ constexpr int pg_stages(int D) { return D == 128 ? 2 : 4; }
__host__ __device__ constexpr int pg_ring_bytes(int D, int NG) { return pg_warps(NG) * pg_stages(D) * pg_stage_bytes(D); }
constexpr int kPgPad = 4;  // floats after a row of a piece in shared memory: its column stores fall on distinct banks
__host__ __device__ constexpr int pg_rows(int NG) { return 8 * NG; }
// one piece in the workspace: rows of D floats, then (reference, sum) pairs
__host__ __device__ constexpr int pg_part_floats(int D, int NG) { return pg_rows(NG) * (D + 2); }
// the same in shared memory
__host__ __device__ constexpr int pg_piece_floats(int D, int NG) { return pg_rows(NG) * (D + kPgPad + 2); }
// (two pieces of every warp fit the ring's place)
static_assert(2 * pg_warps(1) * pg_piece_floats(128, 1) * 4 <= pg_ring_bytes(128, 1) &&
              2 * pg_warps(2) * pg_piece_floats(128, 2) * 4 <= pg_ring_bytes(128, 2) &&
              2 * pg_warps(1) * pg_piece_floats(64, 1) * 4 <= pg_ring_bytes(64, 1) &&
              2 * pg_warps(2) * pg_piece_floats(64, 2) * 4 <= pg_ring_bytes(64, 2), "");
// Units of the line: an item counts its blocks (16 keys) and kPgSetup more for
// its queries, its end and its place in the line; a warp gets at least kPgMin.
constexpr int kPgSetup = 5, kPgMin = 1;
constexpr int kPgMaxCtas = 256;
constexpr int kPgMaxCluster = 8;  // (the portable size)

// Who a piece of an item belongs to, and whether it holds the item's first
// and last block.  seq < 0: no piece.
struct PgDesc {
  int seq, sub, first, last;
};

// x / d of numbers below 2^31 by one multiplication: mul = floor(2^(31 + s) / d)
// + 1 with 2^s >= d is too large by less than 2^s / 2^(31 + s), so the quotient is
// exact.
struct FastDiv {
  uint32_t mul;
  int shift, d;
};
__host__ inline FastDiv fast_div(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return FastDiv{(uint32_t)(((1ull << (31 + s)) / (uint32_t)d) + 1), 31 + s, d};
}
__host__ __device__ __forceinline__ int fdiv(int x, const FastDiv& f) { return (int)(((uint64_t)(uint32_t)x * f.mul) >> f.shift); }

struct PagedArgs {
  KvBatch b;
  int H, G;
  FastDiv dG, dKV, dPage;  // by G, by the K/V heads, by the tokens of a page
  int coarse;              // a unit of the line is 2^coarse blocks
  int whole;               // > 0: an item is a unit, and a cluster of as many CTAs has it to itself
  const void* q;
  int q_type;
  int64_t q_stride;
  const uint8_t* pages;
  float scale;
  void* out;
  int out_type;
  PgDesc* desc;  // [CTAs][2]: the piece begun before the CTA, the piece it begins
  float* part;   // [CTAs][2][pg_part_floats]
  float* part0;  // [CTAs][warps][pg_piece_floats]: pieces that warps begin with, until their CTA joins them
};

// The part of a sequence's geometry that the plan needs.
struct PgSeq {
  int qa, n;      // first row, rows of this call
  int base, len;  // position of the first row (may be negative), cached tokens that the table has room for
  int rows;       // n * G
  int nb, nrb;    // blocks of an item (16 keys), row blocks
};

__host__ __device__ inline PgSeq pg_seq_of(int qa, int qe, int len, int n_tokens, int cap, int G, int R, bool& bad) {
  PgSeq s;
  const bool ok = qa >= 0 && qe >= qa;
  const int n_all = ok ? qe - qa : 0;
  bad = !ok || (n_all > 0 && (len < n_all || len > cap || qe > n_tokens));
  s.qa = qa;
  s.n = ok ? (qe < n_tokens ? qe : n_tokens) - qa : 0;
  if (s.n < 0) s.n = 0;
  s.len = len < 0 ? 0 : len > cap ? cap : len;
  s.base = (len < 0 ? 0 : len) - n_all;  // (below 0 cached tokens no row has a position, as with 0)
  s.rows = s.n * G;
  s.nb = s.len > kKvBlk ? (s.len + kKvBlk - 1) / kKvBlk : 1;  // (one for none: its rows become zeros)
  s.nrb = (s.rows + R - 1) / R;
  return s;
}

template <int NG>
__device__ __forceinline__ PgSeq pg_seq(const PagedArgs& a, int s) {
  bool bad;
  const PgSeq q = pg_seq_of(a.b.q_start[s], a.b.q_start[s + 1], a.b.kv_len[s], a.b.n_tokens,
                            a.b.max_pages * a.b.page_tokens, a.G, pg_rows(NG), bad);
  if (bad) kv_batch_error();
  return q;
}
// Units of an item, and of a sequence.  (The host picks `coarse` so that all
// sequences at their largest stay below 2^31.)
__device__ __forceinline__ int pg_per(const PagedArgs& a, const PgSeq& q) {
  return a.whole ? 1 : ((q.nb + (1 << a.coarse) - 1) >> a.coarse) + kPgSetup;
}
__device__ __forceinline__ int pg_units(const PagedArgs& a, const PgSeq& q) { return q.nrb * a.b.KV * pg_per(a, q); }

// Units of a warp's lanes (each below 2^31) in all, at most kPgFull.
constexpr unsigned kPgFull = 0x7fffffffu;
__device__ __forceinline__ unsigned pg_sum(unsigned v) {
  const unsigned lo = __reduce_add_sync(B2Q_FULL, v & 0xffffu), hi = __reduce_add_sync(B2Q_FULL, v >> 16);
  return hi >= 0x8000u ? kPgFull : min((hi << 16) + lo, kPgFull);
}

// A place in the line: block blk of item (seq, sub), sub = row block * KV + K/V
// head.  The end of the line is sequence n_seqs.
struct PgAt {
  int seq, sub, blk;
  PgSeq q;
};

// The next item's first block.
template <int NG>
__device__ __noinline__ void pg_next_item(const PagedArgs& a, PgAt& p) {
  p.blk = 0;
  if (++p.sub < p.q.nrb * a.b.KV) return;
  p.sub = 0;
  for (++p.seq; p.seq < a.b.n_seqs; ++p.seq) {
    p.q = pg_seq<NG>(a, p.seq);
    if (p.q.nrb) return;
  }
}

__device__ __forceinline__ int pg_scan(int v, int lane) {  // inclusive sum over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(B2Q_FULL, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// The place of unit u within 32 sequences, lane s0 + l with geometry q and
// `inc` units up to its end, v of them its own (by a warp).
__device__ __forceinline__ void pg_place(const PagedArgs& a, int s0, const PgSeq& q, int v, int inc, int u, PgAt& p) {
  const unsigned hit = __ballot_sync(B2Q_FULL, inc > u);
  const int l = hit ? __ffs(hit) - 1 : 31;
  u -= __shfl_sync(B2Q_FULL, inc - v, l);
  p.seq = hit ? s0 + l : a.b.n_seqs;  // (not hit: the arrays changed under the kernel)
  p.q.qa = __shfl_sync(B2Q_FULL, q.qa, l);
  p.q.n = __shfl_sync(B2Q_FULL, q.n, l);
  p.q.base = __shfl_sync(B2Q_FULL, q.base, l);
  p.q.len = __shfl_sync(B2Q_FULL, q.len, l);
  p.q.rows = __shfl_sync(B2Q_FULL, q.rows, l);
  p.q.nb = __shfl_sync(B2Q_FULL, q.nb, l);
  p.q.nrb = __shfl_sync(B2Q_FULL, q.nrb, l);
  const unsigned per = (unsigned)pg_per(a, p.q);
  p.sub = (int)((unsigned)u / per);
  p.blk = max(0, u - p.sub * (int)per - kPgSetup) << a.coarse;
}

// Keys of an item: those its last row attends.
template <int NG>
__device__ __forceinline__ int pg_keys(const PagedArgs& a, const PgAt& p) {
  const int rb = fdiv(p.sub, a.dKV);
  const int last = fdiv(min(p.q.rows, (rb + 1) * pg_rows(NG)) - 1, a.dG);
  return max(0, min(p.q.len, p.q.base + last + 1));
}

__device__ __forceinline__ float pg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void pg_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a * b
__device__ __forceinline__ void pg_mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t h2_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u32_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// code - 8 of nibbles 0 and 1 (from the low end) of both 16-bit halves of w,
// as f16 pairs: 1024 + code and 1024 + 16 code are f16 numbers whose low bits
// are the code's, so one OR and one exact add or multiply-add make the value.
// (w & mask) | magic is one instruction with at most one immediate: the magic
// number and the second constants stay in registers (pg_const).
struct PgConst {
  uint32_t magic, sixteenth, minus72;
};
__device__ __forceinline__ PgConst pg_const() {
  PgConst c;
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(c.magic));
  asm volatile("mov.b32 %0, 0x2c002c00;" : "=r"(c.sixteenth));
  asm volatile("mov.b32 %0, 0xd480d480;" : "=r"(c.minus72));
  return c;
}
__device__ __forceinline__ void pg_unpack2(uint32_t w, const PgConst& c, uint32_t& n0, uint32_t& n1) {
  uint32_t x0, x1;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(x0) : "r"(w), "r"(c.magic));
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(x1) : "r"(w), "r"(c.magic));
  n0 = h2_u32(__hadd2(u32_h2(x0), __floats2half2_rn(-1032.0f, -1032.0f)));
  n1 = h2_u32(__hfma2(u32_h2(x1), u32_h2(c.sixteenth), u32_h2(c.minus72)));
}

__device__ __forceinline__ void pg_store(const PagedArgs& a, int64_t i, float v) {
  if (a.out_type == kElF32) reinterpret_cast<float*>(a.out)[i] = v;
  else if (a.out_type == kElF16) reinterpret_cast<__half*>(a.out)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ void pg_store4(const PagedArgs& a, int64_t i, const float (&v)[4]) {
  if (a.out_type == kElF32) st4(reinterpret_cast<float*>(a.out) + i, v);
  else if (a.out_type == kElF16) st4(reinterpret_cast<__half*>(a.out) + i, v);
  else st4(reinterpret_cast<__nv_bfloat16*>(a.out) + i, v);
}
// Whether row r of the sequence is one, and has a position: one of a length beyond the
// page table, or of fewer cached tokens than new ones, is left as it is.
__device__ __forceinline__ bool pg_row_live(const PagedArgs& a, const PgSeq& q, int r) {
  return r < q.rows && (unsigned)(q.base + fdiv(r, a.dG)) < (unsigned)(a.b.max_pages * a.b.page_tokens);
}
// Index of row r (of a sequence from row qa on) of K/V head h in out (and, with
// the token stride, in q).
__device__ __forceinline__ int64_t pg_out_row(const PagedArgs& a, int qa, int r, int h, int D) {
  const int tok = fdiv(r, a.dG);
  return ((int64_t)(qa + tok) * a.H + h * a.G + r - tok * a.G) * D;
}

// 8 consecutive elements of q as f32 (16-byte aligned)
__device__ __forceinline__ void pg_load8(const PagedArgs& a, int64_t i, float (&v)[8]) {
  if (a.q_type == kElF32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + i);
    const float4 x = p[0], y = p[1];
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + i);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.q_type == kElF16) {
        const float2 f = __half22float2(u32_h2(w[e]));
        v[2 * e] = f.x;
        v[2 * e + 1] = f.y;
      } else {
        v[2 * e] = __uint_as_float(w[e] << 16);
        v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
    }
  }
}

// One value of a chain of pieces at `f`-indexed places: weights 2^(ref_i - ref).
__device__ __forceinline__ float pg_weight(float ref_i, float ref) { return ref_i == -INFINITY ? 0.0f : pg_exp2(ref_i - ref); }

template <int D, int NG, bool QSPLIT, bool PSPLIT>
__global__ void __launch_bounds__(PgThreads<NG>::value, 1) attn_paged_kernel(const __grid_constant__ PagedArgs a) {
  extern __shared__ __align__(128) uint8_t pg_smem[];
  constexpr int S = pg_stages(D), SB = pg_stage_bytes(D), BB = kv_blk_bytes(D);
  constexpr int W = pg_warps(NG);
  constexpr int NB = D / 32, R = pg_rows(NG), PR = D + kPgPad;
  static_assert(NG == 1 || !QSPLIT, "the second part of f32 queries takes the rows of a second group");
  __shared__ uint64_t bars[W][S];
  __shared__ PgDesc s_desc[W][2];
  __shared__ PgAt s_at[W], s_ld[W];
  __shared__ int3 s_end[W];
  __shared__ PgDesc s_out[2];
  __shared__ int s_run[2 * W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();

  // ---- plan: this warp's share of the line: from unit w0 of it to where the
  // next warp's begins ----
  const int nch = (a.b.n_seqs + kPgChunk - 1) / kPgChunk;
  int* sums = reinterpret_cast<int*>(pg_smem);  // units of 32 sequences each (the ring's place)
  if (threadIdx.x < W * S) mbar_init(&bars[0][0] + threadIdx.x, 1);
  if (threadIdx.x < W * 2) (&s_desc[0][0])[threadIdx.x].seq = -1;
  fence_mbar_init();
  PgSeq q0{};
  int v0 = 0;
  if (nch > 1) {
    for (int c = warp; c < nch; c += W) {
      const int s = c * kPgChunk + lane;
      const unsigned w = pg_sum(s < a.b.n_seqs ? pg_units(a, pg_seq<NG>(a, s)) : 0);
      if (lane == 0) sums[c] = (int)w;
    }
    __syncthreads();
    for (int c = lane; c < nch; c += 32) v0 = (int)min((unsigned)v0 + (unsigned)sums[c], kPgFull);
  } else if (lane < a.b.n_seqs) {  // every warp has all of them in its lanes
    q0 = pg_seq<NG>(a, lane);
    v0 = pg_units(a, q0);
  }
  unsigned total = pg_sum(v0);
  // offsets that go up and down give more rows than there are: nothing is done
  if (total == kPgFull || (a.whole && total * a.whole > gridDim.x)) {
    if (threadIdx.x == 0) kv_batch_error();
    total = 0;
  }
  const unsigned nc = a.whole ? total * a.whole : min(gridDim.x, (total + W * kPgMin - 1) / (W * kPgMin));
  const bool working = blockIdx.x < nc;
  if (working) {
    // the remainders go one each to the first CTAs and warps
    const unsigned per = total / nc, odd = total - per * nc;
    const unsigned c0 = per * blockIdx.x + min(blockIdx.x, odd), cn = per + (blockIdx.x < odd);
    for (int x = warp; x <= W; x += W) {  // (the first warp finds the CTA's end as well)
      const int u = a.whole ? (int)blockIdx.x / a.whole : (int)(c0 + cn / W * x + min((unsigned)x, cn % W));
      PgAt p{};
      p.seq = a.b.n_seqs;
      if (nch > 1) {
        int ch = -1, rest = u;
        for (int k = 0; k < nch && ch < 0; k += 32) {
          const int v = k + lane < nch ? sums[k + lane] : 0, inc = pg_scan(v, lane);
          const unsigned hit = __ballot_sync(B2Q_FULL, inc > rest);
          const int l = hit ? __ffs(hit) - 1 : 31;
          if (hit) ch = k + l;
          rest -= __shfl_sync(B2Q_FULL, hit ? inc - v : inc, l);
        }
        if (ch >= 0) {
          const int s = ch * kPgChunk + lane;
          PgSeq q{};
          int v = 0;
          if (s < a.b.n_seqs) {
            q = pg_seq<NG>(a, s);
            v = pg_units(a, q);
          }
          pg_place(a, ch * kPgChunk, q, v, pg_scan(v, lane), rest, p);
        }
      } else if ((unsigned)u < total) {
        pg_place(a, 0, q0, v0, pg_scan(v0, lane), u, p);
      }
      if (a.whole) p.blk = p.q.nb * ((int)blockIdx.x % a.whole * W + x) / (a.whole * W);
      if (lane == 0) {
        if (x < W) s_at[x] = s_ld[x] = p;
        if (x > 0) s_end[x - 1] = make_int3(p.seq, p.sub, p.blk);
      }
    }
  }
  fence_proxy_async_smem();  // the plan's sums were in the ring's place
  __syncthreads();
  bool more = false;  // this warp has blocks left to fetch
  if (working) {
    const PgAt& p = s_at[warp];
    const int3 e = s_end[warp];
    more = p.seq < a.b.n_seqs && !(p.seq == e.x && p.sub == e.y && p.blk == e.z);
  }

  // ---- the ring: copies run S - 1 tiles ahead; a tile's page numbers are
  // fetched one tile before its copies are issued.  Both places, of the next
  // tile to fetch and of the tile in work, lie in shared memory (registers are
  // short), but for what changes from tile to tile ----
  uint8_t* ring = pg_smem + warp * S * SB;
  const int bpp = a.b.page_tokens / kKvBlk;
  constexpr uint32_t kAll = (1u << kPgBlks) - 1;
  int64_t blk_next = -1;  // lane j < kPgBlks: block j of the next tile to copy, -1: none
  bool have = false;      // there is a next tile to copy
  uint32_t valid = 0;     // kPgBlks bits for each of the last stages: blocks that hold keys
  // of the item being fetched: next block, where it (or the share) ends, keys,
  // K/V head; lane j < kPgBlks: the page and the place in it of block j of the next tile
  int ld_blk = 0, ld_end = 0, ld_keys = 0, ld_h = 0, ld_seq = 0, ld_pg = 0, ld_off = 0;
  const int dpg = fdiv(kPgTile, a.dPage), doff = kPgTile - dpg * a.b.page_tokens;
  auto end_of = [&](const PgAt& p) {  // of the item's blocks in this share
    const int3 e = s_end[warp];
    return p.seq == e.x && p.sub == e.y ? e.z : p.q.nb;
  };
  auto next_item = [&](PgAt* p) {  // false: the share ends
    const int3 e = s_end[warp];
    const bool at_end = p->seq == e.x && p->sub == e.y;
    __syncwarp();
    if (at_end) return false;
    if (lane == 0) pg_next_item<NG>(a, *p);
    __syncwarp();
    return p->seq < a.b.n_seqs && !(p->seq == e.x && p->sub == e.y && e.z == 0);
  };
  auto ld_item = [&]() {
    const PgAt& p = s_ld[warp];
    ld_blk = p.blk;
    ld_end = end_of(p);
    ld_keys = pg_keys<NG>(a, p);
    ld_h = p.sub - fdiv(p.sub, a.dKV) * a.b.KV;
    ld_seq = p.seq;
    const int pos = (p.blk + (lane & (kPgBlks - 1))) * kKvBlk;
    ld_pg = fdiv(pos, a.dPage);
    ld_off = pos - ld_pg * a.b.page_tokens;
  };
  auto fetch = [&]() {
    have = more;
    blk_next = -1;
    if (!more) return;
    const int blk = ld_blk + lane;
    if (lane < kPgBlks && blk < ld_end && blk * kKvBlk < ld_keys) {
      const int page = ld_pg < a.b.max_pages ? a.b.page_table[(int64_t)ld_seq * a.b.max_pages + ld_pg] : -1;
      if (page >= 0 && page < a.b.n_pages) blk_next = ((int64_t)page * a.b.KV + ld_h) * bpp + ld_off / kKvBlk;
      else kv_batch_error();
    }
    ld_blk += kPgBlks;
    if (ld_blk < ld_end) {
      ld_pg += dpg;
      ld_off += doff;
      if (ld_off >= a.b.page_tokens) {
        ld_off -= a.b.page_tokens;
        ++ld_pg;
      }
    } else {
      more = next_item(&s_ld[warp]);
      if (more) ld_item();
    }
  };
  int ist = 0;         // the stage of the next copies
  int in_flight = 0;   // tiles issued and not yet waited for
  auto issue = [&]() {  // copies of the next tile (its page numbers are in blk_next)
    const int st = ist;
    ist = ist + 1 == S ? 0 : ist + 1;
    ++in_flight;
    const unsigned m = __ballot_sync(B2Q_FULL, blk_next >= 0);
    valid = (valid & ~(kAll << (kPgBlks * st))) | ((m & kAll) << (kPgBlks * st));
    if (lane == 0) mbar_arrive_expect_tx(&bars[warp][st], __popc(m) * BB);
    __syncwarp();
    if (blk_next >= 0) bulk_g2s(ring + st * SB + lane * BB, a.pages + blk_next * BB, BB, &bars[warp][st]);
  };
  if (more) ld_item();
  fetch();
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (have) {
      issue();
      fetch();
    }

  // ---- the running state of an item's rows ----
  const PgConst kc = pg_const();
  uint32_t qa[D / 16][4];
  float o[NG][D / 16][4];
  float mx[NG], ref[NG], sum[NG], fac[NG];
  int lim[NG];
  int keys = 0, min_lim = 0;
  int at_blk = 0, at_end = 0;
  auto begin = [&]() {
    const PgAt at = s_at[warp];
    at_blk = at.blk;
    at_end = end_of(at);
    const int rb = fdiv(at.sub, a.dKV), h = at.sub - rb * a.b.KV;
    keys = pg_keys<NG>(a, at);
    float qv[NG][NB][8];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int r = rb * R + 8 * n + g;
      const bool live = r < at.q.rows;
      const int tok = fdiv(r, a.dG);
      lim[n] = live ? at.q.base + tok : keys - 1;
      float am = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (live) {
          const int64_t i = (int64_t)(at.q.qa + tok) * a.q_stride + (h * a.G + r - tok * a.G) * D + 32 * b + 8 * t;
          pg_load8(a, i, qv[n][b]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) qv[n][b][e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(qv[n][b][e]));
      }
      am = fmaxf(am, __shfl_xor_sync(B2Q_FULL, am, 1));
      am = fmaxf(am, __shfl_xor_sync(B2Q_FULL, am, 2));
      // the row times 2^(13 - e), 2^e <= its largest magnitude: exact, inside f16
      int e = (int)((__float_as_uint(am) >> 23) & 255u) - 127;
      if (am == 0.0f || e >= 127) e = 13;
      e = max(e, -100);
      const float sc = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
      // and never 0, which would undo the mask's -inf, nor infinite: a product of 0 stays 0
      fac[n] = fminf(fmaxf(a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - 13 + e) << 23), 1e-37f), 3e38f);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int x = 0; x < 8; ++x) qv[n][b][x] *= sc;
      mx[n] = ref[n] = -INFINITY;
      sum[n] = 0.0f;
#pragma unroll
      for (int m = 0; m < D / 16; ++m) o[n][m][0] = o[n][m][1] = o[n][m][2] = o[n][m][3] = 0.0f;
    }
    min_lim = min(at.q.base + fdiv(rb * R, a.dG), keys - 1);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int x = 0; x < 4; ++x) {  // dims (x, x + 4) of the lane's eight: the order of the codes' nibbles
        uint32_t* f = qa[2 * b + (x >> 1)] + 2 * (x & 1);
        const __half2 hi = __floats2half2_rn(qv[0][b][x], qv[0][b][x + 4]);
        f[0] = h2_u32(hi);
        if (QSPLIT) {
          const float2 hf = __half22float2(hi);
          f[1] = h2_u32(__floats2half2_rn(qv[0][b][x] - hf.x, qv[0][b][x + 4] - hf.y));
        } else {
          f[1] = NG == 2 ? h2_u32(__floats2half2_rn(qv[NG - 1][b][x], qv[NG - 1][b][x + 4])) : 0u;
        }
      }
  };

  // ---- one tile: the stage at tb, its blocks vm.  A block (16 keys) goes
  // through scores, softmax and output in one pass of a loop whose code stays in
  // the instruction cache (all four unrolled, twice, waited for instructions
  // half of the time) ----
  auto tile = [&](const uint8_t* tb, uint32_t vm) {
    const int key0 = at_blk * kKvBlk;
    // Exponent of the largest value scale of tokens 2 lane and 2 lane + 1 of the tile.  (A
    // whole number: a row whose reference it moves has a power of two for its largest
    // probability, whose products with the f16 scales are exact; with the logarithm itself
    // f16 outputs were off by 2.65e-4, not 2.45e-4.  The larger of a number and NaN is the
    // number; what is not finite, or zero, counts as the nearest scale that is, and shows
    // in the products.)
    float lg[2];
    {
      const int blk = lane >> 3;
      uint32_t m[2] = {0u, 0u};
      if ((vm >> blk) & 1) {
        const uint8_t* sp = tb + blk * BB + 17 * D + (lane & 7) * 2 * NB * 2;
        if (NB == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(sp);
          m[0] = h2_u32(__hmax2(__habs2(u32_h2(x.x)), __habs2(u32_h2(x.y))));
          m[1] = h2_u32(__hmax2(__habs2(u32_h2(x.z)), __habs2(u32_h2(x.w))));
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(sp);
          m[0] = h2_u32(__habs2(u32_h2(x.x)));
          m[1] = h2_u32(__habs2(u32_h2(x.y)));
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = __half22float2(u32_h2(m[e]));
        lg[e] = (float)(int)(__float_as_uint(fminf(fmaxf(fmaxf(f.x, f.y), 0x1p-24f), 65504.0f)) >> 23) - 127.0f;
      }
    }
    float ta[NG][D / 16][4];
    if (PSPLIT) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int m = 0; m < D / 16; ++m) ta[n][m][0] = ta[n][m][1] = ta[n][m][2] = ta[n][m][3] = 0.0f;
    }
#pragma unroll 1
    for (int j = 0; j < kPgBlks; ++j) {
      if (!((vm >> j) & 1)) continue;
      const uint8_t* bp = tb + j * BB;
      const int kb0 = key0 + j * kKvBlk;
      const bool edge = kb0 + kKvBlk - 1 > min_lim;  // some key is not every row's
      // S: keys 8 x + 2t, + 1 of the block
      float s[NG][2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t w[NB], sc[NB];  // codes of the lane's 8 dims of each block of dims; scales [token][block pairs]
        if (NB == 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(bp + x * 4 * D + lane * (D / 8));
          const uint4 y = *reinterpret_cast<const uint4*>(bp + 8 * D + (x * 8 + 2 * t) * NB * 2);
          w[0] = u.x; w[1] = u.y; w[NB - 2] = u.z; w[NB - 1] = u.w;
          sc[0] = y.x; sc[1] = y.y; sc[NB - 2] = y.z; sc[NB - 1] = y.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(bp + x * 4 * D + lane * (D / 8));
          const uint2 y = *reinterpret_cast<const uint2*>(bp + 8 * D + (x * 8 + 2 * t) * NB * 2);
          w[0] = u.x; w[1] = u.y;
          sc[0] = y.x; sc[1] = y.y;
        }
        float2 d0[NB / 2], d1[NB / 2];  // scales of the lane's two keys
#pragma unroll
        for (int b = 0; b < NB / 2; ++b) {
          d0[b] = __half22float2(u32_h2(sc[b]));
          d1[b] = __half22float2(u32_h2(sc[NB / 2 + b]));
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) s[n][x][0] = s[n][x][1] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float c[4];
          uint32_t n0, n1;
          pg_unpack2(w[b], kc, n0, n1);
          pg_mma0(c, qa[2 * b], n0, n1);
          pg_unpack2(w[b] >> 8, kc, n0, n1);
          pg_mma(c, qa[2 * b + 1], n0, n1);
          const float e0 = (b & 1) ? d0[b >> 1].y : d0[b >> 1].x, e1 = (b & 1) ? d1[b >> 1].y : d1[b >> 1].x;
          if (QSPLIT) {
            s[0][x][0] = fmaf(c[0] + c[2], e0, s[0][x][0]);
            s[0][x][1] = fmaf(c[1] + c[3], e1, s[0][x][1]);
          } else {
            s[0][x][0] = fmaf(c[0], e0, s[0][x][0]);
            s[0][x][1] = fmaf(c[1], e1, s[0][x][1]);
            if (NG == 2) {
              s[NG - 1][x][0] = fmaf(c[2], e0, s[NG - 1][x][0]);
              s[NG - 1][x][1] = fmaf(c[3], e1, s[NG - 1][x][1]);
            }
          }
        }
      }
      if (edge) {
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int k = kb0 + 8 * x + 2 * t + e;
              if (k > lim[n] || k >= keys) s[n][x][e] = -INFINITY;
            }
      }
      // softmax: the reference moves when a product of a probability and a value scale
      // that the row sees may have outgrown it by 2^15 (when it moves, the largest
      // product is 2^6 or above)
      float sl[2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) sl[x][e] = __shfl_sync(B2Q_FULL, lg[e], 8 * j + 4 * x + t);
      bool move = false;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float tm = fmaxf(fmaxf(fmaf(s[n][0][0], fac[n], sl[0][0]), fmaf(s[n][0][1], fac[n], sl[0][1])),
                         fmaxf(fmaf(s[n][1][0], fac[n], sl[1][0]), fmaf(s[n][1][1], fac[n], sl[1][1])));
        tm = fmaxf(tm, __shfl_xor_sync(B2Q_FULL, tm, 1));
        mx[n] = fmaxf(mx[n], fmaxf(tm, __shfl_xor_sync(B2Q_FULL, tm, 2)));
        move = move || mx[n] - 14.0f > ref[n];
      }
      if (__any_sync(B2Q_FULL, move)) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float cr = 1.0f;
          if (mx[n] - 14.0f > ref[n]) {
            const float nref = mx[n] - 6.0f;
            cr = pg_weight(ref[n], nref);
            ref[n] = nref;
          }
          sum[n] *= cr;
          // at the lanes that hold the row's outputs (rows 2t, 2t + 1)
          const float c2[2] = {__shfl_sync(B2Q_FULL, cr, 8 * t), __shfl_sync(B2Q_FULL, cr, 8 * t + 4)};
#pragma unroll
          for (int m = 0; m < D / 16; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[n][m][e] *= c2[e & 1];
              if (PSPLIT) ta[n][m][e] *= c2[e & 1];
            }
        }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float off = ref[n] == -INFINITY ? 0.0f : -ref[n];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[n][x][e] = pg_exp2(fmaf(s[n][x][e], fac[n], off));
        sum[n] += (s[n][0][0] + s[n][0][1]) + (s[n][1][0] + s[n][1][1]);
      }
      // O
      const uint8_t* vb = bp + 9 * D;
      uint32_t va[2][2][2];      // [key pair][key]: codes of the lane's dims, two words (one at D = 64)
      uint32_t vs[NG][2][2][2];  // [rows][key pair][key]: scales of the blocks of dims, two to a word
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        const uint8_t* vp = vb + pr * 4 * D + lane * (D / 8);
        const uint8_t* sp = vb + 8 * D + (pr * 8 + 2 * t) * NB * 2;
        if (NB == 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(vp);
          const uint4 y = *reinterpret_cast<const uint4*>(sp);
          va[pr][0][0] = u.x; va[pr][0][1] = u.y; va[pr][1][0] = u.z; va[pr][1][1] = u.w;
          vs[0][pr][0][0] = y.x; vs[0][pr][0][1] = y.y; vs[0][pr][1][0] = y.z; vs[0][pr][1][1] = y.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(vp);
          const uint2 y = *reinterpret_cast<const uint2*>(sp);
          va[pr][0][0] = u.x; va[pr][1][0] = u.y;
          vs[0][pr][0][0] = y.x; vs[0][pr][1][0] = y.y;
          va[pr][0][1] = va[pr][1][1] = vs[0][pr][0][1] = vs[0][pr][1][1] = 0u;
        }
        if (NG == 2) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            vs[NG - 1][pr][e][0] = vs[0][pr][e][0];
            vs[NG - 1][pr][e][1] = vs[0][pr][e][1];
          }
        }
      }
      if (edge) {  // what a row does not see may hold anything
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (s[n][x][e] == 0.0f) vs[n][x][e][0] = vs[n][x][e][1] = 0u;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        // A: the block's 32 dims as two tiles of 16, keys pairwise; rows g are
        // nibbles 0 / 2 of a pair, rows g + 8 nibbles 1 / 3
        uint32_t f[2][4];
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const uint32_t w = __byte_perm(va[pr][0][b >> 1], va[pr][1][b >> 1], (b & 1) ? 0x7632 : 0x5410);
          pg_unpack2(w, kc, f[0][2 * pr], f[0][2 * pr + 1]);
          pg_unpack2(w >> 8, kc, f[1][2 * pr], f[1][2 * pr + 1]);
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          uint32_t hi[2], lo[2];
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) {
            const float2 y0 = __half22float2(u32_h2(vs[n][pr][0][b >> 1])), y1 = __half22float2(u32_h2(vs[n][pr][1][b >> 1]));
            const float x0 = s[n][pr][0] * ((b & 1) ? y0.y : y0.x), x1 = s[n][pr][1] * ((b & 1) ? y1.y : y1.x);
            const __half2 h = __floats2half2_rn(x0, x1);
            hi[pr] = h2_u32(h);
            if (PSPLIT) {
              const float2 hf = __half22float2(h);
              lo[pr] = h2_u32(__floats2half2_rn(x0 - hf.x, x1 - hf.y));
            }
          }
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            // f32 outputs: a tile's products are summed by themselves, then added
            // rounded (the matrix unit truncates: long chains would show it)
            float(&acc)[4] = PSPLIT ? ta[n][2 * b + m] : o[n][2 * b + m];
            pg_mma(acc, f[m], hi[0], hi[1]);
            if (PSPLIT) pg_mma(acc, f[m], lo[0], lo[1]);
          }
        }
      }
    }
    if (PSPLIT) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int m = 0; m < D / 16; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][m][e] += ta[n][m][e];
    }
  };

  float* const piece0 = a.part0 + ((int64_t)blockIdx.x * W + warp) * pg_piece_floats(D, NG);
  bool tail = false;      // the share ends with a piece
  int first = 1;          // the piece holds the item's first tile
  bool fresh = true;      // begin() before the next tile
  int st = 0;             // the tile's stage and its barrier's phase
  uint32_t phase = 0;
  auto store_piece = [&](float* p) {  // the rows in hand
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[(8 * n + 2 * t + e) * PR + 16 * m + g] = o[n][m][e];
          p[(8 * n + 2 * t + e) * PR + 16 * m + 8 + g] = o[n][m][2 + e];
        }
      if (t == 0) {
        p[R * PR + 2 * (8 * n + g)] = ref[n];
        p[R * PR + 2 * (8 * n + g) + 1] = sum[n];
      }
    }
  };
  while (in_flight > 0) {
    if (fresh) {
      begin();
      first = at_blk == 0;
      fresh = false;
    }
    if (have) {
      issue();
      fetch();
    }
    if (!__all_sync(B2Q_FULL, mbar_wait_bounded(&bars[warp][st], phase))) {
      // a wait gave up (the error word is set): first the copies in flight
      for (int k = 0; k < in_flight; ++k) {
        mbar_drain(&bars[warp][st], phase);
        if (++st == S) {
          st = 0;
          phase ^= 1;
        }
      }
      break;
    }
    --in_flight;
    const uint32_t vm = (valid >> (kPgBlks * st)) & kAll;
    if (vm) tile(ring + st * SB, vm);
    __syncwarp();  // the stage is free for the copy of the tile S further
    if (++st == S) {
      st = 0;
      phase ^= 1;
    }
    at_blk += kPgBlks;
    if (at_blk < at_end) continue;
    // ---- the item, or this warp's share of it, ends ----
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      sum[n] += __shfl_xor_sync(B2Q_FULL, sum[n], 1);
      sum[n] += __shfl_xor_sync(B2Q_FULL, sum[n], 2);
    }
    const PgAt at = s_at[warp];
    const int last = at_end == at.q.nb;
    const bool on = next_item(&s_at[warp]);  // the share goes on
    if (first && last) {
      const int rb = fdiv(at.sub, a.dKV), h = at.sub - rb * a.b.KV;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float l = __shfl_sync(B2Q_FULL, sum[n], 8 * t + 4 * e);
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          const int r = rb * R + 8 * n + 2 * t + e;
          if (pg_row_live(a, at.q, r)) {
            const int64_t i0 = pg_out_row(a, at.q.qa, r, h, D);
#pragma unroll
            for (int m = 0; m < D / 16; ++m) {
              pg_store(a, i0 + 16 * m + g, o[n][m][e] * inv);
              pg_store(a, i0 + 16 * m + 8 + g, o[n][m][2 + e] * inv);
            }
          }
        }
    } else if (on) {  // begun before this share
      store_piece(piece0);
      if (lane == 0) s_desc[warp][0] = PgDesc{at.seq, at.sub, first, last};
    } else {  // the share's last stays in registers until every warp is done with the ring
      tail = true;
      if (lane == 0) s_desc[warp][1] = PgDesc{at.seq, at.sub, first, last};
    }
    fresh = true;
  }
  __syncthreads();

  // ---- the CTA's pieces, in order, in the ring's place: joined when whole ----
  auto piece = [&](int i) {  // slot i = 2 * warp + (begun before it: 0, its last: 1)
    return reinterpret_cast<float*>(pg_smem) + i * pg_piece_floats(D, NG);
  };
  if (tail) store_piece(piece(2 * warp + 1));
  if (s_desc[warp][0].seq >= 0) {
    const float4* src = reinterpret_cast<const float4*>(piece0);
    float4* dst = reinterpret_cast<float4*>(piece(2 * warp));
#pragma unroll 4
    for (int i = lane; i < pg_piece_floats(D, NG) / 4; i += 32) dst[i] = src[i];
  }
  // runs of pieces of the same item: lane i looks at slot i (2 W <= 32)
  const PgDesc* sd = &s_desc[0][0];
  const bool used = lane < 2 * W && sd[min(lane, 2 * W - 1)].seq >= 0;
  const unsigned in_use = __ballot_sync(B2Q_FULL, used);
  bool begins = used;
  if (used) {
    const unsigned below = in_use & ((1u << lane) - 1);
    if (below) {
      const PgDesc &d = sd[lane], &p = sd[31 - __clz(below)];
      begins = d.seq != p.seq || d.sub != p.sub;
    }
  }
  const unsigned runs = __ballot_sync(B2Q_FULL, begins);
  const int n_runs = __popc(runs);
  if (warp == 0 && begins) s_run[__popc(runs & ((1u << lane) - 1))] = lane;
  if (threadIdx.x < 2) s_out[threadIdx.x].seq = -1;
  __syncthreads();
  // eight threads to a row of a run, D / 8 dims each
  constexpr int DT = D / 8;
  for (int u = threadIdx.x >> 3; u < n_runs * R; u += W * 4) {
    const int c = u / R, r = u - c * R, i = s_run[c], x0 = (threadIdx.x & 7) * 4;
    const int stop = c + 1 < n_runs ? s_run[c + 1] : 2 * W;
    const unsigned members = in_use & ~((1u << i) - 1) & (stop < 32 ? (1u << stop) - 1 : ~0u);
    const PgDesc d = sd[i];
    const int whole_last = sd[31 - __clz(members)].last;
    float rf = -INFINITY;
    for (unsigned m = members; m; m &= m - 1) rf = fmaxf(rf, piece(__ffs(m) - 1)[R * PR + 2 * r]);
    float l = 0.0f;
    float4 v[DT / 4];
#pragma unroll
    for (int e = 0; e < DT / 4; ++e) v[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (unsigned m = members; m; m &= m - 1) {
      const float* p = piece(__ffs(m) - 1);
      const float w = pg_weight(p[R * PR + 2 * r], rf);
      l = fmaf(w, p[R * PR + 2 * r + 1], l);
#pragma unroll
      for (int e = 0; e < DT / 4; ++e) {
        const float4 y = *reinterpret_cast<const float4*>(p + r * PR + x0 + 32 * e);
        v[e].x = fmaf(w, y.x, v[e].x);
        v[e].y = fmaf(w, y.y, v[e].y);
        v[e].z = fmaf(w, y.z, v[e].z);
        v[e].w = fmaf(w, y.w, v[e].w);
      }
    }
    if (d.first && whole_last) {
      const PgSeq q = pg_seq<NG>(a, d.seq);
      const int rb = fdiv(d.sub, a.dKV), h = d.sub - rb * a.b.KV;
      if (pg_row_live(a, q, rb * R + r)) {
        const int64_t i0 = pg_out_row(a, q.qa, rb * R + r, h, D) + x0;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < DT / 4; ++e) {
          const float f[4] = {v[e].x * inv, v[e].y * inv, v[e].z * inv, v[e].w * inv};
          pg_store4(a, i0 + 32 * e, f);
        }
      }
    } else {  // left for the join
      const int slot = d.first && !a.whole ? 1 : 0;
      float* p = a.part + ((int64_t)blockIdx.x * 2 + slot) * pg_part_floats(D, NG);
#pragma unroll
      for (int e = 0; e < DT / 4; ++e) *reinterpret_cast<float4*>(p + r * D + x0 + 32 * e) = v[e];
      if (x0 == 0) {
        p[R * D + 2 * r] = rf;
        p[R * D + 2 * r + 1] = l;
        if (r == 0) s_out[slot] = PgDesc{d.seq, d.sub, d.first, whole_last};
      }
    }
  }
  __syncthreads();
  if (a.whole == 1) return;
  if (threadIdx.x < 2) a.desc[(int64_t)blockIdx.x * 2 + threadIdx.x] = s_out[threadIdx.x];
  if (a.whole == 0) return;
  // ---- the cluster's pieces of its item, in order, a share of the row's dims to each CTA ----
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  if (!working) return;
  const int cs = a.whole, rank = (int)blockIdx.x % cs, c0 = (int)blockIdx.x - rank;
  const PgAt at = s_at[0];  // (any place of the item: the plan's, or where its warp stopped)
  for (int x = rank * (32 * W) + (int)threadIdx.x; x < R * (D / 4); x += cs * (32 * W)) {
    const int r = x / (D / 4), d4 = x % (D / 4) * 4;
    float2 rs[kPgMaxCluster];
    float4 y[kPgMaxCluster];
    int has[kPgMaxCluster];
#pragma unroll
    for (int k = 0; k < kPgMaxCluster; ++k) {  // (all on their way at once; a CTA without a piece left anything)
      const int c = c0 + min(k, cs - 1);
      const float* p = a.part + (int64_t)c * 2 * pg_part_floats(D, NG);
      has[k] = k < cs ? __ldcg(&a.desc[(int64_t)c * 2].seq) : -1;
      rs[k] = __ldcg(reinterpret_cast<const float2*>(p + R * D + 2 * r));
      y[k] = __ldcg(reinterpret_cast<const float4*>(p + r * D + d4));
    }
    float rf = -INFINITY, l = 0.0f;
    bool any = false;
#pragma unroll
    for (int k = 0; k < kPgMaxCluster; ++k)
      if (has[k] >= 0) {
        any = true;
        rf = fmaxf(rf, rs[k].x);
      }
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < kPgMaxCluster; ++k)
      if (has[k] >= 0) {
        const float w = pg_weight(rs[k].x, rf);
        l = fmaf(w, rs[k].y, l);
        v.x = fmaf(w, y[k].x, v.x);
        v.y = fmaf(w, y[k].y, v.y);
        v.z = fmaf(w, y[k].z, v.z);
        v.w = fmaf(w, y[k].w, v.w);
      }
    const int rb = fdiv(at.sub, a.dKV), h = at.sub - rb * a.b.KV;
    if (any && pg_row_live(a, at.q, rb * R + r)) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const float f[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
      pg_store4(a, pg_out_row(a, at.q.qa, rb * R + r, h, D) + d4, f);
    }
  }
}

// Items cut between CTAs: CTA c joins the item that c begins and does not
// finish, over the following CTAs' first pieces, in their order.  The threads
// of a row and dim share the pieces among kGrp groups, whose sums are added
// in order.
constexpr int kPgJoinThreads = 512;
static_assert(kPgJoinThreads >= kPgMaxCtas, "");
template <int D, int NG>
__global__ void __launch_bounds__(kPgJoinThreads) attn_paged_join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int R = pg_rows(NG), V = R * D / 4, kGrp = kPgJoinThreads / V;
  __shared__ float s_ref[kPgMaxCtas][R], s_sum[kPgMaxCtas][R];
  __shared__ float4 s_v[kPgJoinThreads];
  __shared__ int s_n;
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.x, nc = gridDim.x;
  const PgDesc d = a.desc[(int64_t)c * 2 + 1];
  if (d.seq < 0) return;
  if (threadIdx.x == 0) s_n = nc - c - 1;
  __syncthreads();
  if ((int)threadIdx.x < nc - c - 1) {  // the following CTAs' first pieces, up to the item's end
    const PgDesc e = a.desc[(int64_t)(c + 1 + threadIdx.x) * 2];
    const bool same = e.seq == d.seq && e.sub == d.sub;
    if (!same || e.last) atomicMin(&s_n, (int)threadIdx.x + (same ? 1 : 0));
  }
  __syncthreads();
  const int n = 1 + s_n;  // pieces
  auto part = [&](int i) -> const float* {
    return a.part + ((int64_t)(c + i) * 2 + (i == 0 ? 1 : 0)) * pg_part_floats(D, NG);
  };
  for (int i = threadIdx.x; i < n * R; i += kPgJoinThreads) {
    const float* p = part(i / R) + R * D + 2 * (i % R);
    s_ref[i / R][i % R] = p[0];
    s_sum[i / R][i % R] = p[1];
  }
  __syncthreads();
  const int grp = threadIdx.x / V, x = threadIdx.x % V, r = x / (D / 4), d4 = (x % (D / 4)) * 4;
  float rf = -INFINITY;
  for (int i = 0; i < n; ++i) rf = fmaxf(rf, s_ref[i][r]);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = grp; i < n; i += kGrp) {
    const float4 p = *reinterpret_cast<const float4*>(part(i) + r * D + d4);
    const float w = pg_weight(s_ref[i][r], rf);
    v.x = fmaf(w, p.x, v.x);
    v.y = fmaf(w, p.y, v.y);
    v.z = fmaf(w, p.z, v.z);
    v.w = fmaf(w, p.w, v.w);
  }
  s_v[threadIdx.x] = v;
  __syncthreads();
  if (grp) return;
  float l = 0.0f;
  for (int i = 0; i < n; ++i) l = fmaf(pg_weight(s_ref[i][r], rf), s_sum[i][r], l);
#pragma unroll
  for (int k = 1; k < kGrp; ++k) {
    const float4 u = s_v[k * V + x];
    v.x += u.x;
    v.y += u.y;
    v.z += u.z;
    v.w += u.w;
  }
  const PgSeq q = pg_seq<NG>(a, d.seq);
  const int rb = fdiv(d.sub, a.dKV), h = d.sub - rb * a.b.KV;
  if (!pg_row_live(a, q, rb * R + r)) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const float f[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
  pg_store4(a, pg_out_row(a, q.qa, rb * R + r, h, D) + d4, f);
}

}  // namespace b2q
