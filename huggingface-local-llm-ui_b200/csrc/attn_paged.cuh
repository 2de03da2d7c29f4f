// attn_paged.cuh -- attention of the newest tokens of many sequences over
// their keys and values in the paged 4-bit cache (kv_page.cuh):
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - max),  j <= position.
//
// The cache is read once, 18 * D bytes for 16 keys and values of a head, and
// that stream is the floor; the work beside it is unpacking the codes.
//
// Items.  The query rows (token, head) of one sequence that share a K/V head
// are cut into blocks of 8 * NG rows; (sequence, row block, K/V head) is an
// item, its keys are cut into tiles of 64.  All items' tiles in one line are
// divided evenly over the CTAs and within a CTA over its warps, whatever the
// lengths (the lengths stay on the device, so a captured call follows them).
// A warp works alone on its tiles: a private ring of bulk copies (147 KB per
// SM over the eight warps), a running softmax, no barrier in the loop.  Items that end
// inside a warp's share are written at once; pieces of cut items meet in
// shared memory (a CTA's warps) and in the workspace (CTAs), where
// attn_paged_join_kernel adds them in order: the same bits every time.
//
// Products, on the warp-level tensor cores (mma.m16n8k16, f16 in, f32 out),
// with the codes as exact small integers and the f16 scales applied in f32:
//   S: A = queries (f32 queries as f16 hi rows 0-7 and lo rows 8-15 of one
//      tile, ~2^-22; 16-bit queries exactly, rows scaled by a power of two),
//      B = key codes; the sum over each 32 dims is multiplied by the key's scale;
//   O: A = value codes (16 dims x 16 keys), B = p_j * scale_j (f16 hi, and lo
//      where the output is f32), one B for each 32 dims.
// The softmax reference is shifted by the largest value scale seen, so that
// p_j * scale_j stays below 2^15 and out of f16's subnormals.
// Every tile's products are summed from zero in the matrix unit and added to
// the running f32 output with one fused multiply-add.
#pragma once

#include "kv_page.cuh"

namespace b2q {

constexpr int kPgWarps = 8, kPgThreads = kPgWarps * 32, kPgTile = 64;
constexpr int kPgChunk = 32;                    // sequences of one partial sum of the plan
constexpr int kPgMaxChunks = 65536 / kPgChunk;  // (n_seqs <= 65535)
__host__ __device__ constexpr int pg_stage_bytes(int D) { return kPgTile / kKvBlk * kv_blk_bytes(D); }
__host__ __device__ constexpr int pg_stages(int D) { return D == 128 ? 2 : 4; }
__host__ __device__ constexpr int pg_ring_bytes(int D) { return kPgWarps * pg_stages(D) * pg_stage_bytes(D); }
constexpr int kPgPad = 4;  // floats after a row of a piece in shared memory: its column stores fall on distinct banks
__host__ __device__ constexpr int pg_rows(int NG) { return 8 * NG; }
// one piece in the workspace: rows of D floats, then (reference, sum) pairs
__host__ __device__ constexpr int pg_part_floats(int D, int NG) { return pg_rows(NG) * (D + 2); }
// the same in shared memory
__host__ __device__ constexpr int pg_piece_floats(int D, int NG) { return pg_rows(NG) * (D + kPgPad + 2); }
// the ring, and behind it the piece each warp's share begins with; the pieces
// the shares end with take the ring's place
__host__ __device__ constexpr int pg_smem_bytes(int D, int NG) {
  return pg_ring_bytes(D) + kPgWarps * pg_piece_floats(D, NG) * 4;
}
constexpr int kPgMaxCtas = 256;

// Who a piece of an item belongs to, and whether it holds the item's first
// and last tile.  seq < 0: no piece.
struct PgDesc {
  int seq, sub, first, last;
};

struct PagedArgs {
  KvBatch b;
  int H, G;
  const void* q;
  int q_type;
  int64_t q_stride;
  const uint8_t* pages;
  float scale;
  void* out;
  int out_type;
  PgDesc* desc;  // [CTAs][2]: the piece begun before the CTA, the piece it begins
  float* part;   // [CTAs][2][pg_part_floats]
};

// The part of a sequence's geometry that the plan needs.
struct PgSeq {
  int qa, n;      // first row, rows of this call
  int base, len;  // position of the first row (may be negative), cached tokens
  int rows;       // n * G
  int nt, nrb;    // tiles of an item, row blocks
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
  s.base = s.len - n_all;
  s.rows = s.n * G;
  s.nt = s.len > kPgTile ? (s.len + kPgTile - 1) / kPgTile : 1;  // (one for none: its rows become zeros)
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
__device__ __forceinline__ int64_t pg_tiles(const PagedArgs& a, const PgSeq& q) { return (int64_t)q.nrb * a.b.KV * q.nt; }

// A place in the line of tiles.
struct PgAt {
  int seq, sub, tile;  // sub = row block * KV + K/V head
  PgSeq q;
};

template <int NG>
__device__ __forceinline__ void pg_next(const PagedArgs& a, PgAt& p, bool more) {
  if (++p.tile < p.q.nt) return;
  p.tile = 0;
  if (++p.sub < p.q.nrb * a.b.KV || !more) return;
  p.sub = 0;
  do {
    ++p.seq;
    if (p.seq >= a.b.n_seqs) {  // (the arrays changed under the kernel)
      p.seq = a.b.n_seqs - 1;
      return;
    }
    p.q = pg_seq<NG>(a, p.seq);
  } while (p.q.nrb == 0);
}

// Keys of an item: those its last row attends.
template <int NG>
__device__ __forceinline__ int pg_keys(const PagedArgs& a, const PgAt& p) {
  const int rb = p.sub / a.b.KV;
  const int last = (min(p.q.rows, (rb + 1) * pg_rows(NG)) - 1) / a.G;
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

__device__ __forceinline__ uint32_t h2_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u32_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// code - 8 of nibbles 0 and 1 (from the low end) of both 16-bit halves of w,
// as f16 pairs: 1024 + code and 1024 + 16 code are f16 numbers whose low bits
// are the code's, so one OR and one exact add or multiply-add make the value.
__device__ __forceinline__ void pg_unpack2(uint32_t w, uint32_t& n0, uint32_t& n1) {
  const uint32_t x0 = (w & 0x000f000fu) | 0x64006400u, x1 = (w & 0x00f000f0u) | 0x64006400u;
  n0 = h2_u32(__hadd2(u32_h2(x0), __floats2half2_rn(-1032.0f, -1032.0f)));
  n1 = h2_u32(__hfma2(u32_h2(x1), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.0f, -72.0f)));
}

__device__ __forceinline__ void pg_store(const PagedArgs& a, int64_t i, float v) {
  if (a.out_type == kElF32) reinterpret_cast<float*>(a.out)[i] = v;
  else if (a.out_type == kElF16) reinterpret_cast<__half*>(a.out)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(v);
}
// Index of row r (of a sequence from row qa on) of K/V head h in out (and, with
// the token stride, in q).
__device__ __forceinline__ int64_t pg_out_row(const PagedArgs& a, int qa, int r, int h, int D) {
  return ((int64_t)(qa + r / a.G) * a.H + h * a.G + r % a.G) * D;
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

template <int D, int NG, bool PSPLIT>
__global__ void __launch_bounds__(kPgThreads, 1) attn_paged_kernel(const __grid_constant__ PagedArgs a) {
  extern __shared__ __align__(128) uint8_t pg_smem[];
  constexpr int S = pg_stages(D), SB = pg_stage_bytes(D), BB = kv_blk_bytes(D);
  constexpr int NB = D / 32, R = pg_rows(NG), PR = D + kPgPad;
  constexpr bool QSPLIT = NG == 1;
  __shared__ uint64_t bars[kPgWarps][S];
  __shared__ PgDesc s_desc[kPgWarps][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();

  // ---- plan: this warp's share of the line of tiles ----
  int64_t* sums = reinterpret_cast<int64_t*>(pg_smem);  // tiles of 32 sequences each (the ring's place)
  const int nch = (a.b.n_seqs + kPgChunk - 1) / kPgChunk;
  for (int c = warp; c < nch; c += kPgWarps) {
    const int s = c * kPgChunk + lane;
    long long w = 0;
    if (s < a.b.n_seqs) w = pg_tiles(a, pg_seq<NG>(a, s));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(B2Q_FULL, w, o);
    if (lane == 0) sums[c] = w;
  }
  if (threadIdx.x < kPgWarps * S) mbar_init(&bars[0][0] + threadIdx.x, 1);
  if (threadIdx.x < kPgWarps * 2) (&s_desc[0][0])[threadIdx.x].seq = -1;
  fence_mbar_init();
  __syncthreads();
  long long total = 0;
  for (int c = lane; c < nch; c += 32) total += sums[c];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(B2Q_FULL, total, o);
  // a CTA takes at least a tile for each of its warps
  const int nc = (int)min((long long)gridDim.x, (total + kPgWarps - 1) / kPgWarps);
  long long w0 = 0, w1 = 0;
  if ((int)blockIdx.x < nc) {
    const long long c0 = total * blockIdx.x / nc, c1 = total * (blockIdx.x + 1) / nc;
    w0 = c0 + (c1 - c0) * warp / kPgWarps;
    w1 = c0 + (c1 - c0) * (warp + 1) / kPgWarps;
  }
  const long long count = w1 - w0;
  PgAt at{};
  if (count > 0) {
    long long rest = w0;  // tiles before the share, from the place searched
    int ch = 0;
    for (int c0 = 0; c0 < nch; c0 += 32) {
      long long v = c0 + lane < nch ? sums[c0 + lane] : 0, inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(B2Q_FULL, inc, o);
        if (lane >= o) inc += u;
      }
      const unsigned hit = __ballot_sync(B2Q_FULL, inc > rest);
      if (hit) {
        const int l = __ffs(hit) - 1;
        ch = c0 + l;
        rest -= __shfl_sync(B2Q_FULL, inc - v, l);
        break;
      }
      rest -= __shfl_sync(B2Q_FULL, inc, 31);
    }
    const int s = ch * kPgChunk + lane;
    PgSeq q{};
    long long v = 0;
    if (s < a.b.n_seqs) {
      q = pg_seq<NG>(a, s);
      v = pg_tiles(a, q);
    }
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(B2Q_FULL, inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned hit = __ballot_sync(B2Q_FULL, inc > rest);
    const int l = hit ? __ffs(hit) - 1 : 0;
    rest -= __shfl_sync(B2Q_FULL, inc - v, l);
    at.seq = min(ch * kPgChunk + l, a.b.n_seqs - 1);
    at.q = pg_seq<NG>(a, at.seq);
    at.sub = (int)(rest / at.q.nt);
    at.tile = (int)(rest - (long long)at.sub * at.q.nt);
  }
  fence_proxy_async_smem();  // the plan's sums were in the ring's place
  __syncthreads();

  // ---- the ring: copies run S - 1 tiles ahead; a tile's page numbers are
  // fetched one tile before its copies are issued ----
  uint8_t* ring = pg_smem + warp * S * SB;
  const int bpp = a.b.page_tokens / kKvBlk;
  PgAt ld = at;
  long long loaded = 0;  // tiles whose page numbers were fetched
  int64_t blk_next = -1;  // lane j < 4: block j of the next tile to copy, -1: none
  uint32_t valid = 0;    // 4 bits for each of the last stages: blocks that hold keys
  auto fetch = [&]() {
    blk_next = -1;
    if (loaded >= count) return;
    if (lane < kPgTile / kKvBlk) {
      const int pos = ld.tile * kPgTile + lane * kKvBlk;
      if (pos < pg_keys<NG>(a, ld)) {
        const int64_t blk = kv_block_of(a.b, ld.seq, pos);
        if (blk >= 0) blk_next = blk + (int64_t)(ld.sub % a.b.KV) * bpp;
      }
    }
    ++loaded;
    pg_next<NG>(a, ld, loaded < count);
  };
  int ist = 0;           // the stage of the next copies
  long long issued = 0;
  auto issue = [&]() {  // copies of the next tile (its page numbers are in blk_next)
    const int st = ist;
    ist = ist + 1 == S ? 0 : ist + 1;
    ++issued;
    const unsigned m = __ballot_sync(B2Q_FULL, blk_next >= 0);
    valid = (valid & ~(15u << (4 * st))) | ((m & 15u) << (4 * st));
    if (lane == 0) mbar_arrive_expect_tx(&bars[warp][st], __popc(m) * BB);
    __syncwarp();
    if (blk_next >= 0) bulk_g2s(ring + st * SB + lane * BB, a.pages + blk_next * BB, BB, &bars[warp][st]);
  };
  fetch();
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < count) {
      issue();
      fetch();
    }

  // ---- the running state of an item's rows ----
  uint32_t qa[D / 16][4];
  float o[NG][D / 16][4];
  float mx[NG], ref[NG], sum[NG], fac[NG];
  int lim[NG];
  int ev = -24;   // exponent of the largest value scale so far
  int keys = 0, min_lim = 0;
  auto begin = [&]() {
    const int rb = at.sub / a.b.KV, h = at.sub - rb * a.b.KV;
    keys = pg_keys<NG>(a, at);
    float qv[NG][NB][8];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int r = rb * R + 8 * n + g;
      const bool live = r < at.q.rows;
      lim[n] = live ? at.q.base + r / a.G : keys - 1;
      float am = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (live) {
          const int64_t i = (int64_t)(at.q.qa + r / a.G) * a.q_stride + (h * a.G + r % a.G) * D + 32 * b + 8 * t;
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
      fac[n] = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - 13 + e) << 23);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int x = 0; x < 8; ++x) qv[n][b][x] *= sc;
      mx[n] = ref[n] = -INFINITY;
      sum[n] = 0.0f;
#pragma unroll
      for (int m = 0; m < D / 16; ++m) o[n][m][0] = o[n][m][1] = o[n][m][2] = o[n][m][3] = 0.0f;
    }
    min_lim = min(at.q.base + (rb * R) / a.G, keys - 1);
    ev = -24;
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
          f[1] = h2_u32(__floats2half2_rn(qv[NG - 1][b][x], qv[NG - 1][b][x + 4]));
        }
      }
  };

  float* const piece0 = reinterpret_cast<float*>(pg_smem + pg_ring_bytes(D)) + warp * pg_piece_floats(D, NG);
  bool tail = false;      // the share ends with a piece
  int first = 1;          // the piece holds the item's first tile
  bool fresh = true;      // begin() before the next tile
  int st = 0;             // the tile's stage and its barrier's phase
  uint32_t phase = 0;
  auto store_piece = [&](float* p) {  // the rows in hand, in shared memory
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
  for (long long i = 0; i < count; ++i) {
    if (fresh) {
      begin();
      first = at.tile == 0;
      fresh = false;
    }
    if (i + S - 1 < count) {
      issue();
      fetch();
    }
    const bool ok = __all_sync(B2Q_FULL, mbar_wait_bounded(&bars[warp][st], phase));
    if (!ok) {  // a wait gave up (the error word is set): first the copies in flight
      for (long long k = i; k < issued; ++k) {
        mbar_wait_bounded(&bars[warp][st], phase);
        if (++st == S) {
          st = 0;
          phase ^= 1;
        }
      }
      break;
    }
    const uint32_t vm = (valid >> (4 * st)) & 15u;
    const uint8_t* tb = ring + st * SB;
    const int key0 = at.tile * kPgTile;
    if (vm) {
      const bool edge = key0 + kPgTile - 1 > min_lim || vm != 15u;  // some key is not every row's
      // largest value scale of the tile (bits of f16 magnitudes order like the numbers)
      {
        constexpr int TL = 8 / NB;  // tokens of a 16-byte piece of scales
        constexpr int LB = kKvBlk / TL;  // pieces of a block
        uint32_t big = 0;
        if (lane < 4 * LB) {
          const int blk = lane / LB, tok = (lane % LB) * TL;
          const uint4 x = *reinterpret_cast<const uint4*>(tb + blk * BB + 17 * D + tok * NB * 2);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = key0 + blk * kKvBlk + tok + e * 2 / NB;
            const uint32_t x0 = w[e] & 0x7fffu, x1 = (w[e] >> 16) & 0x7fffu;
            const uint32_t m = max(x0 < 0x7c00u ? x0 : 0u, x1 < 0x7c00u ? x1 : 0u);  // (a NaN shows anyway)
            if (k < keys && ((vm >> blk) & 1)) big = max(big, m);
          }
        }
        big = __reduce_max_sync(B2Q_FULL, big);
        const int e = big >= 0x400u ? (int)(big >> 10) - 15 : big ? 7 - __clz(big) : -24;
        ev = max(ev, e);  // (subnormal: the leading bit's place, 2^-24 upward)
      }
      // ---- S ----
      float s[NG][8][2];
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        const uint8_t* kb = tb + (nt >> 1) * BB;
        uint32_t w[NB], sc[NB];  // codes of the lane's 8 dims of each block; scales [token][block pairs]
        if (NB == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(kb + (nt & 1) * 4 * D + lane * (D / 8));
          const uint4 y = *reinterpret_cast<const uint4*>(kb + 8 * D + ((nt & 1) * 8 + 2 * t) * NB * 2);
          w[0] = x.x; w[1] = x.y; w[NB - 2] = x.z; w[NB - 1] = x.w;
          sc[0] = y.x; sc[1] = y.y; sc[NB - 2] = y.z; sc[NB - 1] = y.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(kb + (nt & 1) * 4 * D + lane * (D / 8));
          const uint2 y = *reinterpret_cast<const uint2*>(kb + 8 * D + ((nt & 1) * 8 + 2 * t) * NB * 2);
          w[0] = x.x; w[1] = x.y;
          sc[0] = y.x; sc[1] = y.y;
        }
        float2 d0[NB / 2], d1[NB / 2];  // scales of the lane's two keys
#pragma unroll
        for (int b = 0; b < NB / 2; ++b) {
          d0[b] = __half22float2(u32_h2(sc[b]));
          d1[b] = __half22float2(u32_h2(sc[NB / 2 + b]));
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) s[n][nt][0] = s[n][nt][1] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          uint32_t n0, n1;
          pg_unpack2(w[b], n0, n1);
          pg_mma(c, qa[2 * b], n0, n1);
          pg_unpack2(w[b] >> 8, n0, n1);
          pg_mma(c, qa[2 * b + 1], n0, n1);
          const float e0 = (b & 1) ? d0[b >> 1].y : d0[b >> 1].x, e1 = (b & 1) ? d1[b >> 1].y : d1[b >> 1].x;
          if (QSPLIT) {
            s[0][nt][0] = fmaf(c[0] + c[2], e0, s[0][nt][0]);
            s[0][nt][1] = fmaf(c[1] + c[3], e1, s[0][nt][1]);
          } else {
            s[0][nt][0] = fmaf(c[0], e0, s[0][nt][0]);
            s[0][nt][1] = fmaf(c[1], e1, s[0][nt][1]);
            s[NG - 1][nt][0] = fmaf(c[2], e0, s[NG - 1][nt][0]);
            s[NG - 1][nt][1] = fmaf(c[3], e1, s[NG - 1][nt][1]);
          }
        }
      }
      // ---- softmax: p into s ----
      float corr[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float tm = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[n][nt][e] *= fac[n];
            if (edge) {
              const int k = key0 + 8 * nt + 2 * t + e;
              if (k > lim[n] || k >= keys || !((vm >> (nt >> 1)) & 1)) s[n][nt][e] = -INFINITY;
            }
            tm = fmaxf(tm, s[n][nt][e]);
          }
        tm = fmaxf(tm, __shfl_xor_sync(B2Q_FULL, tm, 1));
        tm = fmaxf(tm, __shfl_xor_sync(B2Q_FULL, tm, 2));
        mx[n] = fmaxf(mx[n], tm);
        float nref = 0.0f;
        corr[n] = 1.0f;
        if (mx[n] != -INFINITY) {
          nref = mx[n] + (float)(ev - 14);
          corr[n] = pg_weight(ref[n], nref);
          ref[n] = nref;
        }
        float ps = 0.0f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[n][nt][e] = pg_exp2(s[n][nt][e] - nref);
            ps += s[n][nt][e];
          }
        sum[n] = fmaf(sum[n], corr[n], ps);
      }
      // a row's factor at the lanes that hold its outputs (rows 2t, 2t + 1)
      float cr[NG][2];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        cr[n][0] = __shfl_sync(B2Q_FULL, corr[n], 8 * t);
        cr[n][1] = __shfl_sync(B2Q_FULL, corr[n], 8 * t + 4);
      }
      // ---- O, half the dims at a time ----
      constexpr int HB = NB >= 2 ? NB / 2 : 1;  // 32-dim blocks of a half
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float ta[NG][2 * HB][4];
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int m = 0; m < 2 * HB; ++m) ta[n][m][0] = ta[n][m][1] = ta[n][m][2] = ta[n][m][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* vb = tb + j * BB + 9 * D;
          uint32_t va[2][2];  // [key pair][key]: the half's codes of the lane's dims
          uint32_t sc[2][2];  // [key pair][key]: the half's scales (f16 pair, or one)
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) {
            const uint8_t* vp = vb + pr * 4 * D + lane * (D / 8);
            const uint8_t* sp = vb + 8 * D + (pr * 8 + 2 * t) * NB * 2;
            if (NB == 4) {
              const uint4 x = *reinterpret_cast<const uint4*>(vp);
              const uint4 y = *reinterpret_cast<const uint4*>(sp);
              va[pr][0] = half ? x.y : x.x;
              va[pr][1] = half ? x.w : x.z;
              sc[pr][0] = half ? y.y : y.x;
              sc[pr][1] = half ? y.w : y.z;
            } else {  // one block of 32 dims: four nibbles, one scale
              const uint2 x = *reinterpret_cast<const uint2*>(vp);
              const uint2 y = *reinterpret_cast<const uint2*>(sp);
              va[pr][0] = half ? x.x >> 16 : x.x;
              va[pr][1] = half ? x.y >> 16 : x.y;
              sc[pr][0] = half ? y.x >> 16 : y.x;
              sc[pr][1] = half ? y.y >> 16 : y.y;
            }
          }
#pragma unroll
          for (int b = 0; b < HB; ++b) {
            // A: dims of two tiles of 16, keys pairwise
            uint32_t f[2][4];
#pragma unroll
            for (int pr = 0; pr < 2; ++pr) {
              const uint32_t w = __byte_perm(va[pr][0], va[pr][1], b ? 0x7632 : 0x5410);
              pg_unpack2(w, f[0][2 * pr], f[0][2 * pr + 1]);
              pg_unpack2(w >> 8, f[1][2 * pr], f[1][2 * pr + 1]);
            }
            float dv[2][2];
#pragma unroll
            for (int pr = 0; pr < 2; ++pr)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 d = __half22float2(u32_h2(sc[pr][e]));
                dv[pr][e] = b ? d.y : d.x;
              }
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              uint32_t hi[2], lo[2];
#pragma unroll
              for (int pr = 0; pr < 2; ++pr) {
                float x0 = s[n][2 * j + pr][0] * dv[pr][0], x1 = s[n][2 * j + pr][1] * dv[pr][1];
                if (edge) {  // what no row sees may hold anything
                  x0 = s[n][2 * j + pr][0] == 0.0f ? 0.0f : x0;
                  x1 = s[n][2 * j + pr][1] == 0.0f ? 0.0f : x1;
                }
                const __half2 h = __floats2half2_rn(x0, x1);
                hi[pr] = h2_u32(h);
                if (PSPLIT) {
                  const float2 hf = __half22float2(h);
                  lo[pr] = h2_u32(__floats2half2_rn(x0 - hf.x, x1 - hf.y));
                }
              }
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                // rows g are nibble 0 / 2 of a pair, rows g + 8 nibble 1 / 3
                pg_mma(ta[n][2 * b + m], f[m], hi[0], hi[1]);
                if (PSPLIT) pg_mma(ta[n][2 * b + m], f[m], lo[0], lo[1]);
              }
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int m = 0; m < 2 * HB; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& x = o[n][half * 2 * HB + m][e];
              x = fmaf(x, cr[n][e & 1], ta[n][m][e]);
            }
      }
    }
    __syncwarp();  // the stage is free for the copy of tile i + S
    // ---- the item, or this warp's share of it, ends ----
    const bool last = at.tile + 1 == at.q.nt;
    if (last || i + 1 == count) {
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        sum[n] += __shfl_xor_sync(B2Q_FULL, sum[n], 1);
        sum[n] += __shfl_xor_sync(B2Q_FULL, sum[n], 2);
      }
      if (first && last) {
        const int rb = at.sub / a.b.KV, h = at.sub - rb * a.b.KV;
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float l = __shfl_sync(B2Q_FULL, sum[n], 8 * t + 4 * e);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int r = rb * R + 8 * n + 2 * t + e;
            if (r < at.q.rows) {
              const int64_t i0 = pg_out_row(a, at.q.qa, r, h, D);
#pragma unroll
              for (int m = 0; m < D / 16; ++m) {
                pg_store(a, i0 + 16 * m + g, o[n][m][e] * inv);
                pg_store(a, i0 + 16 * m + 8 + g, o[n][m][2 + e] * inv);
              }
            }
          }
      } else if (i + 1 < count) {  // begun before this share
        store_piece(piece0);
        if (lane == 0) s_desc[warp][0] = PgDesc{at.seq, at.sub, 0, 1};
      } else {  // the share's last stays in registers until every warp is done with the ring
        tail = true;
        if (lane == 0) s_desc[warp][1] = PgDesc{at.seq, at.sub, first, last};
      }
      fresh = true;
    }
    if (++st == S) {
      st = 0;
      phase ^= 1;
    }
    if (i + 1 < count) pg_next<NG>(a, at, true);
  }
  __syncthreads();

  // ---- the CTA's pieces, in order: joined here when whole ----
  auto piece = [&](int i) -> float* {  // slot i = 2 * warp + (begun before it: 0, its last: 1)
    return reinterpret_cast<float*>((i & 1) ? pg_smem : pg_smem + pg_ring_bytes(D)) + (i >> 1) * pg_piece_floats(D, NG);
  };
  if (tail) store_piece(piece(2 * warp + 1));
  __syncthreads();
  const PgDesc* sd = &s_desc[0][0];
  PgDesc out_desc[2];
  out_desc[0].seq = out_desc[1].seq = -1;
  for (int i = 0; i < 2 * kPgWarps;) {
    const PgDesc d = sd[i];
    if (d.seq < 0) {
      ++i;
      continue;
    }
    int j = i + 1, end = i;  // the run of pieces of the same item
    for (; j < 2 * kPgWarps; ++j) {
      if (sd[j].seq < 0) continue;
      if (sd[j].seq != d.seq || sd[j].sub != d.sub) break;
      end = j;
    }
    const int whole_last = sd[end].last;
    const bool whole = d.first && whole_last;
    const int slot = d.first ? 1 : 0;
    if (!whole) out_desc[slot] = PgDesc{d.seq, d.sub, d.first, whole_last};
    for (int r = warp; r < R; r += kPgWarps) {
      float rf = -INFINITY;
      for (int k = i; k <= end; ++k)
        if (sd[k].seq >= 0) rf = fmaxf(rf, piece(k)[R * PR + 2 * r]);
      float l = 0.0f, v[D / 32];
#pragma unroll
      for (int e = 0; e < D / 32; ++e) v[e] = 0.0f;
      for (int k = i; k <= end; ++k) {
        if (sd[k].seq < 0) continue;
        const float* p = piece(k);
        const float w = pg_weight(p[R * PR + 2 * r], rf);
        l = fmaf(w, p[R * PR + 2 * r + 1], l);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) v[e] = fmaf(w, p[r * PR + lane + 32 * e], v[e]);
      }
      if (whole) {
        const PgSeq q = pg_seq<NG>(a, d.seq);
        const int rb = d.sub / a.b.KV, h = d.sub - rb * a.b.KV;
        if (rb * R + r < q.rows) {
          const int64_t i0 = pg_out_row(a, q.qa, rb * R + r, h, D);
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
          for (int e = 0; e < D / 32; ++e) pg_store(a, i0 + lane + 32 * e, v[e] * inv);
        }
      } else {
        float* p = a.part + ((int64_t)blockIdx.x * 2 + slot) * pg_part_floats(D, NG);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) p[r * D + lane + 32 * e] = v[e];
        if (lane == 0) {
          p[R * D + 2 * r] = rf;
          p[R * D + 2 * r + 1] = l;
        }
      }
    }
    i = end + 1;
  }
  if (threadIdx.x < 2) a.desc[(int64_t)blockIdx.x * 2 + threadIdx.x] = out_desc[threadIdx.x];
}

// Items cut between CTAs: CTA c joins the item that c begins and does not
// finish, over the following CTAs' first pieces, in their order.  The threads
// of a row and dim share the pieces among kGrp groups, whose sums are added
// in order.
constexpr int kPgJoinThreads = 512;
template <int D, int NG>
__global__ void __launch_bounds__(kPgJoinThreads) attn_paged_join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int R = pg_rows(NG), V = R * D / 4, kGrp = kPgJoinThreads / V;
  __shared__ float s_ref[kPgMaxCtas][R], s_sum[kPgMaxCtas][R];
  __shared__ float4 s_v[kPgJoinThreads];
  pdl_wait();
  const int c = blockIdx.x, nc = gridDim.x;
  const PgDesc d = a.desc[(int64_t)c * 2 + 1];
  if (d.seq < 0) return;
  int n = 1;  // pieces
  for (int k = c + 1; k < nc; ++k) {
    const PgDesc e = a.desc[(int64_t)k * 2];
    if (e.seq != d.seq || e.sub != d.sub) break;
    ++n;
    if (e.last) break;
  }
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
  const int rb = d.sub / a.b.KV, h = d.sub - rb * a.b.KV;
  if (rb * R + r >= q.rows) return;
  const int64_t i0 = pg_out_row(a, q.qa, rb * R + r, h, D) + d4;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  pg_store(a, i0, v.x * inv);
  pg_store(a, i0 + 1, v.y * inv);
  pg_store(a, i0 + 2, v.z * inv);
  pg_store(a, i0 + 3, v.w * inv);
}

}  // namespace b2q
