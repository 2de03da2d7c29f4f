// kv_page.cuh -- the paged K/V cache of many sequences, held in 4 bits: its
// layout, the append (position rotation and quantisation on the way) and the
// read-back.
//
// The pool is [n_pages][n_kv_heads][page_tokens / 16] blocks; a block holds
// 16 consecutive tokens of one K/V head in 18 * D bytes (D = head_dim):
//   [0, 8D)     key codes       token row of D/2 bytes: words [t 0..3][b 0..D/32-1],
//                               word (t, b) = dims 32b + 8t + n in nibble n
//   [8D, 9D)    key scales      [16][D/32] f16
//   [9D, 17D)   value codes     pieces [tok / 8][g 0..7][tok%8 / 2][tok % 2] of D/16
//                               bytes, nibble j = dim 8j + g
//   [17D, 18D)  value scales    [16][D/32] f16
// A value is (code - 8) * scale, GGML's 4-bit block (one f16 scale to 32
// values), with the bytes of 16 tokens arranged as the operand fragments of
// the attention's matrix instructions (attn_paged.cuh): every lane finds its
// codes in one 16-byte load, without bank conflicts.
//
// A batch names its tokens by three device arrays: sequence s has the packed
// rows q_start[s] .. q_start[s+1]-1, they are the LAST n of its kv_len[s]
// cached tokens, and position p lies in page page_table[s][p / page_tokens].
// Nothing read from the device is trusted: a position or page out of range
// sets g_b2q_batch_error and its token is skipped.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "quant.cuh"

// Set (to 1) by a kernel that met a position, page or offset out of range in
// a batch's device arrays; read and cleared by b2q_check_device_error().
__device__ int g_b2q_batch_error = 0;

namespace b2q {

constexpr int kKvBlk = 16;  // tokens of a block
__host__ __device__ constexpr int kv_blk_bytes(int D) { return 18 * D; }

enum ElemType : int { kElF32 = 0, kElF16 = 1, kElBF16 = 2 };

template <int T>
struct Elem;
template <>
struct Elem<kElF32> { typedef float type; };
template <>
struct Elem<kElF16> { typedef __half type; };
template <>
struct Elem<kElBF16> { typedef __nv_bfloat16 type; };

__device__ __forceinline__ float el_f(float v) { return v; }
__device__ __forceinline__ float el_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float el_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T el_from(float v);
template <>
__device__ __forceinline__ float el_from<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half el_from<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 el_from<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two values as one word of the 16-bit type T (the first in the low half).
template <typename T>
__device__ __forceinline__ uint32_t el_pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t el_pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t el_pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four consecutive elements (16-byte aligned as f32, 8-byte as 16-bit types).
__device__ __forceinline__ void ld4(const float* p, float (&v)[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
template <typename T>
__device__ __forceinline__ void ld4(const T* p, float (&v)[4]) {
  const uint2 x = *reinterpret_cast<const uint2*>(p);
  const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = el_f(e[i]);
}
__device__ __forceinline__ void st4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <typename T>
__device__ __forceinline__ void st4(T* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(el_pack2<T>(v[0], v[1]), el_pack2<T>(v[2], v[3]));
}

// What the kernels need of b2q_kv_config and b2q_kv_batch.
struct KvBatch {
  int n_seqs, n_tokens, KV, D, page_tokens, n_pages, max_pages;
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* page_table;
};

__device__ __forceinline__ void kv_batch_error() { *(volatile int*)&g_b2q_batch_error = 1; }

// Offset in the pool (in blocks) of position `pos` of sequence s for K/V head
// 0, or -1 (and the error word) if the position or its page is out of range.
// Blocks of head h follow at + h * page_tokens / 16.
__device__ __forceinline__ int64_t kv_block_of(const KvBatch& b, int s, int pos) {
  const int pg = pos / b.page_tokens;
  if (pos < 0 || pg >= b.max_pages) {
    kv_batch_error();
    return -1;
  }
  const int page = b.page_table[(int64_t)s * b.max_pages + pg];
  if (page < 0 || page >= b.n_pages) {
    kv_batch_error();
    return -1;
  }
  const int bpp = b.page_tokens / kKvBlk;
  return (int64_t)page * b.KV * bpp + (pos - pg * b.page_tokens) / kKvBlk;
}

// Position `back` tokens before the end of a sequence of `len`; below zero: -1.
__device__ __forceinline__ int kv_pos_of(int len, int back) { return len < back ? -1 : len - back; }

// Position of packed row t if it is one of sequence s.  False for rows behind
// the last sequence, and (with the error word) for offsets that make no sense.
__device__ __forceinline__ bool kv_row_in(const KvBatch& b, int t, int s, int& pos) {
  if (s >= b.n_seqs) return false;
  const int a = b.q_start[s], e = b.q_start[s + 1], len = b.kv_len[s];
  if (a < 0 || t < a || t >= e) {
    kv_batch_error();
    return false;
  }
  pos = kv_pos_of(len, e - t);
  return true;
}

// Sequence and position of packed row t (one thread).  False for rows behind
// the last sequence, and (with the error word) for offsets that make no sense.
__device__ __forceinline__ bool kv_row_of(const KvBatch& b, int t, int& seq, int& pos) {
  int lo = 0, hi = b.n_seqs;  // the number of q_start[1..n_seqs] <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (b.q_start[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  seq = lo;
  return kv_row_in(b, t, lo, pos);
}

// ---------------------------------------------------------------------------
// Append.  A warp takes a row (a head of a token) of D = 128 at a time, two rows
// of D = 64; a lane holds four consecutive dims.
// Rotation (rot_dim r, a multiple of 8; pairs (i, i + r/2)): each product and
// sum rounded to f32 by itself, so that the 4-bit codes are those of the
// formula evaluated in f32 step by step.
// Quantisation of 32 values: m the first value of the largest magnitude,
// scale d = f16(m / -8), kept finite; code = clamp(round(x / d) + 8, 0, 15),
// rounding halves to even.  A block with an infinity or a NaN gets a NaN
// scale: its values read back as NaN, the damage stays where it was written.
// ---------------------------------------------------------------------------
struct AppendArgs {
  KvBatch b;
  int H;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int rot_dim, n_pos;
  const float *cos, *sin;
  uint8_t* pages;
  void* q_out;
};

// Quantise the row x (lane l of it: dims 4l..4l+3) as keys or values into token
// tok of the block at blk.  All lanes of the warp take part, live ones store.
template <int D, bool V>
__device__ __forceinline__ void kv_store_row(uint8_t* blk, int tok, const float (&x)[4], int l, bool live) {
  constexpr int NB = D / 32;
  const int lane = threadIdx.x & 31;
  // the first value of the largest magnitude among the eight lanes of a block of
  // 32 (magnitudes order like their bits, infinities and NaN above all numbers)
  uint32_t ab[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) ab[i] = __float_as_uint(x[i]) & 0x7fffffffu;
  uint32_t big = max(max(ab[0], ab[1]), max(ab[2], ab[3]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) big = max(big, __shfl_xor_sync(B2Q_FULL, big, o));
  float m = x[3];
  bool has = ab[3] == big;
#pragma unroll
  for (int i = 2; i >= 0; --i)
    if (ab[i] == big) { m = x[i]; has = true; }
  const unsigned at = __ballot_sync(B2Q_FULL, has);
  m = __shfl_sync(B2Q_FULL, m, (lane & 24) + __ffs(at >> (lane & 24) & 255u) - 1);
  const bool fin = big < 0x7f800000u;
  // m / -8 beyond f16 keeps the largest finite scale
  const __half dh = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
  const float d = __half2float(dh);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
  // code = round(x / d) + 8: a sum with 1.5 * 2^23 + 8 is rounded to whole numbers,
  // halves to even, and has the code in its low bits.  x * (1 / d) is off by less
  // than 2^-18, so only a product that close to a half asks for the division.
  constexpr float kRound = 12582920.0f;
  uint32_t pk = 0;
  float far = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = fminf(fmaxf(x[i] * inv, -8.0f), 7.0f), r = q + kRound;
    far = fmaxf(far, fabsf(q - (r - kRound)));
    pk |= (__float_as_uint(r) & 15u) << (4 * i);
  }
  if (far > 0.49999f) {
    pk = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      pk |= (__float_as_uint(fminf(fmaxf(__fdiv_rn(x[i], d), -8.0f), 7.0f) + kRound) & 15u) << (4 * i);
  }
  if (!fin || d == 0.0f) pk = 0x8888u;
  uint8_t* base = blk + (V ? 9 * D : 0);
  if (live && (l & 7) == 0)
    *reinterpret_cast<unsigned short*>(base + 8 * D + (tok * NB + (l >> 3)) * 2) = fin ? __half_as_ushort(dh) : (unsigned short)0x7fff;
  if (!V) {
    const uint32_t nb = __shfl_xor_sync(B2Q_FULL, pk, 1);
    if (live && (l & 1) == 0) {
      const int u = l >> 1;  // dims 8u..8u+7
      *reinterpret_cast<uint32_t*>(base + tok * (D / 2) + (u & 3) * (D / 8) + (u >> 2) * 4) = pk | (nb << 16);
    }
    return;
  }
  // values: nibble j of piece g is dim 8j + g, held by lane 2j + (g >> 2).  Eight
  // lanes of the same half of g exchange what is not theirs, nibbles first, then
  // bytes, then halves of words.
  const int j = l >> 1;
  const bool b0 = j & 1, b1 = j & 2, b2 = j & 4;
  uint32_t other = __shfl_xor_sync(B2Q_FULL, b0 ? pk & 0xffu : pk >> 8, 2);
  const uint32_t mine = b0 ? pk >> 8 : pk & 0xffu;
  const uint32_t ev = b0 ? other : mine, od = b0 ? mine : other;
  const uint32_t by = (ev & 15u) | (od & 15u) << 4 | (ev & 0xf0u) << 4 | (od & 0xf0u) << 8;
  other = __shfl_xor_sync(B2Q_FULL, b1 ? by & 0xffu : by >> 8, 4);
  const uint32_t hw = b1 ? other | (by >> 8) << 8 : (by & 0xffu) | other << 8;
  other = __shfl_xor_sync(B2Q_FULL, hw, 8);
  if (live && !b2) {
    const int g = 4 * (l & 1) + 2 * b0 + b1;
    *reinterpret_cast<uint32_t*>(base + (tok >> 3) * (4 * D) + g * (D / 2) + ((tok & 7) >> 1) * (D / 8) +
                                 (tok & 1) * (D / 16) + (j >> 3) * 4) = hw | other << 16;
  }
}

// By all threads of the grid: offsets that decrease set the error word (beside them the
// search for a row's sequence may miss rows).  `first` and `s_ends`: the CTA's copies of
// start[0] and start[1..n_seqs], where `cached`.
__device__ __forceinline__ void kv_check_offsets(const int32_t* start, int n_seqs, int first, const int* s_ends, bool cached) {
  constexpr unsigned kCtas = 256;  // (that share the work)
  if (cached) {
    if (blockIdx.x == 0 && blockIdx.y == 0)
      for (int i = threadIdx.x; i < n_seqs; i += blockDim.x)
        if (s_ends[i] < (i ? s_ends[i - 1] : first)) kv_batch_error();
  } else if (blockIdx.x < kCtas && blockIdx.y == 0) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n_seqs; i += min(gridDim.x, kCtas) * blockDim.x)
      if (start[i + 1] < start[i]) kv_batch_error();
  }
}

// Sequences of a batch whose offsets are copied to shared memory to be searched.
constexpr int kKvSeqs = 1024;

// By the first `rows` threads of a CTA: block and position of packed rows
// row0 .. row0 + rows - 1 (block -1: no row); s_start: [kKvSeqs + 1] for the sequences'
// ends and, last, the first one's start.
__device__ __forceinline__ void kv_rows_of(const KvBatch& b, int row0, int rows, int* s_start, int64_t* s_blk, int* s_pos) {
  const bool in_smem = b.n_seqs <= kKvSeqs;
  if (in_smem) {
    for (int i = threadIdx.x; i < b.n_seqs; i += blockDim.x) s_start[i] = b.q_start[i + 1];
    if (threadIdx.x == blockDim.x - 1) s_start[kKvSeqs] = b.q_start[0];
    __syncthreads();
  }
  if ((int)threadIdx.x < rows) {
    const int t = row0 + threadIdx.x;
    int64_t blk = -1;
    int pos = 0, seq = 0;
    if (t < b.n_tokens) {
      bool ok;
      if (in_smem) {
        int hi = b.n_seqs;
        while (seq < hi) {
          const int mid = (seq + hi) >> 1;
          if (s_start[mid] <= t) seq = mid + 1;
          else hi = mid;
        }
        ok = kv_row_in(b, t, seq, pos);
      } else {
        ok = kv_row_of(b, t, seq, pos);
      }
      if (ok) blk = kv_block_of(b, seq, pos);
    }
    s_blk[threadIdx.x] = blk;
    s_pos[threadIdx.x] = pos;
  }
  __syncthreads();
}

// A CTA takes TOK tokens: four, whose rows of a head a warp takes together; or
// one, where there are few, and a warp takes two of its rows.  The floor is the
// stream of rows in and out, and close behind it the quantiser's instructions: the
// kind of a row (query, key, value) is known to the code of its turn, and four
// CTAs share an SM (64 registers; the rotations come from L1 again for each row).
// 8192 tokens of 32 + 2 * 8 heads, f32 rows in and bf16 queries out: 73 us, 43 of them
// the stream at the copy's rate; 103 with the rotations in registers and two CTAs an SM.  The first
// rows are on their way before it is known where they go (sequence, page: three
// dependent loads).
constexpr int kAppendThreads = 256;

template <int D, int XT, int OT, int TOK>
__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_kernel(const __grid_constant__ AppendArgs a) {
  typedef typename Elem<XT>::type X;
  typedef typename Elem<OT>::type O;
  constexpr int L = D / 4, RW = 32 / L, W = kAppendThreads / 32;
  constexpr int NU = TOK == 1 ? 2 : 1, NI = NU * TOK;  // turns (RW rows) taken together, rows in registers
  __shared__ int64_t s_blk[TOK];
  __shared__ int s_pos[TOK], s_start[kKvSeqs + 1];
  pdl_wait();
  pdl_launch_dependents();
  const int t0 = blockIdx.x * TOK;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (L - 1), sub = lane / L;
  const int KV = a.b.KV, i0 = 4 * l, half = a.rot_dim >> 1;
  const int n_tok = min(TOK, a.b.n_tokens - t0);
  // turns of RW rows: queries, keys, values
  const int uq = a.q ? (a.H + RW - 1) / RW : 0, uk = (KV + RW - 1) / RW, units = uq + 2 * uk;
  const bool rot = i0 < a.rot_dim;
  const int pair = lane + (rot ? (i0 < half ? half / 4 : -half / 4) : 0);  // the lane of the dims' pairs
  const float sign = i0 < half ? -1.0f : 1.0f;
  float x[NI][4];
  auto load = [&](int u0) {
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      const int u = u0 + k * W, kind = u < uq ? 0 : u < uq + uk ? 1 : 2;
      const int h = (kind == 0 ? u : kind == 1 ? u - uq : u - uq - uk) * RW + sub;
      const int64_t stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
      const X* src = reinterpret_cast<const X*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + t0 * stride + h * D + i0;
      const bool live = u < units && h < (kind == 0 ? a.H : KV);
#pragma unroll
      for (int j = 0; j < TOK; ++j) {
        if (live && j < n_tok) ld4(src, x[k * TOK + j]);
        else x[k * TOK + j][0] = x[k * TOK + j][1] = x[k * TOK + j][2] = x[k * TOK + j][3] = 0.0f;
        src += stride;
      }
    }
  };
  load(warp);
  kv_rows_of(a.b, t0, TOK, s_start, s_blk, s_pos);
  if (a.rot_dim && threadIdx.x < TOK && s_blk[threadIdx.x] >= 0 && s_pos[threadIdx.x] >= a.n_pos) {
    kv_batch_error();
    s_blk[threadIdx.x] = -1;
  }
  kv_check_offsets(a.b.q_start, a.b.n_seqs, s_start[kKvSeqs], s_start, a.b.n_seqs <= kKvSeqs);
  __syncthreads();
  const int bpp = a.b.page_tokens / kKvBlk;
  auto turn = [&](auto kind_c, int u, float (&v)[4], int j) {  // row `sub` of turn u of the kind, token j
    constexpr int kind = decltype(kind_c)::value;
    const int h = u * RW + sub;
    const int64_t blk0 = s_blk[j];
    const bool live = blk0 >= 0 && h < (kind == 0 ? a.H : KV);
    if (kind != 2 && a.rot_dim) {
      float c[4], s[4];
      const int64_t o = rot && blk0 >= 0 ? (int64_t)s_pos[j] * half + (i0 < half ? i0 : i0 - half) : 0;
      ld4(a.cos + o, c);
      ld4(a.sin + o, s);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // each product rounded, then their sum or difference
        const float p = __fmul_rn(__shfl_sync(B2Q_FULL, v[e], pair), s[e]), y = fmaf(sign, p, __fmul_rn(v[e], c[e]));
        v[e] = rot ? y : v[e];
      }
    }
    if (kind == 0) {
      if (live) st4(reinterpret_cast<O*>(a.q_out) + ((int64_t)(t0 + j) * a.H + h) * D + i0, v);
    } else {
      uint8_t* blk = a.pages + (live ? blk0 + (int64_t)h * bpp : 0) * kv_blk_bytes(D);
      kv_store_row<D, kind == 2>(blk, s_pos[j] & (kKvBlk - 1), v, l, live);
    }
  };
  for (int u0 = warp; u0 < units; u0 += NU * W) {
    if (u0 != warp) load(u0);
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      const int u = u0 + k * W;
      if (u < uq) {
#pragma unroll
        for (int j = 0; j < TOK; ++j) turn(std::integral_constant<int, 0>(), u, x[k * TOK + j], j);
      } else if (u < uq + uk) {
#pragma unroll
        for (int j = 0; j < TOK; ++j) turn(std::integral_constant<int, 1>(), u - uq, x[k * TOK + j], j);
      } else if (u < units) {
#pragma unroll
        for (int j = 0; j < TOK; ++j) turn(std::integral_constant<int, 2>(), u - uq - uk, x[k * TOK + j], j);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Read-back: the rows the append of the same batch would write.
// ---------------------------------------------------------------------------
struct GatherArgs {
  KvBatch b;
  const uint8_t* pages;
  void *k_out, *v_out;  // [n_tokens][KV * D], either may be null
  int heads;            // K/V heads of a CTA
};

// 8 values of codes in nibbles, times d, in the type O at p (16-byte aligned).
template <typename O>
__device__ __forceinline__ void kv_put8(O* p, const float (&c)[8], float d);
template <>
__device__ __forceinline__ void kv_put8<float>(float* p, const float (&c)[8], float d) {
  reinterpret_cast<float4*>(p)[0] = make_float4(c[0] * d, c[1] * d, c[2] * d, c[3] * d);
  reinterpret_cast<float4*>(p)[1] = make_float4(c[4] * d, c[5] * d, c[6] * d, c[7] * d);
}
template <typename O>
__device__ __forceinline__ void kv_put8(O* p, const float (&c)[8], float d) {
  *reinterpret_cast<uint4*>(p) = make_uint4(el_pack2<O>(c[0] * d, c[1] * d), el_pack2<O>(c[2] * d, c[3] * d),
                                            el_pack2<O>(c[4] * d, c[5] * d), el_pack2<O>(c[6] * d, c[7] * d));
}
// code - 8 of a nibble: 2^23 + code is an f32 number with the code in its low bits
__device__ __forceinline__ float kv_code(uint32_t nibble) {
  return __uint_as_float(0x4b000000u | (nibble & 15u)) - 8388616.0f;
}

// A CTA takes 32 packed rows and some of the K/V heads, a warp 8 rows of a head
// at a time: lane (g, t) row g; of the keys its own eight dims of each 32, of the
// values the groups of eight dims j = t, t + 4, ..., whose eight codes lie in the
// row's eight pieces, so that four lanes write 64 or 128 consecutive bytes.
constexpr int kGatherRows = 32;

template <int D, int OT>
__global__ void __launch_bounds__(256) kv_gather_kernel(const __grid_constant__ GatherArgs a) {
  typedef typename Elem<OT>::type O;
  constexpr int NB = D / 32;
  __shared__ int64_t s_blk[kGatherRows];  // block of head 0, -1: no row
  __shared__ int s_pos[kGatherRows], s_start[kKvSeqs + 1];
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = blockIdx.x * kGatherRows;
  kv_rows_of(a.b, row0, kGatherRows, s_start, s_blk, s_pos);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int bpp = a.b.page_tokens / kKvBlk, KV = a.b.KV;
  const int h0 = blockIdx.y * a.heads, heads = min(a.heads, KV - h0);
  for (int u = warp; u < kGatherRows / 8 * heads; u += 8) {
    const int h = h0 + (u >> 2), r = (u & 3) * 8 + g;
    const int64_t blk = s_blk[r];
    if (blk < 0) continue;
    const int tok = s_pos[r] & (kKvBlk - 1);
    const uint8_t* bp = a.pages + (blk + (int64_t)h * bpp) * kv_blk_bytes(D);
    const int64_t o = ((int64_t)(row0 + r) * KV + h) * D;
    uint32_t kw[NB], vw[8][NB / 2];
    uint32_t ks[NB / 2], vs[NB / 2];
    if (a.k_out) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(bp + tok * (D / 2) + t * (D / 8));
      const uint32_t* sp = reinterpret_cast<const uint32_t*>(bp + 8 * D + tok * NB * 2);
#pragma unroll
      for (int b = 0; b < NB; ++b) kw[b] = p[b];
#pragma unroll
      for (int b = 0; b < NB / 2; ++b) ks[b] = sp[b];
    }
    if (a.v_out) {
      const uint8_t* vp = bp + 9 * D + (tok >> 3) * (4 * D) + ((tok & 7) >> 1) * (D / 8) + (tok & 1) * (D / 16);
      const uint32_t* sp = reinterpret_cast<const uint32_t*>(bp + 17 * D + tok * NB * 2);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int w = 0; w < NB / 2; ++w) vw[e][w] = reinterpret_cast<const uint32_t*>(vp + e * (D / 2))[w];
#pragma unroll
      for (int b = 0; b < NB / 2; ++b) vs[b] = sp[b];
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float c[8];
      if (a.k_out) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = kv_code(kw[b] >> (4 * e));
        kv_put8<O>(reinterpret_cast<O*>(a.k_out) + o + 32 * b + 8 * t, c, f16_bits_fast((b & 1) ? ks[b >> 1] >> 16 : ks[b >> 1] & 0xffffu));
      }
      if (a.v_out) {  // j = 4 b + t
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = kv_code(vw[e][b >> 1] >> (4 * (4 * (b & 1) + t)));
        kv_put8<O>(reinterpret_cast<O*>(a.v_out) + o + 32 * b + 8 * t, c, f16_bits_fast((b & 1) ? vs[b >> 1] >> 16 : vs[b >> 1] & 0xffffu));
      }
    }
  }
  kv_check_offsets(a.b.q_start, a.b.n_seqs, s_start[kKvSeqs], s_start, a.b.n_seqs <= kKvSeqs);
}

}  // namespace b2q
