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

// Sequence and position of packed row t (one thread).  False for rows behind
// the last sequence, and (with the error word) for offsets that make no sense.
__device__ __forceinline__ bool kv_row_of(const KvBatch& b, int t, int& seq, int& pos) {
  int lo = 0, hi = b.n_seqs;  // the number of q_start[1..n_seqs] <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (b.q_start[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= b.n_seqs) return false;
  seq = lo;
  const int a = b.q_start[lo], e = b.q_start[lo + 1];
  if (a < 0 || t < a || t >= e) {
    kv_batch_error();
    return false;
  }
  pos = kv_pos_of(b.kv_len[lo], e - t);
  return true;
}

// ---------------------------------------------------------------------------
// Append.  One warp per row (a head of a token) of D = 128, two rows of
// D = 64; a lane holds four consecutive dims.
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

template <int D>
__device__ __forceinline__ void kv_store_row(uint8_t* blk, int tok, bool is_v, const float (&x)[4], int l, bool live) {
  // l: lane of the row (dims 4l..4l+3); all lanes of the warp take part, the live rows' store
  float m = x[0], a = fabsf(x[0]);
  bool fin = a <= 3.402823466e38f;
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const float ai = fabsf(x[i]);
    fin = fin && ai <= 3.402823466e38f;
    if (ai > a) { a = ai; m = x[i]; }
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const float a2 = __shfl_xor_sync(B2Q_FULL, a, o), m2 = __shfl_xor_sync(B2Q_FULL, m, o);
    // the first of equals: the other lane's only if it lies before this one
    if (a2 > a || (a2 == a && (l & o))) { a = a2; m = m2; }
    fin = __shfl_xor_sync(B2Q_FULL, (int)fin, o) && fin;
  }
  // m / -8 beyond f16 keeps the largest finite scale
  const float ds = fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f);
  const __half dh = __float2half_rn(ds);
  const float d = __half2float(dh);
  uint32_t pk = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float r = d == 0.0f ? 0.0f : rintf(__fdiv_rn(x[i], d));
    const int c = fin ? (int)fminf(fmaxf(r + 8.0f, 0.0f), 15.0f) : 8;
    pk |= (uint32_t)c << (4 * i);
  }
  const unsigned short sc = fin ? __half_as_ushort(dh) : (unsigned short)0x7fff;
  constexpr int NB = D / 32;  // blocks of 32 dims
  uint8_t* base = blk + (is_v ? 9 * D : 0);
  if (live && (l & 7) == 0) *reinterpret_cast<unsigned short*>(base + 8 * D + (tok * NB + (l >> 3)) * 2) = sc;
  const uint32_t nb = __shfl_xor_sync(B2Q_FULL, pk, 1);
  // value pieces: nibble j of piece g is dim 8j + g, held by lane 2j + (g >> 2)
  uint32_t w = 0;
  const int g = (l >> (D == 128 ? 1 : 0)) & 7, half = D == 128 ? l & 1 : 0;
  const int row0 = (threadIdx.x & 31) & ~(D / 4 - 1);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t o = __shfl_sync(B2Q_FULL, pk, row0 + 2 * (half * 8 + j) + (g >> 2));
    w |= ((o >> (4 * (g & 3))) & 15u) << (4 * j);
  }
  if (!live) return;
  if (!is_v) {
    if ((l & 1) == 0) {
      const int u = l >> 1;  // dims 8u..8u+7
      *reinterpret_cast<uint32_t*>(base + tok * (D / 2) + (u & 3) * (D / 8) + (u >> 2) * 4) = pk | (nb << 16);
    }
  } else if (l < D / 8) {
    *reinterpret_cast<uint32_t*>(base + (tok >> 3) * (4 * D) + g * (D / 2) + ((tok & 7) >> 1) * (D / 8) +
                                 (tok & 1) * (D / 16) + half * 4) = w;
  }
}

constexpr int kAppendThreads = 256;

template <int D, int XT, int OT>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ AppendArgs a) {
  typedef typename Elem<XT>::type X;
  typedef typename Elem<OT>::type O;
  constexpr int L = D / 4, RW = 32 / L;
  const int t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (L - 1), sub = lane / L;
  int seq, pos;
  if (!kv_row_of(a.b, t, seq, pos)) return;
  const int64_t blk0 = kv_block_of(a.b, seq, pos);
  if (blk0 < 0) return;
  if (a.rot_dim && pos >= a.n_pos) {
    kv_batch_error();
    return;
  }
  const int KV = a.b.KV, bpp = a.b.page_tokens / kKvBlk, tok = pos & (kKvBlk - 1);
  const int half = a.rot_dim >> 1, i0 = 4 * l;
  const bool rot = i0 < a.rot_dim;
  float c[4] = {1, 1, 1, 1}, s[4] = {0, 0, 0, 0};
  if (rot) {
    const int64_t o = (int64_t)pos * half + (i0 < half ? i0 : i0 - half);
    ld4(a.cos + o, c);
    ld4(a.sin + o, s);
  }
  const int src = (lane & ~(L - 1)) + (rot ? (i0 < half ? l + half / 4 : l - half / 4) : l);
  const int rows0 = a.q ? 0 : a.H, rows = a.H + 2 * KV;
  for (int r0 = rows0 + warp * RW; r0 < rows; r0 += (kAppendThreads / 32) * RW) {
    const int r = r0 + sub;
    const bool live = r < rows;
    const bool is_q = r < a.H, is_v = r >= a.H + KV;
    const int h = is_q ? r : is_v ? r - a.H - KV : r - a.H;
    float x[4] = {0, 0, 0, 0};
    if (live)
      ld4(reinterpret_cast<const X*>(is_q ? a.q : is_v ? a.v : a.k) +
              (int64_t)t * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + h * D + i0,
          x);
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = __shfl_sync(B2Q_FULL, x[i], src);
      y[i] = !rot || is_v ? x[i]
             : i0 < half  ? __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(p, s[i]))
                          : __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(p, s[i]));
    }
    if (is_q && live) st4(reinterpret_cast<O*>(a.q_out) + ((int64_t)t * a.H + h) * D + i0, y);
    // rows of a warp pair may be a query and a key: all lanes go through the
    // shuffles, the stores are the live key and value rows'
    if (__any_sync(B2Q_FULL, live && !is_q)) {
      uint8_t* blk = a.pages + (blk0 + (int64_t)(is_q || !live ? 0 : h) * bpp) * kv_blk_bytes(D);
      kv_store_row<D>(blk, tok, is_v, y, l, live && !is_q);
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
};

__device__ __forceinline__ float kv_key_at(const uint8_t* blk, int D, int tok, int dim) {
  const int byte = tok * (D / 2) + ((dim >> 3) & 3) * (D / 8) + (dim >> 5) * 4 + ((dim & 7) >> 1);
  const float d = f16_bits_fast(*reinterpret_cast<const unsigned short*>(blk + 8 * D + (tok * (D / 32) + (dim >> 5)) * 2));
  return (float)((int)((blk[byte] >> (4 * (dim & 1))) & 15) - 8) * d;
}
__device__ __forceinline__ float kv_value_at(const uint8_t* blk, int D, int tok, int dim) {
  const uint8_t* v = blk + 9 * D;
  const int g = dim & 7, j = dim >> 3;
  const int byte = (tok >> 3) * (4 * D) + g * (D / 2) + ((tok & 7) >> 1) * (D / 8) + (tok & 1) * (D / 16) + (j >> 1);
  const float d = f16_bits_fast(*reinterpret_cast<const unsigned short*>(v + 8 * D + (tok * (D / 32) + (dim >> 5)) * 2));
  return (float)((int)((v[byte] >> (4 * (j & 1))) & 15) - 8) * d;
}

template <int D, int OT>
__global__ void __launch_bounds__(256) kv_gather_kernel(const __grid_constant__ GatherArgs a) {
  typedef typename Elem<OT>::type O;
  const int t = blockIdx.x;
  int seq, pos;
  if (!kv_row_of(a.b, t, seq, pos)) return;
  const int64_t blk0 = kv_block_of(a.b, seq, pos);
  if (blk0 < 0) return;
  const int bpp = a.b.page_tokens / kKvBlk, tok = pos & (kKvBlk - 1);
  for (int i = threadIdx.x; i < a.b.KV * D; i += blockDim.x) {
    const uint8_t* blk = a.pages + (blk0 + (int64_t)(i / D) * bpp) * kv_blk_bytes(D);
    const int64_t o = (int64_t)t * a.b.KV * D + i;
    if (a.k_out) reinterpret_cast<O*>(a.k_out)[o] = el_from<O>(kv_key_at(blk, D, tok, i % D));
    if (a.v_out) reinterpret_cast<O*>(a.v_out)[o] = el_from<O>(kv_value_at(blk, D, tok, i % D));
  }
}

}  // namespace b2q
