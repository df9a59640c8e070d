// quant_block.cu — quantisation to e4m3 with one fp32 scale per block of
// 1 x 128 or 128 x 128 elements, of a matrix or of its transpose.
//
//   a = max(largest finite |x| of the block, 2^-100)
//   scale = a / 448,  q = e4m3(x * (448 / a)),  each step rounded to fp32
//
// Memory-bound: 2 or 4 bytes read and 1 written per element. 8192 x 10240 bf16
// in rows 44-46 us = 0.84-0.88 of the copy bandwidth, in 128 x 128 blocks as they
// lie 48 us = 0.79, transposed 47 us with either block; f32 in rows 71 us, in
// 128 x 128 blocks 77 us, transposed 64 us (128 x 128) and 67 us (1 x 128) = 1.0
// and 0.96; 8191 x 4100 f32 in 128 x 128 blocks, transposed, 30.6 us = 0.84.
// Rows of X that are not 16-byte aligned are read element by element: 8192 x 10240
// bf16 160 us in 128 x 128 blocks and 205 in 1 x 128, 8191 x 4100 f32 71 and 90.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "sm100.cuh"
#include "tc_kernel.cuh"

namespace choreo_sm100 {

struct QuantParams {
  int64_t rows, cols;          // of op(X)
  int64_t row_tiles, col_tiles;
  const void* x;
  int64_t ldx;
  uint8_t* q;
  int64_t ldq;
  float* scale;
  int64_t scale_row, scale_blk;
  int32_t q_vec;               // bytes (16, 8) that a store to q's rows may have, 0: one
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | e4m3x2(c, d) << 16;
}

constexpr float kMaxFinite = 3.4028234663852886e38f;
constexpr float kTinyMax = 7.888609052210118e-31f;  // 2^-100: keeps 448 / a finite

// An infinite x becomes NaN (the conversion would store 448).
__device__ __forceinline__ float finite_or_nan(float x) { return fabsf(x) <= kMaxFinite ? x : __int_as_float(0x7fffffff); }
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= kMaxFinite ? a : 0.f;
}
__device__ __forceinline__ float factor_of(float amax) { return __fdiv_rn(448.f, fmaxf(amax, kTinyMax)); }
__device__ __forceinline__ float scale_of(float amax) { return __fdiv_rn(fmaxf(amax, kTinyMax), 448.f); }

// One 16-byte piece of a row of X: 8 elements (4 of f32).
template <typename T>
struct Piece {
  static constexpr int kElems = 16 / static_cast<int>(sizeof(T));
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      float lo, hi;
      unpack2(w[i / 2], lo, hi, static_cast<T*>(nullptr));
      return (i & 1) ? hi : lo;
    }
  }
  // Elements past `left` read as zero.
  __device__ __forceinline__ void load(const T* p, int64_t left) {
    if (left >= kElems) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      return;
    }
    w[0] = w[1] = w[2] = w[3] = 0;
#pragma unroll
    for (int i = 0; i < kElems; ++i)
      if (i < left) {
        if constexpr (sizeof(T) == 4)
          w[i] = __float_as_uint(p[i]);
        else
          w[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + i)) << (16 * (i & 1));
      }
  }
  // Magnitude bits of word j: of two 16-bit elements or of one of 32 bits.
  __device__ __forceinline__ uint32_t top_of(int j) const { return w[j] & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu); }
  // Largest magnitude, as ordered bits: two 16-bit halves or one 32-bit value.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      return max(max(w[0] & 0x7fffffffu, w[1] & 0x7fffffffu), max(w[2] & 0x7fffffffu, w[3] & 0x7fffffffu));
    } else {
      return __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    }
  }
  __device__ __forceinline__ float finite_top() const {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kElems; ++i) m = fmaxf(m, finite_abs(get(i)));
    return m;
  }
};
template <typename T>
__device__ __forceinline__ uint32_t top_max(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4)
    return max(a, b);
  else
    return __vmaxu2(a, b);
}
// The magnitude that `top` bits stand for; *all_finite: no NaN or infinity among them.
template <typename T>
__device__ __forceinline__ float top_value(uint32_t top, bool* all_finite) {
  if constexpr (sizeof(T) == 4) {
    *all_finite = top < 0x7f800000u;
    return __uint_as_float(top);
  } else {
    const uint32_t m = max(top & 0xffffu, top >> 16);
    *all_finite = m < (std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u);
    float lo, hi;
    unpack2(m, lo, hi, static_cast<T*>(nullptr));
    return lo;
  }
}
// kElems quantised values of a piece; `clean`: no NaN or infinity in it.
template <typename T>
__device__ __forceinline__ void quantize_piece(const Piece<T>& v, float inv, bool clean, uint32_t (&q)[2]) {
  float f[Piece<T>::kElems];
#pragma unroll
  for (int i = 0; i < Piece<T>::kElems; ++i) f[i] = v.get(i) * inv;
  if (!clean) {
#pragma unroll
    for (int i = 0; i < Piece<T>::kElems; ++i) f[i] = finite_or_nan(v.get(i)) * inv;
  }
  q[0] = e4m3x4(f[0], f[1], f[2], f[3]);
  if constexpr (sizeof(T) == 2) q[1] = e4m3x4(f[4], f[5], f[6], f[7]);
}
// The same with a factor of its own for each element.
template <typename T>
__device__ __forceinline__ void quantize_piece(const Piece<T>& v, const float (&inv)[Piece<T>::kElems], bool clean,
                                               uint32_t (&q)[2]) {
  float f[Piece<T>::kElems];
#pragma unroll
  for (int i = 0; i < Piece<T>::kElems; ++i) f[i] = v.get(i) * inv[i];
  if (!clean) {
#pragma unroll
    for (int i = 0; i < Piece<T>::kElems; ++i) f[i] = finite_or_nan(v.get(i)) * inv[i];
  }
  q[0] = e4m3x4(f[0], f[1], f[2], f[3]);
  if constexpr (sizeof(T) == 2) q[1] = e4m3x4(f[4], f[5], f[6], f[7]);
}
// Stores kElems bytes of a row of q, those before column `cols`.
template <int kElems>
__device__ __forceinline__ void store_q(uint8_t* q, const uint32_t (&v)[2], int64_t left, bool vec) {
  if (vec && left >= kElems) {
    if constexpr (kElems == 8)
      *reinterpret_cast<uint2*>(q) = make_uint2(v[0], v[1]);
    else
      *reinterpret_cast<uint32_t*>(q) = v[0];
    return;
  }
#pragma unroll
  for (int i = 0; i < kElems; ++i)
    if (i < left) q[i] = static_cast<uint8_t>(v[i / 4] >> (8 * (i & 3)));
}

// inv and scale of UNROLL blocks per lane group, from their amax: lane l of a
// group divides for block l % UNROLL only and the group shares the factors (a
// correctly rounded division is some 15 instructions, and as many as the rest
// of a block's work if every lane did both for every block).
template <int UNROLL>
__device__ __forceinline__ float pick(const float (&v)[UNROLL], int i) {
  float r = v[0];
#pragma unroll
  for (int u = 1; u < UNROLL; ++u) r = i == u ? v[u] : r;
  return r;
}

// Largest finite magnitude of the kLanes lanes' pieces, in every lane of the
// group; *clean: no NaN or infinity in the warp's pieces.
template <typename T, int kLanes>
__device__ __forceinline__ float group_amax(const Piece<T>& v, bool* clean) {
  uint32_t top = v.top();
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) top = top_max<T>(top, __shfl_xor_sync(0xffffffffu, top, o));
  float amax = top_value<T>(top, clean);
  *clean = __all_sync(0xffffffffu, *clean);
  if (!*clean) {
    amax = v.finite_top();
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  return amax;
}

// 1 x 128 blocks along X's rows. A block is 16 lanes' 16-byte loads (32 lanes'
// for f32); a warp takes UNROLL consecutive 512-byte runs of one row, all loads
// in flight at once, and 8 neighbouring rows share a CTA so that their scales
// fall into one 32-byte sector. Bound by memory: 3 (5) bytes per element.
template <typename T, int UNROLL>
__global__ void __launch_bounds__(256, 5) quant_rows_kernel(const QuantParams p, int64_t runs) {
  constexpr int E = Piece<T>::kElems;
  constexpr int kLanes = 128 / E;  // lanes of one block
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = blockIdx.x / runs;
  const int64_t r = group * 8 + warp;
  if (r >= p.rows) return;
  const int64_t run0 = (blockIdx.x - group * runs) * (UNROLL * 32 * E);
  const int64_t c0 = run0 + lane * E;
  const T* x = static_cast<const T*>(p.x) + r * p.ldx + c0;
  Piece<T> v[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) v[u].load(x + u * 32 * E, p.cols - c0 - u * 32 * E);
  float amax[UNROLL];
  bool clean[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) amax[u] = group_amax<T, kLanes>(v[u], &clean[u]);
  const int mine = lane % kLanes;
  const float own = pick<UNROLL>(amax, mine % UNROLL);
  const float inv = factor_of(own);
  const int64_t own_col = run0 + mine * 32 * E + lane / kLanes * 128;
  if (mine < UNROLL && own_col < p.cols) p.scale[r * p.scale_row + own_col / 128 * p.scale_blk] = scale_of(own);
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t c = c0 + u * 32 * E;
    uint32_t q[2];
    quantize_piece<T>(v[u], __shfl_sync(0xffffffffu, inv, (lane & ~(kLanes - 1)) | u), clean[u], q);
    store_q<E>(p.q + r * p.ldq + c, q, p.cols - c, p.q_vec != 0);
  }
}

// Largest finite magnitude over the CTA's threads.
template <typename T, int kWarps>
__device__ __forceinline__ float cta_amax(uint32_t top, float finite_top, uint32_t* warp_top, float* warp_finite,
                                          bool* all_clean) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = top_max<T>(top, __shfl_xor_sync(0xffffffffu, top, o));
    finite_top = fmaxf(finite_top, __shfl_xor_sync(0xffffffffu, finite_top, o));
  }
  if (lane == 0) {
    warp_top[warp] = top;
    warp_finite[warp] = finite_top;
  }
  __syncthreads();
  float m = 0.f;
  bool all = true;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    bool clean;
    top_value<T>(warp_top[w], &clean);
    all = all && clean;
    m = fmaxf(m, warp_finite[w]);
  }
  *all_clean = all;
  return m;
}

// Largest finite magnitude of the CTA's pieces; *clean: no NaN or infinity.
template <typename T, int kPieces, int kWarps>
__device__ __forceinline__ float tile_amax(const Piece<T> (&v)[kPieces], uint32_t* warp_top, float* warp_finite,
                                           bool* clean) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) top = top_max<T>(top, v[i].top());
  bool own_clean;
  float m = top_value<T>(top, &own_clean);
  if (!own_clean) {
    m = 0.f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) m = fmaxf(m, v[i].finite_top());
  }
  return cta_amax<T, kWarps>(top, m, warp_top, warp_finite, clean);
}

// One 128 x 128 tile of X per CTA with one scale, stored as it lies. Thread:
// kPieces pieces of 16 bytes; a warp load takes 32 / kLanes whole tile rows.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) quant_tile_kernel(const QuantParams p) {
  constexpr int kWarps = kThreads / 32;
  constexpr int E = Piece<T>::kElems;
  constexpr int kPieces = 128 * 128 / E / kThreads;
  constexpr int kLanes = 128 / E;
  constexpr int kRows = 32 / kLanes;  // rows of one warp load
  __shared__ uint32_t warp_top[kWarps];
  __shared__ float warp_finite[kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rt = blockIdx.x / p.col_tiles, ct = blockIdx.x - rt * p.col_tiles;
  const int64_t r0 = rt * 128, c = ct * 128 + lane % kLanes * E;
  const T* x = static_cast<const T*>(p.x);
  Piece<T> v[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int64_t r = r0 + (i * kWarps + warp) * kRows + lane / kLanes;
    v[i].load(x + (r < p.rows ? r : p.rows - 1) * p.ldx + c, r < p.rows ? p.cols - c : 0);
  }
  bool clean;
  const float amax = tile_amax<T, kPieces, kWarps>(v, warp_top, warp_finite, &clean);
  const float inv = factor_of(amax);
  if (threadIdx.x == 0) p.scale[rt * p.scale_row + ct * p.scale_blk] = scale_of(amax);
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int64_t r = r0 + (i * kWarps + warp) * kRows + lane / kLanes;
    if (r >= p.rows) continue;
    uint32_t q[2];
    quantize_piece<T>(v[i], inv, clean, q);
    store_q<E>(p.q + r * p.ldq + c, q, p.cols - c, p.q_vec != 0);
  }
}

// One 128 x 128 tile of X per CTA, turned: rows of X are columns of op(X).
// SQUARE: one scale for the tile, else one per column of X.
//
// A thread loads the same columns of X (16 bytes) in groups of four rows, so a
// warp load covers whole tile rows, the largest value of a column is a maximum
// over registers and then over the warps, and four rows' codes of a column are
// one word after a 4 x 4 byte transpose. Only codes go through shared memory (16
// KB, not the tile's 32 or 64). There word g (rows 4 g .. of X) of column c
// stands at g ^ (c / E * E / 4): the lanes of a store, at neighbouring c / E,
// meet 32 banks, and a 16-byte load still finds its four words in one chunk, in
// an order that depends on the column only. 8 lanes write one 128-byte row.
//
// Turning the elements and quantising afterwards, as this kernel did first, took
// 76 and 96 us for f32 and 50 and 56 us for bf16 at 8192 x 10240: its tile filled
// 64 KB, and a 1 x 128 block cost shuffles over 16 or 32 lanes. Three CTAs an SM
// for f32 (2: 76 us, 4 spills: 85), four for 16 bits (5: 46 us here but 8.5
// against 7.9 at 4096 x 2048, 3: 53, 6 spills).
template <typename T, bool SQUARE, int kMinCtas>
__global__ void __launch_bounds__(256, kMinCtas) quant_turn_kernel(const QuantParams p) {
  constexpr int kWarps = 8;
  constexpr int E = Piece<T>::kElems;
  constexpr int kLanes = 128 / E;
  constexpr int kSteps = kLanes / kWarps;  // groups of four rows a thread takes
  __shared__ uint4 turned_raw[128 * 8];
  __shared__ uint4 warp_cols[kWarps][SQUARE ? 1 : kLanes];  // each warp's column maxima, as top bits
  __shared__ float col_inv[SQUARE ? 1 : 128];
  __shared__ uint32_t warp_top[kWarps];
  __shared__ float warp_finite[kWarps];
  uint32_t* turned = reinterpret_cast<uint32_t*>(turned_raw);
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane % kLanes;
  // Neighbouring CTAs read neighbouring columns of X (2 to 4 % over the other order).
  const int64_t ct = blockIdx.x / p.row_tiles, rt = blockIdx.x - ct * p.row_tiles;
  const int64_t r0 = rt * 128, c0 = ct * 128;  // row and column of op(X): column and row of X
  const T* x = static_cast<const T*>(p.x);
  auto group_of = [&](int s) { return (s * kWarps + warp) * (32 / kLanes) + lane / kLanes; };
  Piece<T> v[kSteps * 4];
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int64_t k = c0 + group_of(s) * 4 + h;
      const int64_t r = r0 + piece * E;
      v[s * 4 + h].load(x + (k < p.cols ? k : p.cols - 1) * p.ldx + r, k < p.cols ? p.rows - r : 0);
    }
  bool clean = true;
  float inv[SQUARE ? 1 : E];
  if constexpr (SQUARE) {
    const float amax = tile_amax<T, kSteps * 4, kWarps>(v, warp_top, warp_finite, &clean);
    inv[0] = factor_of(amax);
    if (threadIdx.x == 0) p.scale[rt * p.scale_row + ct * p.scale_blk] = scale_of(amax);
  } else {
    uint32_t top[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      top[j] = v[0].top_of(j);
#pragma unroll
      for (int i = 1; i < kSteps * 4; ++i) top[j] = top_max<T>(top[j], v[i].top_of(j));
      if (kLanes == 16) top[j] = top_max<T>(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
    }
    if (lane < kLanes) warp_cols[warp][lane] = make_uint4(top[0], top[1], top[2], top[3]);
    __syncthreads();
    // Thread c finishes column c.
    const int c = threadIdx.x;
    float amax = 0.f;
    bool finite = true;
    if (c < 128) {
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t word = reinterpret_cast<const uint32_t*>(warp_cols[w])[sizeof(T) == 4 ? c : c / 2];
        m = max(m, sizeof(T) == 4 ? word : ((c & 1) ? word >> 16 : word & 0xffffu));
      }
      amax = top_value<T>(m, &finite);
    }
    clean = __syncthreads_or(finite ? 0 : 1) == 0;
    if (!clean) {  // NaN or an infinity in the tile: the columns' largest finite values
      float* fin = reinterpret_cast<float*>(turned);  // [warp][column]
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < kSteps * 4; ++i) m = fmaxf(m, finite_abs(v[i].get(e)));
        if (kLanes == 16) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (lane < kLanes) fin[warp * 128 + piece * E + e] = m;
      }
      __syncthreads();
      if (c < 128) {
        amax = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) amax = fmaxf(amax, fin[w * 128 + c]);
      }
      // (the barrier below also separates these reads from the codes' stores)
    }
    if (c < 128) {
      col_inv[c] = factor_of(amax);
      if (r0 + c < p.rows) p.scale[(r0 + c) * p.scale_row + ct * p.scale_blk] = scale_of(amax);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) inv[e] = col_inv[piece * E + e];
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    uint32_t q[4][2];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      if constexpr (SQUARE)
        quantize_piece<T>(v[s * 4 + h], inv[0], clean, q[h]);
      else
        quantize_piece<T>(v[s * 4 + h], inv, clean, q[h]);
    }
    uint32_t* dst = turned + piece * E * 32 + (group_of(s) ^ (piece * (E / 4)));
#pragma unroll
    for (int b = 0; b < E / 4; ++b) {  // columns 4 b .. 4 b + 3 of the piece
      const uint32_t lo01 = __byte_perm(q[0][b], q[1][b], 0x5140), lo23 = __byte_perm(q[2][b], q[3][b], 0x5140);
      const uint32_t hi01 = __byte_perm(q[0][b], q[1][b], 0x7362), hi23 = __byte_perm(q[2][b], q[3][b], 0x7362);
      dst[(4 * b + 0) * 32] = __byte_perm(lo01, lo23, 0x5410);
      dst[(4 * b + 1) * 32] = __byte_perm(lo01, lo23, 0x7632);
      dst[(4 * b + 2) * 32] = __byte_perm(hi01, hi23, 0x5410);
      dst[(4 * b + 3) * 32] = __byte_perm(hi01, hi23, 0x7632);
    }
  }
  __syncthreads();
  const int part = lane & 7;  // 16 columns of op(X)
  const int64_t left = p.cols - c0 - part * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (i * kWarps + warp) * 4 + (lane >> 3);
    const int turn = row / E * (E / 4);
    const uint4 w = turned_raw[row * 8 + (part ^ (turn >> 2))];
    uint32_t a = w.x, b = w.y, c = w.z, d = w.w;
    if (turn & 1) {
      const uint32_t a0 = a, c0s = c;
      a = b, b = a0, c = d, d = c0s;
    }
    if (turn & 2) {
      const uint32_t a0 = a, b0 = b;
      a = c, c = a0, b = d, d = b0;
    }
    if (r0 + row >= p.rows || left <= 0) continue;
    uint8_t* q = p.q + (r0 + row) * p.ldq + c0 + part * 16;
    if (left >= 16 && p.q_vec == 16) {
      *reinterpret_cast<uint4*>(q) = make_uint4(a, b, c, d);
    } else {
      const uint32_t first[2] = {a, b}, second[2] = {c, d};
      store_q<8>(q, first, left, p.q_vec != 0);
      store_q<8>(q + 8, second, left - 8, p.q_vec != 0);
    }
  }
}

// Any alignment of X: the same tile through shared memory as f32, element by
// element.
template <typename T, bool SQUARE, bool TRANS>
__global__ void __launch_bounds__(256) quant_unaligned_kernel(const QuantParams p) {
  extern __shared__ uint4 turned_raw[];
  float* tile = reinterpret_cast<float*>(turned_raw);  // 128 rows of op(X), pitch 129
  __shared__ uint32_t warp_top[8];
  __shared__ float warp_finite[8];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rt = blockIdx.x / p.col_tiles, ct = blockIdx.x - rt * p.col_tiles;
  const int64_t r0 = rt * 128, c0 = ct * 128;
  const T* x = static_cast<const T*>(p.x);
  for (int i = warp; i < 128; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = lane + 32 * j;
      if constexpr (!TRANS) {
        const bool in = r0 + i < p.rows && c0 + c < p.cols;
        tile[i * 129 + c] = in ? to_f32<T>(x[(r0 + i) * p.ldx + c0 + c]) : 0.f;
      } else {
        const bool in = c0 + i < p.cols && r0 + c < p.rows;
        tile[c * 129 + i] = in ? to_f32<T>(x[(c0 + i) * p.ldx + r0 + c]) : 0.f;
      }
    }
  }
  __syncthreads();
  float inv = 0.f;
  if constexpr (SQUARE) {
    float m = 0.f;
    for (int i = warp; i < 128; i += 8)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = fmaxf(m, finite_abs(tile[i * 129 + lane + 32 * j]));
    bool clean;
    const float amax = cta_amax<float, 8>(0, m, warp_top, warp_finite, &clean);
    inv = factor_of(amax);
    if (threadIdx.x == 0) p.scale[rt * p.scale_row + ct * p.scale_blk] = scale_of(amax);
  }
  for (int i = warp; i < 128; i += 8) {
    const int64_t r = r0 + i;
    if (r >= p.rows) break;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = tile[i * 129 + 4 * lane + j];
    if constexpr (!SQUARE) {
      float m = fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3])));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      inv = factor_of(m);
      if (lane == 0) p.scale[r * p.scale_row + ct * p.scale_blk] = scale_of(m);
    }
    const uint32_t w[2] = {e4m3x4(finite_or_nan(v[0]) * inv, finite_or_nan(v[1]) * inv, finite_or_nan(v[2]) * inv,
                                  finite_or_nan(v[3]) * inv), 0};
    const int64_t c = c0 + 4 * lane;
    store_q<4>(p.q + r * p.ldq + c, w, p.cols - c, p.q_vec != 0);
  }
}

}  // namespace choreo_sm100

namespace choreo_impl {
using namespace choreo_sm100;

namespace {

template <typename Kern, typename... Args>
int launch_quant(Kern kern, int64_t grid, int threads, int smem, std::atomic<uint64_t>& done, cudaStream_t s,
                 Args... args) {
  if (grid > INT32_MAX) return fail(CHOREO_ERR_UNSUPPORTED, "quantize: more than 2^31-1 tiles");
  if (smem > 0)
    if (int rc = set_smem_limit_once(kern, smem, done, "cudaFuncSetAttribute(quantize)")) return rc;
  const cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(threads), smem, s, args...);
  return e == cudaSuccess ? CHOREO_OK : cuda_fail(e, "quantize launch");
}

template <typename T, int UNROLL>
int launch_rows(const QuantParams& p, cudaStream_t s) {
  constexpr int64_t span = UNROLL * 32 * Piece<T>::kElems;
  const int64_t runs = (p.cols + span - 1) / span;
  std::atomic<uint64_t> none{0};
  return launch_quant(quant_rows_kernel<T, UNROLL>, (p.rows + 7) / 8 * runs, 256, 0, none, s, p, runs);
}

template <typename T, bool SQUARE, bool TRANS>
int launch_tile(const QuantParams& p, bool x_vec, cudaStream_t s) {
  const int64_t grid = p.row_tiles * p.col_tiles;
  if (!x_vec) {
    static std::atomic<uint64_t> done{0};
    return launch_quant(quant_unaligned_kernel<T, SQUARE, TRANS>, grid, 256, 128 * 129 * 4, done, s, p);
  }
  if constexpr (SQUARE || TRANS) {
    static std::atomic<uint64_t> done{0};
    constexpr int kThreads = 256;
    if constexpr (TRANS)
      return launch_quant(quant_turn_kernel<T, SQUARE, sizeof(T) == 4 ? 3 : 4>, grid, 256, 0, done, s, p);
    else
      return launch_quant(quant_tile_kernel<T, kThreads>, grid, kThreads, 0, done, s, p);
  } else {
    // Four loads in flight a thread where that still leaves every SM two CTAs;
    // a few rows are spread over as many SMs as one load each can reach.
    const int64_t wide = (p.rows + 7) / 8 * ((p.cols + 128 * Piece<T>::kElems - 1) / (128 * Piece<T>::kElems));
    return wide >= 2 * current_sm_count() ? launch_rows<T, 4>(p, s) : launch_rows<T, 1>(p, s);
  }
}

template <typename T>
int dispatch_quant(const QuantParams& p, bool rows, bool trans, bool x_vec, cudaStream_t s) {
  if (rows) return trans ? launch_tile<T, false, true>(p, x_vec, s) : launch_tile<T, false, false>(p, x_vec, s);
  return trans ? launch_tile<T, true, true>(p, x_vec, s) : launch_tile<T, true, false>(p, x_vec, s);
}

}  // namespace
}  // namespace choreo_impl

using namespace choreo_impl;

extern "C" int choreo_quantize_block(const choreo_quant_desc* d, void* stream) {
  if (d == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "quantize: null descriptor");
  if (d->rows < 0 || d->cols < 0)
    return fail(CHOREO_ERR_INVALID_ARG, "quantize: negative size (%lld x %lld)", (long long)d->rows, (long long)d->cols);
  if (!is_float_type(d->dtype)) return fail(CHOREO_ERR_UNSUPPORTED, "quantize: unsupported dtype %d", d->dtype);
  if (d->block_rows != 1 && d->block_rows != 128)
    return fail(CHOREO_ERR_UNSUPPORTED, "quantize: block_rows %d is neither 1 nor 128", d->block_rows);
  if (d->rows == 0 || d->cols == 0) return ok();
  if (d->rows > INT32_MAX || d->cols > INT32_MAX)
    return fail(CHOREO_ERR_UNSUPPORTED, "quantize: dimensions above 2^31-1 are not supported");
  if (d->x == nullptr || d->q == nullptr || d->scale == nullptr)
    return fail(CHOREO_ERR_INVALID_ARG, "quantize: Tensor has null data pointer");
  QuantParams p{};
  p.rows = d->transpose ? d->cols : d->rows;
  p.cols = d->transpose ? d->rows : d->cols;
  if (d->ldx < d->cols)
    return fail(CHOREO_ERR_INVALID_ARG, "quantize: ldx=%lld smaller than %lld", (long long)d->ldx, (long long)d->cols);
  if (d->ldq < p.cols)
    return fail(CHOREO_ERR_INVALID_ARG, "quantize: ldq=%lld smaller than %lld", (long long)d->ldq, (long long)p.cols);
  const int64_t row_blocks = (p.rows + d->block_rows - 1) / d->block_rows;
  const int64_t col_blocks = (p.cols + 127) / 128;
  if ((row_blocks > 1 && d->scale_row <= 0) || (col_blocks > 1 && d->scale_blk <= 0))
    return fail(CHOREO_ERR_INVALID_ARG, "quantize: scale strides must be positive");
  int rc;
  if ((rc = check_device_ptr(d->x, "quantize X"))) return rc;
  if ((rc = check_device_ptr(d->q, "quantize q"))) return rc;
  if ((rc = check_device_ptr(d->scale, "quantize scale"))) return rc;
  p.x = d->x;
  p.ldx = d->ldx;
  p.q = static_cast<uint8_t*>(d->q);
  p.ldq = d->ldq;
  p.scale = d->scale;
  p.scale_row = d->scale_row;
  p.scale_blk = d->scale_blk;
  p.row_tiles = (p.rows + 127) / 128;
  p.col_tiles = col_blocks;
  const bool x_vec =
      ((reinterpret_cast<uintptr_t>(d->x) | static_cast<uintptr_t>(d->ldx * dtype_bytes(d->dtype))) & 15u) == 0;
  const uintptr_t q_bits = reinterpret_cast<uintptr_t>(d->q) | static_cast<uintptr_t>(d->ldq);
  p.q_vec = (q_bits & 15u) == 0 ? 16 : ((q_bits & 7u) == 0 ? 8 : 0);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool rows = d->block_rows == 1, trans = d->transpose != 0;
  switch (d->dtype) {
    case CHOREO_DTYPE_F16: rc = dispatch_quant<__half>(p, rows, trans, x_vec, s); break;
    case CHOREO_DTYPE_BF16: rc = dispatch_quant<__nv_bfloat16>(p, rows, trans, x_vec, s); break;
    default: rc = dispatch_quant<float>(p, rows, trans, x_vec, s); break;
  }
  return rc ? rc : ok();
}
