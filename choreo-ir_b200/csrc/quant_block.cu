// quant_block.cu — quantisation to e4m3 with one fp32 scale per block of
// 1 x 128 or 128 x 128 elements, of a matrix or of its transpose.
//
//   a = max(largest finite |x| of the block, 2^-100)
//   scale = a / 448,  q = e4m3(x * (448 / a)),  each step rounded to fp32
//
// Memory-bound: 2 or 4 bytes read and 1 written per element.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "internal.h"
#include "sm100.cuh"
#include "tc_kernel.cuh"

namespace choreo_sm100 {

struct QuantParams {
  int64_t rows, cols;          // of op(X)
  const void* x;
  int64_t ldx;
  uint8_t* q;
  int64_t ldq;
  float* scale;
  int64_t scale_row, scale_blk;
  int32_t x_vec, q_vec;        // 16-byte loads of X's rows / 4-byte stores of q's rows are legal
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// x * inv, with an infinite x made NaN (the conversion would store 448).
__device__ __forceinline__ float scaled(float x, float inv) {
  return fabsf(x) <= 3.4028234663852886e38f ? x * inv : __int_as_float(0x7fffffff);
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.4028234663852886e38f ? a : 0.f;
}
constexpr float kTinyMax = 7.888609052210118e-31f;  // 2^-100: keeps 448 / a finite

__device__ __forceinline__ void factors(float amax, float& inv, float& scale) {
  const float a = fmaxf(amax, kTinyMax);
  inv = __fdiv_rn(448.f, a);
  scale = __fdiv_rn(a, 448.f);
}

template <typename T>
__device__ __forceinline__ float load_elem(const T* p) { return to_f32<T>(*p); }

// Block of 128 x 128 elements of op(X) per CTA (256 threads), staged in shared
// memory as fp32; ROWS: one scale per row (1 x 128 blocks), else one per CTA.
// TRANS reads X's rows along op(X)'s columns.
template <typename T, bool ROWS, bool TRANS>
__global__ void __launch_bounds__(256) quant_tile_kernel(const QuantParams p) {
  extern __shared__ float tile[];  // 128 rows of op(X), pitch 129
  __shared__ float warp_max[8];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 128;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(p.x);
  for (int i = warp; i < 128; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = lane + 32 * j;
      if constexpr (!TRANS) {
        const bool in = r0 + i < p.rows && c0 + c < p.cols;
        tile[i * 129 + c] = in ? load_elem(x + (r0 + i) * p.ldx + c0 + c) : 0.f;
      } else {
        const bool in = c0 + i < p.cols && r0 + c < p.rows;
        tile[c * 129 + i] = in ? load_elem(x + (c0 + i) * p.ldx + r0 + c) : 0.f;
      }
    }
  }
  __syncthreads();
  float inv = 0.f, scale = 0.f;
  if constexpr (!ROWS) {
    float m = 0.f;
    for (int i = warp; i < 128; i += 8)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = fmaxf(m, finite_abs(tile[i * 129 + lane + 32 * j]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) warp_max[warp] = m;
    __syncthreads();
    m = warp_max[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = fmaxf(m, warp_max[w]);
    factors(m, inv, scale);
    if (threadIdx.x == 0)
      p.scale[static_cast<int64_t>(blockIdx.y) * p.scale_row + static_cast<int64_t>(blockIdx.x) * p.scale_blk] = scale;
  }
  for (int i = warp; i < 128; i += 8) {
    const int64_t r = r0 + i;
    if (r >= p.rows) break;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = tile[i * 129 + 4 * lane + j];
    if constexpr (ROWS) {
      float m = fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3])));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      factors(m, inv, scale);
      if (lane == 0) p.scale[r * p.scale_row + static_cast<int64_t>(blockIdx.x) * p.scale_blk] = scale;
    }
    const uint32_t w = e4m3x2(scaled(v[0], inv), scaled(v[1], inv)) |
                       e4m3x2(scaled(v[2], inv), scaled(v[3], inv)) << 16;
    const int64_t c = c0 + 4 * lane;
    uint8_t* q = p.q + r * p.ldq + c;
    if (p.q_vec && c + 4 <= p.cols) {
      *reinterpret_cast<uint32_t*>(q) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < p.cols) q[j] = static_cast<uint8_t>(w >> (8 * j));
    }
  }
}

}  // namespace choreo_sm100

namespace choreo_impl {
using namespace choreo_sm100;

namespace {

template <typename T, bool ROWS, bool TRANS>
int launch_quant(const QuantParams& p, cudaStream_t s) {
  constexpr int smem = 128 * 129 * 4;
  auto kern = quant_tile_kernel<T, ROWS, TRANS>;
  static std::atomic<uint64_t> done{0};
  if (int rc = set_smem_limit_once(kern, smem, done, "cudaFuncSetAttribute(quantise)")) return rc;
  const dim3 grid(static_cast<unsigned>((p.cols + 127) / 128), static_cast<unsigned>((p.rows + 127) / 128));
  const cudaError_t e = launch_pdl(kern, grid, dim3(256), smem, s, p);
  return e == cudaSuccess ? CHOREO_OK : cuda_fail(e, "quantise launch");
}

template <typename T>
int dispatch_quant(const QuantParams& p, bool rows, bool trans, cudaStream_t s) {
  if (rows) return trans ? launch_quant<T, true, true>(p, s) : launch_quant<T, true, false>(p, s);
  return trans ? launch_quant<T, false, true>(p, s) : launch_quant<T, false, false>(p, s);
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
  p.x_vec = ((reinterpret_cast<uintptr_t>(d->x) | static_cast<uintptr_t>(d->ldx * dtype_bytes(d->dtype))) & 15u) == 0;
  p.q_vec = ((reinterpret_cast<uintptr_t>(d->q) | static_cast<uintptr_t>(d->ldq)) & 3u) == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool rows = d->block_rows == 1, trans = d->transpose != 0;
  switch (d->dtype) {
    case CHOREO_DTYPE_F16: rc = dispatch_quant<__half>(p, rows, trans, s); break;
    case CHOREO_DTYPE_BF16: rc = dispatch_quant<__nv_bfloat16>(p, rows, trans, s); break;
    default: rc = dispatch_quant<float>(p, rows, trans, s); break;
  }
  return rc ? rc : ok();
}
