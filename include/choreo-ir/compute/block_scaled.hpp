/**
 * @file block_scaled.hpp
 * @brief 8-bit operands with one scale per block of 128 over the C ABI
 *        (choreo_quantize_block, choreo_gemm_block_scaled). Device tensors
 *        only; e4m3 codes are held as uint8_t. The reference has no
 *        counterpart (its 8-bit type is INT8, without a product).
 */
#ifndef CHOREO_IR_COMPUTE_BLOCK_SCALED_HPP
#define CHOREO_IR_COMPUTE_BLOCK_SCALED_HPP

#include <cuda_runtime.h>

#include <type_traits>

#include "../../choreo_b200.h"
#include "gated_ffn.hpp"
#include "matmul.hpp"
#include "validation.hpp"

namespace choreo_ir {
namespace compute {

/// An e4m3 matrix (rows padded to 16 bytes, as the product wants them) and its
/// scales, those of one k-block side by side.
struct BlockScaled {
  index_t rows = 0, cols = 0;
  index_t block_rows = 1;          // 1: a scale per 1 x 128, 128: per 128 x 128
  Tensor<uint8_t> codes;           // rows x (cols rounded up to 16)
  Tensor<float> scales;            // ceil(cols / 128) x ceil(rows / block_rows)

  BlockScaled(index_t r, index_t c, index_t block)
      : rows(r), cols(c), block_rows(checked(block)), codes(Shape({r, (c + 15) / 16 * 16}), MemoryType::DEVICE),
        scales(Shape({(c + 127) / 128, (r + block - 1) / block}), MemoryType::DEVICE) {}
  static index_t checked(index_t block) {
    if (block != 1 && block != 128) throw ValidationError("BlockScaled: block_rows must be 1 or 128");
    return block;
  }
  index_t ld() const { return (cols + 15) / 16 * 16; }
  index_t row_blocks() const { return (rows + block_rows - 1) / block_rows; }
};

/// Quantises X (its transpose with `transpose`) into `out`, whose extents must
/// match. X is f16, bf16 or f32, row-major.
template <typename T>
void quantize_block(const Tensor<T>& X, BlockScaled& out, bool transpose = false, cudaStream_t stream = nullptr) {
  constexpr int dt = choreo_ir::detail::abi_dtype<T>();
  static_assert(dt >= 0, "quantize_block needs f16, bf16 or float");
  if (X.ndims() != 2) throw ValidationError("quantize_block: X must be 2-D");
  const index_t r = X.shape()[transpose ? 1 : 0], c = X.shape()[transpose ? 0 : 1];
  if (r != out.rows || c != out.cols)
    throw ValidationError("quantize_block: output must be " + detail::dims(r, c));
  choreo_quant_desc d{};
  d.rows = X.shape()[0];
  d.cols = X.shape()[1];
  d.dtype = dt;
  d.transpose = transpose ? 1 : 0;
  d.ldx = detail::row_major(X, d.rows, d.cols, "quantize_block", "X");
  d.x = X.data();
  d.block_rows = static_cast<int32_t>(out.block_rows);
  d.q = out.codes.data();
  d.ldq = out.ld();
  d.scale = out.scales.data();
  d.scale_row = 1;
  d.scale_blk = out.row_blocks();
  choreo_ir::detail::status_check(choreo_quantize_block(&d, stream));
}

/// Allocating form.
template <typename T>
BlockScaled quantize_block(const Tensor<T>& X, index_t block_rows = 1, bool transpose = false,
                           cudaStream_t stream = nullptr) {
  if (X.ndims() != 2) throw ValidationError("quantize_block: X must be 2-D");
  if (block_rows != 1 && block_rows != 128) throw ValidationError("quantize_block: block_rows must be 1 or 128");
  BlockScaled out(X.shape()[transpose ? 1 : 0], X.shape()[transpose ? 0 : 1], block_rows);
  quantize_block(X, out, transpose, stream);
  return out;
}

/// C = act(alpha * A B^T + beta * D + bias): A M x K in 1 x 128 blocks, B N x K
/// in 1 x 128 or 128 x 128 blocks, D the addend (C itself when null). bias,
/// relu, stream and synchronize are taken from `config`.
template <typename TC>
void gemm_block_scaled(const BlockScaled& A, const BlockScaled& B, Tensor<TC>& C, float alpha = 1.0f, float beta = 0.0f,
                       const Tensor<TC>* D = nullptr, const GEMMConfig& config = GEMMConfig()) {
  constexpr int dt = choreo_ir::detail::abi_dtype<TC>();
  static_assert(dt >= 0, "gemm_block_scaled writes f16, bf16 or float");
  if (A.block_rows != 1) throw ValidationError("gemm_block_scaled: A needs 1 x 128 blocks");
  if (A.cols != B.cols) throw ValidationError("gemm_block_scaled: A and B differ in K");
  choreo_gemm_block_desc d{};
  d.m = A.rows;
  d.n = B.rows;
  d.k = A.cols;
  d.a = A.codes.data();
  d.lda = A.ld();
  d.scale_a = A.scales.data();
  d.scale_a_row = 1;
  d.scale_a_blk = A.row_blocks();
  d.b = B.codes.data();
  d.ldb = B.ld();
  d.scale_b = B.scales.data();
  d.scale_b_row = 1;
  d.scale_b_blk = B.row_blocks();
  d.block_b = static_cast<int32_t>(B.block_rows);
  d.dtype_c = dt;
  d.ldc = detail::row_major(C, d.m, d.n, "gemm_block_scaled", "C");
  d.c = C.data();
  d.alpha = alpha;
  d.beta = beta;
  if (D != nullptr) {
    d.ld_addend = detail::row_major(*D, d.m, d.n, "gemm_block_scaled", "D");
    d.addend = D->data();
  }
  d.bias = config.bias;
  d.dtype_bias = static_cast<int32_t>(config.bias_dtype);
  d.relu = config.relu ? 1 : 0;
  choreo_ir::detail::status_check(choreo_gemm_block_scaled(&d, config.stream));
  if (config.synchronize) choreo_ir::detail::status_check(choreo_sync_status(config.stream));
}

}  // namespace compute
}  // namespace choreo_ir

#endif  // CHOREO_IR_COMPUTE_BLOCK_SCALED_HPP
