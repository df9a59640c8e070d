/**
 * @file gated_ffn.hpp
 * @brief The gated feed-forward product H = act(X Wg) * (X Wu) and its
 *        backward pass over the C ABI (choreo_gated_ffn). Device tensors
 *        only. As in matmul.hpp, operand layout comes from the strides: the
 *        weights are K x N, row-major or as the transpose() view of N x K
 *        storage, both in the same layout. The reference has no counterpart.
 */
#ifndef CHOREO_IR_COMPUTE_GATED_FFN_HPP
#define CHOREO_IR_COMPUTE_GATED_FFN_HPP

#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "../../choreo_b200.h"
#include "matmul.hpp"
#include "validation.hpp"

namespace choreo_ir {
namespace compute {

enum class Activation : int32_t {
  SILU = CHOREO_ACT_SILU,
  GELU = CHOREO_ACT_GELU,
  GELU_TANH = CHOREO_ACT_GELU_TANH,
  RELU = CHOREO_ACT_RELU
};

struct GatedFfnConfig {
  Activation activation = Activation::SILU;
  cudaStream_t stream = nullptr;
  // Synchronize the stream and check the kernel status word after the call.
  bool synchronize = false;
};

namespace detail {

template <typename View>
using element_t = std::remove_cv_t<std::remove_pointer_t<decltype(std::declval<View>().data())>>;

// Tensor carries where it lives; a view is taken to be device memory, which
// the C ABI checks.
template <typename T>
void require_device(const Tensor<T>& t, const char* what) {
  if (t.memory_type() == MemoryType::HOST) throw ValidationError(std::string(what) + ": device tensors required");
}
template <typename T>
void require_device(const TensorView<T>&, const char*) {}

/// A row-major matrix of the given extents; its leading dimension.
template <typename View>
index_t row_major(const View& t, index_t rows, index_t cols, const char* what, const char* name) {
  require_device(t, what);
  if (t.ndims() != 2 || t.shape()[0] != rows || t.shape()[1] != cols)
    throw ValidationError(std::string(what) + ": " + name + " must be " + detail::dims(rows, cols));
  const index_t ld = t.stride()[0];
  if (cols > 1 && t.stride()[1] != 1)
    throw ValidationError(std::string(what) + ": " + name + " must be row-major (last dimension contiguous)");
  return rows == 1 && ld < cols ? cols : ld;
}

struct FfnWeights {
  index_t ld = 0;
  bool trans = false;   // stored N x K
};
template <typename VG, typename VU>
FfnWeights ffn_weights(const VG& Wg, const VU& Wu, index_t K, const char* what) {
  require_device(Wg, what);
  require_device(Wu, what);
  if (Wg.ndims() != 2 || Wu.ndims() != 2 || Wg.shape()[0] != K || Wu.shape()[0] != K || Wg.shape()[1] != Wu.shape()[1])
    throw ValidationError(std::string(what) + ": the weights must be K x N with K = " + std::to_string(K));
  const MatrixStrides g = matrix_strides(Wg.shape(), Wg.stride()), u = matrix_strides(Wu.shape(), Wu.stride());
  if (!g.valid || !u.valid || g.transposed != u.transposed || g.ld != u.ld)
    throw ValidationError(std::string(what) + ": the weights must share one layout with a contiguous row or column");
  return FfnWeights{g.ld, g.transposed};
}

template <typename T>
void* mutable_data(const T* p) {
  return const_cast<std::remove_const_t<T>*>(p);
}

}  // namespace detail

/// H = act(X Wg) * (X Wu); gate and up, when given, receive X Wg and X Wu for
/// the backward pass. Tensors or views of f16 or bf16.
template <typename VX, typename VG, typename VU, typename VH>
void gated_ffn(const VX& X, const VG& Wg, const VU& Wu, const VH& H, const GatedFfnConfig& cfg = GatedFfnConfig(),
               const VH* gate = nullptr, const VH* up = nullptr) {
  using T = detail::element_t<VX>;
  static_assert(std::is_same_v<T, float16_t> || std::is_same_v<T, bfloat16_t>, "gated_ffn needs f16 or bf16");
  static_assert(std::is_same_v<T, detail::element_t<VG>> && std::is_same_v<T, detail::element_t<VU>> &&
                    std::is_same_v<T, detail::element_t<VH>>, "gated_ffn: one element type");
  const char* what = "gated_ffn";
  if (X.ndims() != 2) throw ValidationError("gated_ffn: X must be 2-D");
  choreo_ffn_desc d{};
  d.m = X.shape()[0];
  d.k = X.shape()[1];
  const detail::FfnWeights w = detail::ffn_weights(Wg, Wu, d.k, what);
  d.n = Wg.shape()[1];
  d.dtype = choreo_ir::detail::abi_dtype<T>();
  d.act = static_cast<int32_t>(cfg.activation);
  d.ldx = detail::row_major(X, d.m, d.k, what, "X");
  d.ldw = w.ld;
  d.trans_w = w.trans ? 1 : 0;
  d.ldh = detail::row_major(H, d.m, d.n, what, "H");
  d.x = X.data();
  d.w_gate = Wg.data();
  d.w_up = Wu.data();
  d.h = detail::mutable_data(H.data());
  if (gate || up) {
    if (!gate || !up) throw ValidationError("gated_ffn: gate and up are kept together");
    d.ld_gu = detail::row_major(*gate, d.m, d.n, what, "gate");
    if (detail::row_major(*up, d.m, d.n, what, "up") != d.ld_gu)
      throw ValidationError("gated_ffn: gate and up must have the same row stride");
    d.gate = detail::mutable_data(gate->data());
    d.up = detail::mutable_data(up->data());
  }
  choreo_launch_config q;
  choreo_ir::detail::status_check(choreo_gated_ffn_query(&d, &q));
  void* ws = nullptr;
  if (q.workspace_bytes > 0)
    choreo_ir::detail::cuda_check(cudaMallocAsync(&ws, static_cast<size_t>(q.workspace_bytes), cfg.stream),
                                  "gated_ffn workspace");
  const int rc = choreo_gated_ffn(&d, ws, static_cast<size_t>(q.workspace_bytes), cfg.stream);
  if (ws) cudaFreeAsync(ws, cfg.stream);
  choreo_ir::detail::status_check(rc);
  if (cfg.synchronize) choreo_ir::detail::status_check(choreo_sync_status(cfg.stream));
}

/// Allocating form: H in device memory.
template <typename T>
Tensor<T> gated_ffn(const Tensor<T>& X, const Tensor<T>& Wg, const Tensor<T>& Wu,
                    const GatedFfnConfig& cfg = GatedFfnConfig()) {
  if (X.ndims() != 2 || Wg.ndims() != 2) throw ValidationError("gated_ffn: X and the weights must be 2-D");
  Tensor<T> H(Shape({X.shape()[0], Wg.shape()[1]}), MemoryType::DEVICE);
  gated_ffn(X, Wg, Wu, H, cfg);
  return H;
}

/// What the backward pass writes and reads besides its operands; null: left
/// out (gate and up null: computed again). T is X's type, TW T or float.
template <typename T, typename TW = T>
struct GatedFfnGrads {
  Tensor<T>* dX = nullptr;
  Tensor<TW>* dWg = nullptr;   // laid out like the weights' storage: K x N, or N x K for transpose() views of it
  Tensor<TW>* dWu = nullptr;
  Tensor<T>* H = nullptr;
  const Tensor<T>* gate = nullptr;
  const Tensor<T>* up = nullptr;
  bool accumulate = false;     // add to what dWg and dWu hold
};

/// Gradients of gated_ffn from dH (choreo_gated_ffn_backward). Operands as in
/// gated_ffn: tensors or views, the weights row-major K x N or as transpose()
/// views of N x K storage.
template <typename T, typename TW, typename VD, typename VX, typename VG, typename VU>
void gated_ffn_backward(const VD& dH, const VX& X, const VG& Wg, const VU& Wu, const GatedFfnGrads<T, TW>& out,
                        const GatedFfnConfig& cfg = GatedFfnConfig()) {
  static_assert(std::is_same_v<T, float16_t> || std::is_same_v<T, bfloat16_t>, "gated_ffn needs f16 or bf16");
  static_assert(std::is_same_v<T, detail::element_t<VD>> && std::is_same_v<T, detail::element_t<VX>> &&
                    std::is_same_v<T, detail::element_t<VG>> && std::is_same_v<T, detail::element_t<VU>>,
                "gated_ffn_backward: one element type");
  static_assert(std::is_same_v<TW, T> || std::is_same_v<TW, float>, "weight gradients: the weights' type or float");
  const char* what = "gated_ffn_backward";
  if (X.ndims() != 2) throw ValidationError("gated_ffn_backward: X must be 2-D");
  choreo_ffn_grad_desc d{};
  d.m = X.shape()[0];
  d.k = X.shape()[1];
  const detail::FfnWeights w = detail::ffn_weights(Wg, Wu, d.k, what);
  d.n = Wg.shape()[1];
  d.dtype = choreo_ir::detail::abi_dtype<T>();
  d.dtype_dw = choreo_ir::detail::abi_dtype<TW>();
  d.act = static_cast<int32_t>(cfg.activation);
  d.ldx = detail::row_major(X, d.m, d.k, what, "X");
  d.ldw = w.ld;
  d.trans_w = w.trans ? 1 : 0;
  d.ld_dh = detail::row_major(dH, d.m, d.n, what, "dH");
  d.x = X.data();
  d.w_gate = Wg.data();
  d.w_up = Wu.data();
  d.dh = dH.data();
  auto optional = [&](const auto* t, index_t rows, index_t cols, const char* name, int64_t* ld) -> void* {
    if (t == nullptr) return nullptr;
    const index_t l = detail::row_major(*t, rows, cols, what, name);
    if (*ld != 0 && *ld != l) throw ValidationError(std::string(what) + ": " + name + ": row strides differ");
    *ld = l;
    return detail::mutable_data(t->data());
  };
  d.gate = optional(out.gate, d.m, d.n, "gate", &d.ld_gu);
  d.up = optional(out.up, d.m, d.n, "up", &d.ld_gu);
  d.dx = optional(out.dX, d.m, d.k, "dX", &d.ld_dx);
  const index_t w_rows = w.trans ? d.n : d.k, w_cols = w.trans ? d.k : d.n;
  d.dw_gate = optional(out.dWg, w_rows, w_cols, "dWg", &d.ld_dw);
  d.dw_up = optional(out.dWu, w_rows, w_cols, "dWu", &d.ld_dw);
  d.h = optional(out.H, d.m, d.n, "H", &d.ldh);
  d.accumulate_dw = out.accumulate ? 1 : 0;
  choreo_launch_config q;
  choreo_ir::detail::status_check(choreo_gated_ffn_backward_query(&d, &q));
  void* ws = nullptr;
  choreo_ir::detail::cuda_check(cudaMallocAsync(&ws, static_cast<size_t>(q.workspace_bytes), cfg.stream),
                                "gated_ffn_backward workspace");
  const int rc = choreo_gated_ffn_backward(&d, ws, static_cast<size_t>(q.workspace_bytes), cfg.stream);
  cudaFreeAsync(ws, cfg.stream);
  choreo_ir::detail::status_check(rc);
  if (cfg.synchronize) choreo_ir::detail::status_check(choreo_sync_status(cfg.stream));
}

}  // namespace compute
}  // namespace choreo_ir

#endif  // CHOREO_IR_COMPUTE_GATED_FFN_HPP
