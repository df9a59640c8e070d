// gated_ffn.h — host declarations shared by the gated feed-forward product
// (gated_ffn.cu) and its backward pass (gated_ffn_grad.cu).
#pragma once
#include "internal.h"

namespace choreo_sm100 {
struct TcParams;
}

namespace choreo_impl {

// Operands X, Wg and Wu as the kernels read them: repacked into the workspace
// where the TMA cannot address them.
struct FfnOperands {
  OperandPlan x, w;   // w: each of the two weights
  int64_t bytes = 0;
};
void plan_ffn_operands(FfnOperands* o, const void* x, int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw,
                       bool trans_w, int64_t m, int64_t n, int64_t k);
int repack_ffn_operands(const FfnOperands& o, char* ws, const void** x, int64_t* ldx, const void** w_gate,
                        const void** w_up, int64_t* ldw, cudaStream_t s);

// Contracts common to the forward and the backward call.
int check_ffn_common(const char* what, int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t act, const void* x,
                     int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw, int32_t trans_w);
int check_workspace(const char* what, const void* workspace, size_t have, int64_t need);

// One launch of the gate tiles. dh == null: h, and G and U into out1 and out2
// unless those are null. dh != null: dG and dU into out1 and out2, and h
// unless it is null. Operands TMA-legal.
struct GateProblem {
  int64_t m, n, k;
  bool bf16;
  int act;
  const void* x; int64_t ldx;
  const void* w_gate; const void* w_up; int64_t ldw; bool w_mn;   // w_mn: weights stored K x N
  void* h; int64_t ldh;
  void* out1; void* out2; int64_t ld12;
  const void* dh; int64_t ld_dh;
};
TcConfig select_gate_config(int64_t m, int64_t n, int64_t k);
int launch_gate_tiles(const GateProblem& p, cudaStream_t stream);

// Tensor map of a 16-bit row-major matrix, rank 3 with one batch item.
int encode_matrix(CUtensorMap* map, bool bf16, const void* p, int64_t rows, int64_t cols, int64_t ld,
                  uint32_t box_cols, uint32_t box_rows);

// The fields of TcParams that follow from the problem and the tile shape; the
// launch grid in *grid.
int fill_tc_params(choreo_sm100::TcParams* kp, int64_t m, int64_t n, int64_t tiles_n, int64_t k_blocks, int64_t items,
                   const TcConfig& cfg, bool bf16, int* grid);

}  // namespace choreo_impl
