// gated_ffn_grad.cu — the backward pass of the gated feed-forward product:
//   1. dG and dU: one elementwise pass over dH and the kept G and U, or, when
//      they were not kept, the gate tiles again with the gradient epilogue.
//   2. dX = dG Wg^T + dU Wu^T: one product over 2 N (SelectLoader by k-block).
//   3. dWg = X^T dG and dWu = X^T dU: one launch, two batch items.
// Every sum runs in a fixed order in fp32, so results repeat bit for bit.
#include <algorithm>
#include <cstring>

#include "gated_ffn.cuh"
#include "gated_ffn.h"
#include "internal.h"

namespace choreo_sm100 {

struct GradElems {
  int64_t m, n;
  const void *dh, *gate, *up;
  int64_t ld_dh, ld_gu;
  void *dg, *du;
  int64_t ld_out;       // multiple of 8; dg and du 16-byte aligned
  void* h;
  int64_t ldh;
  int32_t in_vec, h_vec;  // 16-byte accesses are legal for the inputs / for h
};

// dG, dU (and h) from dH, G and U: 6 bytes read and 4 (6) written per element,
// so bound by memory; eight elements a thread in 16-byte accesses. 2049 x 5632
// f16: 20.7 us alone from a cold cache for 17.6 us of bytes (part of the writes
// stay in L2), 48 registers and so 5 CTAs an SM.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) gate_grad_kernel(const GradElems e) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t chunks = e.ld_out / 8;
  const int64_t total = e.m * chunks;
  const uint16_t* dh = static_cast<const uint16_t*>(e.dh);
  const uint16_t* gate = static_cast<const uint16_t*>(e.gate);
  const uint16_t* up = static_cast<const uint16_t*>(e.up);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / chunks;
    const int64_t c0 = (i - r * chunks) * 8;
    const bool full = c0 + 8 <= e.n;
    uint32_t d[4], g[4], u[4];
    if (e.in_vec && full) {
      const uint4 dv = *reinterpret_cast<const uint4*>(dh + r * e.ld_dh + c0);
      const uint4 gv = *reinterpret_cast<const uint4*>(gate + r * e.ld_gu + c0);
      const uint4 uv = *reinterpret_cast<const uint4*>(up + r * e.ld_gu + c0);
      d[0] = dv.x, d[1] = dv.y, d[2] = dv.z, d[3] = dv.w;
      g[0] = gv.x, g[1] = gv.y, g[2] = gv.z, g[3] = gv.w;
      u[0] = uv.x, u[1] = uv.y, u[2] = uv.z, u[3] = uv.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[j] = g[j] = u[j] = 0;
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (c0 + 2 * j + q < e.n) {
            d[j] |= static_cast<uint32_t>(dh[r * e.ld_dh + c0 + 2 * j + q]) << (16 * q);
            g[j] |= static_cast<uint32_t>(gate[r * e.ld_gu + c0 + 2 * j + q]) << (16 * q);
            u[j] |= static_cast<uint32_t>(up[r * e.ld_gu + c0 + 2 * j + q]) << (16 * q);
          }
      }
    }
    uint32_t og[4], ou[4], oh[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float dd[2], gg[2], uu[2], a[2], b[2], h[2];
      unpack2(d[j], dd[0], dd[1], static_cast<T*>(nullptr));
      unpack2(g[j], gg[0], gg[1], static_cast<T*>(nullptr));
      unpack2(u[j], uu[0], uu[1], static_cast<T*>(nullptr));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float v, dv;
        act_value_slope<ACT>(gg[q], v, dv);
        a[q] = dd[q] * uu[q] * dv;
        b[q] = dd[q] * v;
        h[q] = v * uu[q];
      }
      og[j] = pack2(a[0], a[1], static_cast<T*>(nullptr));
      ou[j] = pack2(b[0], b[1], static_cast<T*>(nullptr));
      oh[j] = pack2(h[0], h[1], static_cast<T*>(nullptr));
    }
    // the workspace rows are padded to 8 elements: whole vectors, also at the edge
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(e.dg) + r * e.ld_out + c0) = make_uint4(og[0], og[1], og[2], og[3]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(e.du) + r * e.ld_out + c0) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
    if (e.h != nullptr) {
      uint16_t* h = static_cast<uint16_t*>(e.h) + r * e.ldh + c0;
      if (e.h_vec && full) {
        *reinterpret_cast<uint4*>(h) = make_uint4(oh[0], oh[1], oh[2], oh[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + j < e.n) h[j] = static_cast<uint16_t>(oh[j / 2] >> (16 * (j & 1)));
      }
    }
  }
}

}  // namespace choreo_sm100

namespace choreo_impl {
using namespace choreo_sm100;

namespace {

constexpr unsigned kSelectTiles = kTileWide256 | kTilePair256 | kTileSingle128;
// The 256 x 256 pair tile runs these products as fast as the wide one where both
// need the same number of rounds, so the cost model gives them nearly one rate
// (wide256's is 1.21) and the rounds decide: dWg and dWu at 2049 x 2048 x 5632,
// six rounds of half tiles wide and five in pairs, 93 and 86 us; dX at 4096 x
// 2048 x 5632, two either way, 160 and 165.
constexpr double kPairRate = 1.15;

template <typename Kern>
int launch_select(Kern kern, int smem, std::atomic<uint64_t>& attr_done, const TwoMaps& ta, const TwoMaps& tb,
                  const TwoMaps& tc, const SelectParams& kp, int grid, cudaStream_t s) {
  if (int rc = set_smem_limit_once(kern, smem, attr_done, "cudaFuncSetAttribute(gated backward)")) return rc;
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kThreads), smem, s, ta, tb, tc, kp);
  return e == cudaSuccess ? CHOREO_OK : cuda_fail(e, "gated feed-forward backward launch");
}

template <bool BY_K, bool A_MN, bool B_MN, typename OutT>
int dispatch_tile(const TcConfig& cfg, const TwoMaps& ta, const TwoMaps& tb, const TwoMaps& tc, const SelectParams& kp,
                  int grid, cudaStream_t s) {
  using Epi = SelectEpi<OutT, BY_K>;
  if (cfg.wide) {
    static std::atomic<uint64_t> done{0};
    return launch_select(tc_gemm_pair_wide_kernel<kWideStages, SelectLoader<BY_K, A_MN, B_MN, 128, true>, Epi>,
                         tc_wide_smem_bytes<kWideStages>(), done, ta, tb, tc, kp, grid, s);
  }
  if (cfg.pair) {
    constexpr int ST = pair_stages_for(256);
    static std::atomic<uint64_t> done{0};
    return launch_select(tc_gemm_pair_kernel<256, ST, SelectLoader<BY_K, A_MN, B_MN, 128, true>, Epi>,
                         tc_pair_smem_bytes<256, ST>(), done, ta, tb, tc, kp, grid, s);
  }
  constexpr int ST = stages_for(128);
  static std::atomic<uint64_t> done{0};
  return launch_select(tc_gemm_kernel<128, ST, SelectLoader<BY_K, A_MN, B_MN, 128, false>, Epi>,
                       tc_smem_bytes<128, ST>(), done, ta, tb, tc, kp, grid, s);
}

template <bool BY_K, bool A_MN, bool B_MN>
int dispatch(const TcConfig& cfg, int dtype_c, const TwoMaps& ta, const TwoMaps& tb, const TwoMaps& tc,
             const SelectParams& kp, int grid, cudaStream_t s) {
  switch (dtype_c) {
    case CHOREO_DTYPE_F16: return dispatch_tile<BY_K, A_MN, B_MN, __half>(cfg, ta, tb, tc, kp, grid, s);
    case CHOREO_DTYPE_BF16: return dispatch_tile<BY_K, A_MN, B_MN, __nv_bfloat16>(cfg, ta, tb, tc, kp, grid, s);
    default: return dispatch_tile<BY_K, A_MN, B_MN, float>(cfg, ta, tb, tc, kp, grid, s);
  }
}

// Output(s) of a select launch: whether bulk tensor stores and 16-byte vectors
// are legal for every one, and their maps. rows x cols each, `items` of them
// per output at `stride` (K-split partials).
int encode_outputs(SelectParams* kp, TwoMaps* tc, int dtype_c, void* c0, void* c1, int64_t rows, int64_t cols,
                   int64_t ld, int64_t items, int64_t stride) {
  const int eb = dtype_bytes(dtype_c);
  std::memset(tc, 0, sizeof(*tc));
  kp->c = c0;
  kp->c1 = c1;
  kp->ldc = ld;
  kp->stride_c = stride;
  bool legal = (ld * eb) % 16 == 0 && (items == 1 || (stride * eb) % 16 == 0);
  for (void* c : {c0, c1})
    if (reinterpret_cast<uintptr_t>(c) & 15u) legal = false;
  kp->c_vec_ok = kp->c_tma = legal ? 1 : 0;
  if (kp->c_tma == 0) return CHOREO_OK;
  kp->n_bulk = bulk_columns(cols, eb);
  const CUtensorMapDataType dt = dtype_c == CHOREO_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : dtype_c == CHOREO_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), static_cast<uint64_t>(items)};
  const uint64_t bstride = static_cast<uint64_t>(items > 1 ? stride : rows * ld) * eb;
  const uint64_t strides[2] = {static_cast<uint64_t>(ld) * eb, bstride};
  const uint32_t box[3] = {static_cast<uint32_t>(128 / eb), 32, 1};
  for (int i = 0; i < 2; ++i) {
    void* c = i == 0 ? c0 : c1;
    if (c == nullptr) continue;
    if (int rc = encode_tmap(&tc->m[i], dt, 3, c, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  return CHOREO_OK;
}

int launch_gate_grad(const GradElems& e, bool bf16, int act, cudaStream_t s) {
  const int64_t work = e.m * (e.ld_out / 8);
  const unsigned grid =
      static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((work + 255) / 256, int64_t{8} * current_sm_count())));
  auto go = [&](auto kern) {
    const cudaError_t err = launch_pdl(kern, dim3(grid), dim3(256), 0, s, e);
    return err == cudaSuccess ? static_cast<int>(CHOREO_OK) : cuda_fail(err, "gate gradient launch");
  };
  if (bf16) {
    switch (act) {
      case CHOREO_ACT_SILU: return go(gate_grad_kernel<__nv_bfloat16, CHOREO_ACT_SILU>);
      case CHOREO_ACT_GELU: return go(gate_grad_kernel<__nv_bfloat16, CHOREO_ACT_GELU>);
      case CHOREO_ACT_GELU_TANH: return go(gate_grad_kernel<__nv_bfloat16, CHOREO_ACT_GELU_TANH>);
      default: return go(gate_grad_kernel<__nv_bfloat16, CHOREO_ACT_RELU>);
    }
  }
  switch (act) {
    case CHOREO_ACT_SILU: return go(gate_grad_kernel<__half, CHOREO_ACT_SILU>);
    case CHOREO_ACT_GELU: return go(gate_grad_kernel<__half, CHOREO_ACT_GELU>);
    case CHOREO_ACT_GELU_TANH: return go(gate_grad_kernel<__half, CHOREO_ACT_GELU_TANH>);
    default: return go(gate_grad_kernel<__half, CHOREO_ACT_RELU>);
  }
}

// Where the workspace's parts start; dX's plan.
struct GradPlan {
  FfnOperands ops;
  int64_t n_pad = 0;
  int64_t dg = 0, du = 0;        // offsets
  int64_t partials = 0;          // offset of dX's K-split partials
  int64_t bytes = 0, min_bytes = 0;
  TilePlan dx;                   // with a K split when that is faster
  TcConfig dx_unsplit{};
};

GradPlan plan_grad(const choreo_ffn_grad_desc& d) {
  GradPlan g;
  plan_ffn_operands(&g.ops, d.x, d.ldx, d.w_gate, d.w_up, d.ldw, d.trans_w != 0, d.m, d.n, d.k);
  g.n_pad = round_up(d.n, 8);
  const int64_t side = round_up(d.m * g.n_pad * 2, 256);
  g.dg = g.ops.bytes;
  g.du = g.dg + side;
  g.min_bytes = g.bytes = g.du + side;
  if (d.dx != nullptr) {
    const int64_t kb = 2 * ((d.n + kBK - 1) / kBK);
    const int sms = current_sm_count();
    g.dx = plan_tiles(d.m, d.k, kb, 1, sms, true, 2, kSelectTiles, kPairRate);
    g.dx_unsplit = g.dx.split > 1 ? plan_tiles(d.m, d.k, kb, 1, sms, false, 2, kSelectTiles, kPairRate).cfg : g.dx.cfg;
    if (g.dx.split > 1) {
      g.partials = g.bytes;
      g.bytes += round_up(g.dx.split * d.m * d.k * 4, 256);
    }
  }
  return g;
}

int launch_dx(const choreo_ffn_grad_desc& d, const GradPlan& g, bool split, const void* dg, const void* du,
              const void* w_gate, const void* w_up, int64_t ldw, float* partials, cudaStream_t s) {
  const bool bf16 = d.dtype == CHOREO_DTYPE_BF16;
  const TcConfig& cfg = split ? g.dx.cfg : g.dx_unsplit;
  const int64_t kb1 = (d.n + kBK - 1) / kBK;
  const int64_t items = split ? g.dx.split : 1;
  TwoMaps ta, tb, tc;
  int rc;
  for (int i = 0; i < 2; ++i) {
    rc = encode_matrix(&ta.m[i], bf16, i == 0 ? dg : du, d.m, d.n, g.n_pad, 64, cfg.wide ? 256u : 128u);
    if (rc) return rc;
    // W K x N is the product's B stored N x K (contracted index contiguous); W N x K is its transpose
    const void* w = i == 0 ? w_gate : w_up;
    rc = d.trans_w ? encode_matrix(&tb.m[i], bf16, w, d.n, d.k, ldw, 64, 64)
                   : encode_matrix(&tb.m[i], bf16, w, d.k, d.n, ldw, 64, 128);
    if (rc) return rc;
  }
  SelectParams kp;
  std::memset(&kp, 0, sizeof(kp));
  int grid = 0;
  rc = fill_tc_params(&kp, d.m, d.k, (d.k + cfg.bn - 1) / cfg.bn, 2 * kb1 / items, items, cfg, bf16, &grid);
  if (rc) return rc;
  kp.k_blocks_1 = static_cast<int32_t>(kb1);
  kp.split_kb = split ? kp.num_k_blocks : 0;
  const int dtype_c = split ? CHOREO_DTYPE_F32 : d.dtype;
  rc = split ? encode_outputs(&kp, &tc, dtype_c, partials, nullptr, d.m, d.k, d.k, items, d.m * d.k)
             : encode_outputs(&kp, &tc, dtype_c, d.dx, nullptr, d.m, d.k, d.ld_dx, 1, 0);
  if (rc) return rc;
  rc = d.trans_w ? dispatch<true, false, true>(cfg, dtype_c, ta, tb, tc, kp, grid, s)
                 : dispatch<true, false, false>(cfg, dtype_c, ta, tb, tc, kp, grid, s);
  if (rc || !split) return rc;
  return launch_splitk_reduce(partials, items, d.m, d.k, d.dx, d.ld_dx, d.dtype, 1.f, 0.f, nullptr, CHOREO_DTYPE_F32, 0,
                              s);
}

int launch_dw(const choreo_ffn_grad_desc& d, int64_t n_pad, const void* dg, const void* du, const void* x, int64_t ldx,
              cudaStream_t s) {
  const bool bf16 = d.dtype == CHOREO_DTYPE_BF16;
  // dW K x N = X^T dG, or its transpose N x K = dG^T X: the summed index M is
  // the slow one of both operands, so both tiles are MN-major.
  const int64_t rows = d.trans_w ? d.n : d.k, cols = d.trans_w ? d.k : d.n;
  const int64_t kb = (d.m + kBK - 1) / kBK;
  const TcConfig cfg =
      plan_tiles(rows, cols, kb, 2, current_sm_count(), false, dtype_bytes(d.dtype_dw), kSelectTiles, kPairRate).cfg;
  TwoMaps ta, tb, tc;
  int rc;
  for (int i = 0; i < 2; ++i) {
    const void* g = i == 0 ? dg : du;
    CUtensorMap* mx = d.trans_w ? &tb.m[i] : &ta.m[i];
    CUtensorMap* mg = d.trans_w ? &ta.m[i] : &tb.m[i];
    if ((rc = encode_matrix(mx, bf16, x, d.m, d.k, ldx, 64, 64))) return rc;
    if ((rc = encode_matrix(mg, bf16, g, d.m, d.n, n_pad, 64, 64))) return rc;
  }
  SelectParams kp;
  std::memset(&kp, 0, sizeof(kp));
  int grid = 0;
  rc = fill_tc_params(&kp, rows, cols, (cols + cfg.bn - 1) / cfg.bn, kb, 2, cfg, bf16, &grid);
  if (rc) return rc;
  kp.beta = d.accumulate_dw ? 1.f : 0.f;
  if ((rc = encode_outputs(&kp, &tc, d.dtype_dw, d.dw_gate, d.dw_up, rows, cols, d.ld_dw, 1, 0))) return rc;
  return dispatch<false, true, true>(cfg, d.dtype_dw, ta, tb, tc, kp, grid, s);
}

int validate_grad(const choreo_ffn_grad_desc* d) {
  const char* what = "gated FFN backward";
  if (d == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "%s: null descriptor", what);
  int rc = check_ffn_common(what, d->m, d->n, d->k, d->dtype, d->act, d->x, d->ldx, d->w_gate, d->w_up, d->ldw,
                            d->trans_w);
  if (rc) return rc;
  if (d->dh == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "%s: dH has null data pointer", what);
  if (d->ld_dh < d->n)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: ld_dh=%lld smaller than N=%lld", what, (long long)d->ld_dh, (long long)d->n);
  if ((d->gate == nullptr) != (d->up == nullptr))
    return fail(CHOREO_ERR_INVALID_ARG, "%s: gate and up are kept together: one is NULL", what);
  if (d->gate && d->ld_gu < d->n)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: ld_gu=%lld smaller than N=%lld", what, (long long)d->ld_gu,
                (long long)d->n);
  if ((d->dw_gate == nullptr) != (d->dw_up == nullptr))
    return fail(CHOREO_ERR_INVALID_ARG, "%s: dw_gate and dw_up are computed together: one is NULL", what);
  if (d->dx == nullptr && d->dw_gate == nullptr)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: neither dX nor the weight gradients are wanted", what);
  if (d->dx && d->ld_dx < d->k)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: ld_dx=%lld smaller than K=%lld", what, (long long)d->ld_dx, (long long)d->k);
  if (d->dw_gate) {
    const int64_t inner = d->trans_w ? d->k : d->n;
    if (d->ld_dw < inner)
      return fail(CHOREO_ERR_INVALID_ARG, "%s: ld_dw=%lld smaller than %lld", what, (long long)d->ld_dw,
                  (long long)inner);
    if (d->dtype_dw != d->dtype && d->dtype_dw != CHOREO_DTYPE_F32)
      return fail(CHOREO_ERR_UNSUPPORTED, "%s: dtype_dw %d is neither dtype nor f32", what, d->dtype_dw);
  }
  if (d->h && d->ldh < d->n)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: ldh=%lld smaller than N=%lld", what, (long long)d->ldh, (long long)d->n);
  const struct {
    const void* p;
    const char* name;
  } ptrs[] = {{d->x, "gated FFN backward X"},         {d->w_gate, "gated FFN backward Wg"},
              {d->w_up, "gated FFN backward Wu"},     {d->dh, "gated FFN backward dH"},
              {d->gate, "gated FFN backward gate"},   {d->up, "gated FFN backward up"},
              {d->dx, "gated FFN backward dX"},       {d->dw_gate, "gated FFN backward dWg"},
              {d->dw_up, "gated FFN backward dWu"},   {d->h, "gated FFN backward H"}};
  for (const auto& q : ptrs)
    if (q.p && (rc = check_device_ptr(q.p, q.name))) return rc;
  return CHOREO_OK;
}

}  // namespace
}  // namespace choreo_impl

using namespace choreo_impl;

extern "C" {

int choreo_gated_ffn_backward_query(const choreo_ffn_grad_desc* d, choreo_launch_config* out) {
  int rc = validate_grad(d);
  if (rc) return rc;
  if (out == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "gated FFN backward query: null output");
  std::memset(out, 0, sizeof(*out));
  const GradPlan g = plan_grad(*d);
  out->kernel = 4;
  out->split_k = 1;
  if (d->dx != nullptr) {
    const TcConfig& c = g.dx.cfg;
    out->tile_m = tile_rows_of(c);
    out->tile_n = c.bn;
    out->tile_k = kBK;
    out->stages = c.stages;
    out->cluster_m = c.pair ? 2 : 1;
    out->tiles = ((d->m + out->tile_m - 1) / out->tile_m) * ((d->k + c.bn - 1) / c.bn) * g.dx.split;
    const int sms = current_sm_count();
    out->grid_x = static_cast<int32_t>(c.pair ? 2 * std::min<int64_t>(out->tiles, sms / 2)
                                              : std::min<int64_t>(out->tiles, sms));
    out->grid_y = out->grid_z = 1;
    out->block_x = kTcThreads;
    out->smem_bytes = c.smem;
    out->tmem_cols = c.wide ? 512 : 2 * c.bn;
    out->split_k = g.dx.split;
  }
  out->workspace_bytes = g.bytes;
  out->workspace_min_bytes = g.min_bytes;
  return ok();
}

int choreo_gated_ffn_backward(const choreo_ffn_grad_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = validate_grad(d);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const GradPlan g = plan_grad(*d);
  if ((rc = check_workspace("gated FFN backward", workspace, workspace_bytes, g.min_bytes))) return rc;
  const bool split = g.dx.split > 1 && workspace_bytes >= static_cast<size_t>(g.bytes);
  char* ws = static_cast<char*>(workspace);
  const bool bf16 = d->dtype == CHOREO_DTYPE_BF16;
  const void *x = d->x, *w_gate = d->w_gate, *w_up = d->w_up;
  int64_t ldx = d->ldx, ldw = d->ldw;
  if ((rc = repack_ffn_operands(g.ops, ws, &x, &ldx, &w_gate, &w_up, &ldw, s))) return rc;
  void* dg = ws + g.dg;
  void* du = ws + g.du;
  if (d->gate != nullptr) {
    GradElems e{};
    e.m = d->m;
    e.n = d->n;
    e.dh = d->dh;
    e.ld_dh = d->ld_dh;
    e.gate = d->gate;
    e.up = d->up;
    e.ld_gu = d->ld_gu;
    e.dg = dg;
    e.du = du;
    e.ld_out = g.n_pad;
    e.h = d->h;
    e.ldh = d->ldh;
    const uintptr_t in = reinterpret_cast<uintptr_t>(d->dh) | reinterpret_cast<uintptr_t>(d->gate) |
                         reinterpret_cast<uintptr_t>(d->up) | static_cast<uintptr_t>(d->ld_dh * 2) |
                         static_cast<uintptr_t>(d->ld_gu * 2);
    e.in_vec = (in & 15u) == 0 ? 1 : 0;
    e.h_vec = ((reinterpret_cast<uintptr_t>(d->h) | static_cast<uintptr_t>(d->ldh * 2)) & 15u) == 0 ? 1 : 0;
    rc = launch_gate_grad(e, bf16, d->act, s);
  } else {
    GateProblem p{};
    p.m = d->m;
    p.n = d->n;
    p.k = d->k;
    p.bf16 = bf16;
    p.act = d->act;
    p.x = x;
    p.ldx = ldx;
    p.w_gate = w_gate;
    p.w_up = w_up;
    p.ldw = ldw;
    p.w_mn = d->trans_w == 0;
    p.h = d->h;
    p.ldh = d->ldh;
    p.out1 = dg;
    p.out2 = du;
    p.ld12 = g.n_pad;
    p.dh = d->dh;
    p.ld_dh = d->ld_dh;
    rc = launch_gate_tiles(p, s);
  }
  if (rc) return rc;
  if (d->dx != nullptr) {
    rc = launch_dx(*d, g, split, dg, du, w_gate, w_up, ldw, reinterpret_cast<float*>(ws + g.partials), s);
    if (rc) return rc;
  }
  if (d->dw_gate != nullptr) {
    rc = launch_dw(*d, g.n_pad, dg, du, x, ldx, s);
    if (rc) return rc;
  }
  return ok();
}

}  // extern "C"
