// gated_ffn.cu — the gated feed-forward product H = act(X Wg) * (X Wu): the
// launch of its tile kernels, their planning, and the C entry points.
#include <algorithm>
#include <cstring>

#include "gated_ffn.cuh"
#include "gated_ffn.h"
#include "internal.h"
#include "skinny.cuh"

namespace choreo_impl {
using namespace choreo_sm100;

namespace {

template <typename Kern>
int launch_tiles(Kern kern, int smem, std::atomic<uint64_t>& attr_done, const CUtensorMap& ta, const TwoMaps& tb,
                 const GateMaps& tc, const GateParams& kp, int grid, cudaStream_t s) {
  if (int rc = set_smem_limit_once(kern, smem, attr_done, "cudaFuncSetAttribute(gated)")) return rc;
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kThreads), smem, s, ta, tb, tc, kp);
  return e == cudaSuccess ? CHOREO_OK : cuda_fail(e, "gated feed-forward launch");
}

template <bool W_MN, typename OutT, bool GRAD>
int dispatch_tile(const TcConfig& cfg, const CUtensorMap& ta, const TwoMaps& tb, const GateMaps& tc,
                  const GateParams& kp, int grid, cudaStream_t s) {
  using Epi = GateEpi<OutT, GRAD>;
  if (cfg.pair) {
    constexpr int ST = pair_stages_for(256);
    static std::atomic<uint64_t> done{0};
    return launch_tiles(tc_gemm_pair_kernel<256, ST, GateLoader<W_MN, 128, true>, Epi>, tc_pair_smem_bytes<256, ST>(),
                        done, ta, tb, tc, kp, grid, s);
  }
  constexpr int ST = stages_for(128);
  static std::atomic<uint64_t> done{0};
  return launch_tiles(tc_gemm_kernel<128, ST, GateLoader<W_MN, 128, false>, Epi>, tc_smem_bytes<128, ST>(), done, ta,
                      tb, tc, kp, grid, s);
}

template <bool GRAD>
int dispatch(const TcConfig& cfg, bool w_mn, bool bf16, const CUtensorMap& ta, const TwoMaps& tb, const GateMaps& tc,
             const GateParams& kp, int grid, cudaStream_t s) {
  if (w_mn)
    return bf16 ? dispatch_tile<true, __nv_bfloat16, GRAD>(cfg, ta, tb, tc, kp, grid, s)
                : dispatch_tile<true, __half, GRAD>(cfg, ta, tb, tc, kp, grid, s);
  return bf16 ? dispatch_tile<false, __nv_bfloat16, GRAD>(cfg, ta, tb, tc, kp, grid, s)
              : dispatch_tile<false, __half, GRAD>(cfg, ta, tb, tc, kp, grid, s);
}

bool tma_legal(const void* p, int64_t ld, int elem) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * elem) % 16 == 0;
}

}  // namespace

int encode_matrix(CUtensorMap* map, bool bf16, const void* p, int64_t rows, int64_t cols, int64_t ld,
                  uint32_t box_cols, uint32_t box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld) * 2, static_cast<uint64_t>(rows) * ld * 2};
  const uint32_t box[3] = {box_cols, box_rows, 1};
  return encode_tmap(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p, dims,
                     strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int fill_tc_params(TcParams* kp, int64_t m, int64_t n, int64_t tiles_n, int64_t k_blocks, int64_t items,
                   const TcConfig& cfg, bool bf16, int* grid) {
  std::memset(kp, 0, sizeof(*kp));
  kp->m = static_cast<int32_t>(m);
  kp->n = static_cast<int32_t>(n);
  kp->num_k_blocks = static_cast<int32_t>(k_blocks);
  const int64_t tile_rows = tile_rows_of(cfg);
  kp->num_m_blocks = static_cast<int32_t>((m + tile_rows - 1) / tile_rows);
  kp->num_n_blocks = static_cast<int32_t>(tiles_n);
  kp->batch = static_cast<int32_t>(items);
  kp->num_tiles = static_cast<int64_t>(kp->num_m_blocks) * tiles_n * items;
  const L2Plan l2 = l2_plan();
  kp->group_m = group_tiles(l2, static_cast<int>(tile_rows), kp->num_m_blocks);
  kp->l2_policy_a = l2.policy_a;
  kp->l2_policy_b = l2.policy_b;
  kp->ab_bf16 = bf16 ? 1 : 0;
  kp->alpha = 1.f;
  kp->status = status_word();
  kp->timeout_ns = wait_timeout_ns();
  kp->clock_probe = clock_probe();
  kp->handover_kb = tuning().t.handover_kb;
  if (kp->status == nullptr) return CHOREO_ERR_CUDA;
  const int sms = current_sm_count();
  *grid = cfg.pair ? 2 * static_cast<int>(std::min<int64_t>(kp->num_tiles, sms / 2))
                   : static_cast<int>(std::min<int64_t>(kp->num_tiles, sms));
  return CHOREO_OK;
}

TcConfig select_gate_config(int64_t m, int64_t n, int64_t k) {
  // A tile of BN accumulator columns covers BN/2 columns of H: the GEMM cost
  // model for M x 2N x K, among the shapes the gate kernels are built for. The
  // 512 x 256 pair tile is not: it took 204 us against the 256 x 256 tile's 170 at
  // 4096 x 4096 x 4096, 137 against 114 at 1024 x 4096 x 10240, and on a loop of
  // 8192 x 4096 x 10240 under the power cap 1120 against 1095.
  return plan_tiles(m, 2 * n, (k + kBK - 1) / kBK, 1, current_sm_count(), false, 2, kTilePair256 | kTileSingle128).cfg;
}

namespace {
constexpr int kSkinnyCols = 64;  // columns of H in a skinny tile

bool use_skinny(int64_t m, bool grad) { return m <= kSkinnyRows && !grad; }

int launch_gate_skinny(const GateProblem& p, cudaStream_t stream) {
  CUtensorMap tx;
  TwoMaps tw;
  int rc = encode_matrix(&tx, p.bf16, p.x, p.m, p.k, p.ldx, 64, static_cast<uint32_t>(skinny_tokens(p.m)));
  if (rc) return rc;
  for (int i = 0; i < 2; ++i) {
    const void* w = i == 0 ? p.w_gate : p.w_up;
    rc = p.w_mn ? encode_matrix(&tw.m[i], p.bf16, w, p.k, p.n, p.ldw, 64, 64)
                : encode_matrix(&tw.m[i], p.bf16, w, p.n, p.k, p.ldw, 64, 64);
    if (rc) return rc;
  }
  SkinnyParams kp;
  std::memset(&kp, 0, sizeof(kp));
  kp.m = static_cast<int32_t>(p.m);
  kp.n = static_cast<int32_t>(p.n);
  kp.num_k_blocks = static_cast<int32_t>((p.k + kBK - 1) / kBK);
  const int64_t tiles = (p.n + kSkinnyCols - 1) / kSkinnyCols;
  kp.split = skinny_split(tiles, kp.num_k_blocks, current_sm_count());
  kp.ab_bf16 = p.bf16 ? 1 : 0;
  kp.act = p.act;
  kp.c = p.h;
  kp.ldc = p.ldh;
  kp.out1 = p.out1;
  kp.out2 = p.out2;
  kp.ld12 = p.ld12;
  kp.status = status_word();
  kp.timeout_ns = wait_timeout_ns();
  if (kp.status == nullptr) return CHOREO_ERR_CUDA;
  return p.w_mn ? launch_skinny<kGateCols>(tw, tx, kp, tiles, stream)
                : launch_skinny<kGateRows>(tw, tx, kp, tiles, stream);
}
}  // namespace

int launch_gate_tiles(const GateProblem& p, cudaStream_t stream) {
  if (use_skinny(p.m, p.dh != nullptr)) return launch_gate_skinny(p, stream);
  const TcConfig cfg = select_gate_config(p.m, p.n, p.k);
  CUtensorMap ta;
  TwoMaps tb;
  GateMaps tc;
  std::memset(&tc, 0, sizeof(tc));
  int rc = encode_matrix(&ta, p.bf16, p.x, p.m, p.k, p.ldx, 64, 128);
  if (rc) return rc;
  const uint32_t half = cfg.pair ? 128u : 64u;  // rows of one weight in the tile
  for (int i = 0; i < 2; ++i) {
    const void* w = i == 0 ? p.w_gate : p.w_up;
    rc = p.w_mn ? encode_matrix(&tb.m[i], p.bf16, w, p.k, p.n, p.ldw, 64, 64)
                : encode_matrix(&tb.m[i], p.bf16, w, p.n, p.k, p.ldw, 64, half);
    if (rc) return rc;
  }
  GateParams kp;
  std::memset(&kp, 0, sizeof(kp));
  int grid = 0;
  const int64_t hcols = cfg.bn / 2;
  rc = fill_tc_params(&kp, p.m, p.n, (p.n + hcols - 1) / hcols, (p.k + kBK - 1) / kBK, 1, cfg, p.bf16, &grid);
  if (rc) return rc;
  kp.act = p.act;
  kp.c = p.h;
  kp.ldc = p.ldh;
  if (p.h != nullptr && tma_legal(p.h, p.ldh, 2)) {
    kp.c_vec_ok = kp.c_tma = 1;
    if ((rc = encode_matrix(&tc.m[0], p.bf16, p.h, p.m, p.n, p.ldh, 64, 32))) return rc;
  }
  kp.out1 = p.out1;
  kp.out2 = p.out2;
  kp.ld12 = p.ld12;
  if (p.out1 != nullptr && tma_legal(p.out1, p.ld12, 2) && tma_legal(p.out2, p.ld12, 2)) {
    kp.vec12 = kp.tma12 = 1;
    if ((rc = encode_matrix(&tc.m[1], p.bf16, p.out1, p.m, p.n, p.ld12, 64, 32))) return rc;
    if ((rc = encode_matrix(&tc.m[2], p.bf16, p.out2, p.m, p.n, p.ld12, 64, 32))) return rc;
  }
  kp.dh = p.dh;
  kp.ld_dh = p.ld_dh;
  kp.dh_vec = p.dh != nullptr && tma_legal(p.dh, p.ld_dh, 2) ? 1 : 0;
  return p.dh == nullptr ? dispatch<false>(cfg, p.w_mn, p.bf16, ta, tb, tc, kp, grid, stream)
                         : dispatch<true>(cfg, p.w_mn, p.bf16, ta, tb, tc, kp, grid, stream);
}

void plan_ffn_operands(FfnOperands* o, const void* x, int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw,
                       bool trans_w, int64_t m, int64_t n, int64_t k) {
  o->x = plan_operand(x, ldx, 0, 1, m, k);
  const int64_t outer = trans_w ? n : k, inner = trans_w ? k : n;
  // One leading dimension serves both weights, so they are repacked together.
  const void* odd = tma_legal(w_gate, ldw, 2) ? w_up : w_gate;
  o->w = plan_operand(odd, ldw, 0, 1, outer, inner);
  o->x.offset = 0;
  o->w.offset = o->x.bytes;
  o->bytes = o->x.bytes + 2 * o->w.bytes;
}

int repack_ffn_operands(const FfnOperands& o, char* ws, const void** x, int64_t* ldx, const void** w_gate,
                        const void** w_up, int64_t* ldw, cudaStream_t s) {
  if (o.x.repack) {
    void* dst = ws + o.x.offset;
    if (int rc = launch_repack16(*x, *ldx, 0, dst, o.x.ld_pad, 0, o.x.outer, o.x.inner, 1, s)) return rc;
    *x = dst;
    *ldx = o.x.ld_pad;
  }
  if (o.w.repack) {
    const void** w[2] = {w_gate, w_up};
    for (int i = 0; i < 2; ++i) {
      void* dst = ws + o.w.offset + i * o.w.bytes;
      if (int rc = launch_repack16(*w[i], *ldw, 0, dst, o.w.ld_pad, 0, o.w.outer, o.w.inner, 1, s)) return rc;
      *w[i] = dst;
    }
    *ldw = o.w.ld_pad;
  }
  return CHOREO_OK;
}

int check_ffn_common(const char* what, int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t act, const void* x,
                     int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw, int32_t trans_w) {
  if (m <= 0 || n <= 0 || k <= 0)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: Invalid dimensions: M=%lld, N=%lld, K=%lld", what, (long long)m,
                (long long)n, (long long)k);
  // 2 N accumulator columns and tile coordinates are 32-bit
  if (m > INT32_MAX / 2 || n > INT32_MAX / 4 || k > INT32_MAX / 2)
    return fail(CHOREO_ERR_UNSUPPORTED, "%s: M and K above 2^30-1 or N above 2^29-1 are not supported", what);
  if (!is_tc_type(dtype)) return fail(CHOREO_ERR_UNSUPPORTED, "%s: dtype %d is not f16 or bf16", what, dtype);
  if (act < CHOREO_ACT_SILU || act > CHOREO_ACT_RELU)
    return fail(CHOREO_ERR_UNSUPPORTED, "%s: unknown activation %d", what, act);
  if (x == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "%s: X has null data pointer", what);
  if (w_gate == nullptr || w_up == nullptr)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: a weight has null data pointer", what);
  if (ldx < k) return fail(CHOREO_ERR_INVALID_ARG, "%s: ldx=%lld smaller than K=%lld", what, (long long)ldx, (long long)k);
  const int64_t inner = trans_w ? k : n;
  if (ldw < inner)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: ldw=%lld smaller than %lld", what, (long long)ldw, (long long)inner);
  return CHOREO_OK;
}

int check_workspace(const char* what, const void* workspace, size_t have, int64_t need) {
  if (need == 0) return CHOREO_OK;
  if (workspace == nullptr || have < static_cast<size_t>(need))
    return fail(CHOREO_ERR_WORKSPACE, "%s: needs a workspace of %lld bytes, got %zu", what, (long long)need,
                workspace ? have : size_t{0});
  if (int rc = check_device_ptr(workspace, what)) return rc;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return fail(CHOREO_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", what);
  return CHOREO_OK;
}

namespace {

int validate_ffn(const choreo_ffn_desc* d) {
  if (d == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "gated FFN: null descriptor");
  int rc = check_ffn_common("gated FFN", d->m, d->n, d->k, d->dtype, d->act, d->x, d->ldx, d->w_gate, d->w_up, d->ldw,
                            d->trans_w);
  if (rc) return rc;
  if (d->h == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "gated FFN: H has null data pointer");
  if (d->ldh < d->n)
    return fail(CHOREO_ERR_INVALID_ARG, "gated FFN: ldh=%lld smaller than N=%lld", (long long)d->ldh, (long long)d->n);
  if ((d->gate == nullptr) != (d->up == nullptr))
    return fail(CHOREO_ERR_INVALID_ARG, "gated FFN: gate and up are kept together: one is NULL");
  if (d->gate && d->ld_gu < d->n)
    return fail(CHOREO_ERR_INVALID_ARG, "gated FFN: ld_gu=%lld smaller than N=%lld", (long long)d->ld_gu,
                (long long)d->n);
  if ((rc = check_device_ptr(d->x, "gated FFN X"))) return rc;
  if ((rc = check_device_ptr(d->w_gate, "gated FFN Wg"))) return rc;
  if ((rc = check_device_ptr(d->w_up, "gated FFN Wu"))) return rc;
  if ((rc = check_device_ptr(d->h, "gated FFN H"))) return rc;
  if (d->gate && ((rc = check_device_ptr(d->gate, "gated FFN gate")) || (rc = check_device_ptr(d->up, "gated FFN up"))))
    return rc;
  return CHOREO_OK;
}

}  // namespace
}  // namespace choreo_impl

using namespace choreo_impl;

extern "C" {

int choreo_gated_ffn_query(const choreo_ffn_desc* d, choreo_launch_config* out) {
  int rc = validate_ffn(d);
  if (rc) return rc;
  if (out == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "gated FFN query: null output");
  std::memset(out, 0, sizeof(*out));
  const int sms = current_sm_count();
  out->kernel = 4;
  out->grid_y = out->grid_z = 1;
  out->tile_k = kBK;
  out->split_k = 1;
  FfnOperands o;
  plan_ffn_operands(&o, d->x, d->ldx, d->w_gate, d->w_up, d->ldw, d->trans_w != 0, d->m, d->n, d->k);
  out->workspace_bytes = out->workspace_min_bytes = o.bytes;
  if (use_skinny(d->m, false)) {
    const int nt = skinny_tokens(d->m);
    out->tile_m = nt;
    out->tile_n = kSkinnyCols;
    out->tiles = (d->n + kSkinnyCols - 1) / kSkinnyCols;
    out->split_k = skinny_split(out->tiles, (d->k + kBK - 1) / kBK, sms);
    out->cluster_m = static_cast<int32_t>(out->split_k);
    out->tiles *= out->split_k;
    out->grid_x = static_cast<int32_t>(out->tiles);
    out->block_x = kSkinnyThreads;
    skinny_shape(nt, true, out);
    return ok();
  }
  const TcConfig c = select_gate_config(d->m, d->n, d->k);
  out->tile_m = tile_rows_of(c);
  out->tile_n = c.bn / 2;
  out->stages = c.stages;
  out->cluster_m = c.pair ? 2 : 1;
  out->tiles = ((d->m + out->tile_m - 1) / out->tile_m) * ((d->n + out->tile_n - 1) / out->tile_n);
  out->grid_x = static_cast<int32_t>(c.pair ? 2 * std::min<int64_t>(out->tiles, sms / 2)
                                            : std::min<int64_t>(out->tiles, sms));
  out->block_x = kTcThreads;
  out->smem_bytes = c.smem;
  out->tmem_cols = 2 * c.bn;
  return ok();
}

int choreo_gated_ffn(const choreo_ffn_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = validate_ffn(d);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FfnOperands o;
  plan_ffn_operands(&o, d->x, d->ldx, d->w_gate, d->w_up, d->ldw, d->trans_w != 0, d->m, d->n, d->k);
  if ((rc = check_workspace("gated FFN (an operand is not 16-byte aligned and is repacked)", workspace,
                            workspace_bytes, o.bytes)))
    return rc;
  GateProblem p{};
  p.m = d->m;
  p.n = d->n;
  p.k = d->k;
  p.bf16 = d->dtype == CHOREO_DTYPE_BF16;
  p.act = d->act;
  p.x = d->x;
  p.ldx = d->ldx;
  p.w_gate = d->w_gate;
  p.w_up = d->w_up;
  p.ldw = d->ldw;
  p.w_mn = d->trans_w == 0;
  if ((rc = repack_ffn_operands(o, static_cast<char*>(workspace), &p.x, &p.ldx, &p.w_gate, &p.w_up, &p.ldw, s)))
    return rc;
  p.h = d->h;
  p.ldh = d->ldh;
  p.out1 = d->gate;
  p.out2 = d->up;
  p.ld12 = d->ld_gu;
  rc = launch_gate_tiles(p, s);
  return rc ? rc : ok();
}

}  // extern "C"
