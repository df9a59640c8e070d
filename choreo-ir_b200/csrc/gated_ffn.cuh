// gated_ffn.cuh — device code of the gated feed-forward product and its
// backward pass, on the shared tcgen05 mainloops (tc_kernel.cuh).
//
//   H  = act(G) * U,  G = X Wg,  U = X Wu
//   dG = dH * U * act'(G),  dU = dH * act(G)
//   dX = dG Wg^T + dU Wu^T,  dWg = X^T dG,  dWu = X^T dU
//
// Two loaders feed the mainloops:
//   GateLoader    B tile = the same BN/2 columns of Wg and of Wu, so a tile's
//                 accumulator holds G in its first BN/2 columns and U in the
//                 others and the product needs no second kernel and no memory
//                 for G and U. A CTA pair's B tile is split by N anyway: the
//                 leader stages Wg's columns and its peer Wu's.
//   SelectLoader  two operand pairs chosen by the k-block (dX: one fp32 sum
//                 over 2 N, no second pass over dX) or by the batch item
//                 (dWg and dWu: one launch, so one part-empty last wave).
//
// Bound by the tensor cores (and, on long calls, the 1 kW cap): 8192 x 4096 x
// 10240 bf16 forward 1164k cycles, with G and U kept 1218k, the plain product
// of the same size 1256k (1204k in the same tiles), the MMAs alone 1133k. The
// forward call takes 1.06-1.10 ms back to back, the backward pass with G and U
// computed again 3.16-3.27 ms.
#pragma once
#include "../../include/choreo_b200.h"
#include "tc_kernel.cuh"

namespace choreo_sm100 {

// ------------------------------------------------------------------ activation
// Value and slope of the gate activation. exp through __expf (2 ulp near 0,
// relative error ~ |g| 2^-24 beyond): far below the 16-bit outputs' rounding.

// The normal distribution function, through erfc(x) = t exp(P(t) - x^2),
// t = 1 / (1 + x / 2): a Chebyshev fit of degree 9 of the logarithm (the form
// of Press et al., Numerical Recipes, "Error Function"), fitted in 64 bits to
// 1.0e-7. No branch and no cancellation in the lower tail: relative error below
// 2e-6 for g > -4 and 2e-5 for g > -12 in fp32, against 2^-12 (fp16) of the
// outputs' rounding.
__device__ __forceinline__ float normal_cdf(float g) {
  const float a = fabsf(g) * 0.7071067811865476f;
  const float t = __fdividef(1.f, fmaf(0.5f, a, 1.f));
  float q = 0.1708727777f;
  q = fmaf(q, t, -0.8221522570f);
  q = fmaf(q, t, 1.488515854f);
  q = fmaf(q, t, -1.135203958f);
  q = fmaf(q, t, 0.2788680792f);
  q = fmaf(q, t, -0.1862880588f);
  q = fmaf(q, t, 0.09678418934f);
  q = fmaf(q, t, 0.3740919530f);
  q = fmaf(q, t, 1.000023723f);
  q = fmaf(q, t, -1.265512228f);
  const float half_erfc = 0.5f * t * __expf(fmaf(-a, a, q));
  return g < 0.f ? half_erfc : 1.f - half_erfc;
}

template <int ACT>
__device__ __forceinline__ float act_value(float g) {
  if constexpr (ACT == CHOREO_ACT_SILU) return __fdividef(g, 1.f + __expf(-g));
  if constexpr (ACT == CHOREO_ACT_GELU) return g * normal_cdf(g);
  if constexpr (ACT == CHOREO_ACT_GELU_TANH) {
    // (1 + tanh z) / 2 = 1 / (1 + exp(-2 z))
    const float z2 = 1.5957691216057308f * g * fmaf(0.044715f * g, g, 1.f);
    return __fdividef(g, 1.f + __expf(-z2));
  }
  return g < 0.f ? 0.f : g;  // NaN passes
}
template <int ACT>
__device__ __forceinline__ void act_value_slope(float g, float& v, float& dv) {
  if constexpr (ACT == CHOREO_ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    v = g * s;
    dv = fmaf(v, 1.f - s, s);
  } else if constexpr (ACT == CHOREO_ACT_GELU) {
    const float phi = normal_cdf(g);
    v = g * phi;
    dv = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), phi);
  } else if constexpr (ACT == CHOREO_ACT_GELU_TANH) {
    const float gg = fminf(g * g, 1e30f);  // finite: far out the slope's second term is 0 * gg
    const float s = __fdividef(1.f, 1.f + __expf(-1.5957691216057308f * g * fmaf(0.044715f, gg, 1.f)));
    v = g * s;
    dv = fmaf(v * (1.f - s), 1.5957691216057308f * fmaf(0.134145f, gg, 1.f), s);
  } else {
    v = g < 0.f ? 0.f : g;
    dv = g > 0.f ? 1.f : 0.f;
  }
}

// ------------------------------------------------------------------ loaders
// A = X, K-major (X is M x K). B = Wg and Wu, stored K x N (W_MN) or N x K.
// BNL = B columns this CTA stages: all of the tile's BN for a single CTA
// (half of them Wg's), the leader's Wg or the peer's Wu half for a pair.
template <bool W_MN, int BNL, bool PAIR>
struct GateLoader {
  using MapA = CUtensorMap;
  using MapB = TwoMaps;
  static constexpr bool kAMn = false;
  static constexpr bool kBMn = W_MN;
  static constexpr int kHalf = PAIR ? BNL : BNL / 2;  // columns of one weight in the tile
  static_assert(!W_MN || kHalf % 64 == 0, "an MN-major chunk holds 64 columns");

  __device__ __forceinline__ static void issue_w(const CUtensorMap* w, int h0, int kb, uint32_t dst, uint32_t bar,
                                                 uint64_t pol) {
    const int k0 = kb * kBK;
    if constexpr (!W_MN) {
      load3<PAIR>(dst, w, bar, k0, h0, 0, pol);
    } else {
#pragma unroll
      for (int j = 0; j < kHalf / 64; ++j) load3<PAIR>(dst + j * 8192, w, bar, h0 + j * 64, k0, 0, pol);
    }
  }
  __device__ __forceinline__ static void issue_b(const TwoMaps* tb, int n0, int kb, uint32_t dst_b, uint32_t bar,
                                                 uint64_t pol_b) {
    if constexpr (PAIR) {
      // n0 = tile * 2 * BNL + rank * BNL
      issue_w(&tb->m[(n0 / BNL) & 1], n0 / (2 * BNL) * BNL, kb, dst_b, bar, pol_b);
    } else {
      issue_w(&tb->m[0], n0 / 2, kb, dst_b, bar, pol_b);
      issue_w(&tb->m[1], n0 / 2, kb, dst_b + kHalf * kBK * 2, bar, pol_b);
    }
  }
  __device__ __forceinline__ static void issue(const CUtensorMap* ta, const TwoMaps* tb, const TcParams&, int, int m0,
                                               int n0, int kb, uint32_t dst_a, uint32_t dst_b, uint32_t bar,
                                               uint64_t pol_a, uint64_t pol_b) {
    load3<PAIR>(dst_a, ta, bar, kb * kBK, m0, 0, pol_a);
    issue_b(tb, n0, kb, dst_b, bar, pol_b);
  }
};

struct SelectParams : TcParams {
  int32_t k_blocks_1;  // by k-block: blocks of the first operand pair (the second pair's follow)
  void* c1;            // by batch item: the second output
};

// Two operand pairs; BY_K: the k-blocks of pair 0 and then those of pair 1 in
// one sum, else batch item 0 or 1.
template <bool BY_K, bool A_MN, bool B_MN, int BNL, bool PAIR>
struct SelectLoader {
  using MapA = TwoMaps;
  using MapB = TwoMaps;
  static constexpr bool kAMn = A_MN;
  static constexpr bool kBMn = B_MN;
  // Pair and k origin of k-block kb of batch item (or K split) b.
  __device__ __forceinline__ static int pick(const SelectParams& p, int b, int kb, int& k0) {
    if constexpr (BY_K) {
      const int g = p.split_kb > 0 ? b * p.split_kb + kb : kb;
      const int second = g >= p.k_blocks_1 ? 1 : 0;
      k0 = (g - (second ? p.k_blocks_1 : 0)) * kBK;
      return second;
    } else {
      k0 = kb * kBK;
      return b;
    }
  }
  template <int ROWS, bool MN>
  __device__ __forceinline__ static void issue_side(const CUtensorMap* t, int r0, int k0, uint32_t dst, uint32_t bar,
                                                    uint64_t pol) {
    if constexpr (!MN) {
      load3<PAIR>(dst, t, bar, k0, r0, 0, pol);
    } else {
#pragma unroll
      for (int j = 0; j < ROWS / 64; ++j) load3<PAIR>(dst + j * 8192, t, bar, r0 + j * 64, k0, 0, pol);
    }
  }
  __device__ __forceinline__ static void issue(const TwoMaps* ta, const TwoMaps* tb, const SelectParams& p, int b,
                                               int m0, int n0, int kb, uint32_t dst_a, uint32_t dst_b, uint32_t bar,
                                               uint64_t pol_a, uint64_t pol_b) {
    int k0;
    const int s = pick(p, b, kb, k0);
    issue_side<kBM, A_MN>(&ta->m[s], m0, k0, dst_a, bar, pol_a);
    issue_side<BNL, B_MN>(&tb->m[s], n0, k0, dst_b, bar, pol_b);
  }
  struct WideCursor {
    int b, m0, n0;
  };
  __device__ __forceinline__ static WideCursor wide_cursor(const TcParams&, int b, int m0, int n0) {
    return WideCursor{b, m0, n0};
  }
  __device__ __forceinline__ static void issue_wide(const TwoMaps* ta, const TwoMaps* tb, const SelectParams& p,
                                                    WideCursor& c, int kb, uint32_t dst_a, uint32_t dst_b,
                                                    uint32_t bar, uint64_t pol_a, uint64_t pol_b) {
    int k0;
    const int s = pick(p, c.b, kb, k0);
    issue_side<2 * kBM, A_MN>(&ta->m[s], c.m0, k0, dst_a, bar, pol_a);
    issue_side<BNL, B_MN>(&tb->m[s], c.n0, k0, dst_b, bar, pol_b);
  }
};

// LinearEpi with SelectLoader's parameters; BY_K: one output (batch items are
// K splits), else one output per batch item.
template <typename OutT, bool BY_K>
struct SelectEpi {
  using MapC = TwoMaps;
  using Params = SelectParams;
  template <int BN>
  using Pre = BiasRegs<BN / 2>;
  template <int BN>
  __device__ __forceinline__ static void prefetch(Pre<BN>&, int, int, const SelectParams&, int) {}
  template <int BN, typename Release>
  __device__ __forceinline__ static void run(uint32_t tacc, int nb, int col_half, int row0, int b,
                                             const SelectParams& p, const TwoMaps* tma_c, uint32_t stage_buf, int lane,
                                             const Pre<BN>& br, Release&& release) {
    TcParams q = p;
    const CUtensorMap* map = &tma_c->m[0];
    if constexpr (!BY_K) {
      if (b != 0) {
        q.c = p.c1;
        map = &tma_c->m[1];
      }
      b = 0;
    }
    q.bias = nullptr;
    epilogue_warp<BN / 2, OutT>(tacc + col_half * (BN / 2), nb * BN + col_half * (BN / 2), row0, b, q, map, stage_buf,
                                lane, br, release);
  }
};

// ------------------------------------------------------------------ epilogues of the gate tiles
struct GateMaps {
  CUtensorMap m[3];  // h, then gate and up (forward) or dG and dU (backward)
};
__device__ __forceinline__ void tma_prefetch_desc(const GateMaps* maps) { tma_prefetch_desc(&maps->m[0]); }

struct GateParams : TcParams {
  int32_t act;
  // forward: where G and U are kept (null: nowhere); backward: dG and dU
  void* out1;
  void* out2;
  int64_t ld12;
  int32_t tma12, vec12;
  // backward
  const void* dh;
  int64_t ld_dh;
  int32_t dh_vec;
};

// One warp's kCols columns of one 16-bit output, packed in pairs: through the
// staging buffer and a bulk tensor store when the columns fill its 128-byte
// rows and the output is TMA-addressable, else 16-byte vectors or elements. (A
// bulk tensor store clips columns in whole 16 bytes, so it is not used where
// the matrix ends inside 16 bytes.)
template <int kCols, typename OutT>
__device__ __forceinline__ void gate_store(const uint32_t (&q)[kCols / 32][16], const CUtensorMap* map, bool tma,
                                           bool vec, void* base, int64_t ld, int h0, int row0, int m, int n,
                                           uint32_t stage_buf, int lane) {
  if constexpr (kCols == 64) {
    if (tma && (h0 + 64 <= n || n % 8 == 0)) {
      if (lane == 0) bulk_wait_read_all();  // the warp's previous store has read the buffer
      __syncwarp();
      const uint32_t row_addr = stage_buf + static_cast<uint32_t>(lane) * 128u;
      stage_packed_32(q[0], row_addr, lane, 0);
      stage_packed_32(q[1], row_addr, lane, 4);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(map, stage_buf, h0, row0, 0);
        bulk_commit_group();
      }
      return;
    }
  }
  const int row = row0 + lane;
  if (row >= m) return;
  uint16_t* dst = static_cast<uint16_t*>(base) + static_cast<int64_t>(row) * ld + h0;
#pragma unroll
  for (int c = 0; c < kCols / 32; ++c) {
    if (vec && h0 + c * 32 + 32 <= n) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        reinterpret_cast<uint4*>(dst + c * 32)[j] =
            make_uint4(q[c][4 * j], q[c][4 * j + 1], q[c][4 * j + 2], q[c][4 * j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (h0 + c * 32 + j < n) dst[c * 32 + j] = static_cast<uint16_t>(q[c][j / 2] >> (16 * (j & 1)));
    }
  }
}

template <int kChunks, typename OutT>
__device__ __forceinline__ void gate_pack(const uint32_t (&r)[kChunks][32], uint32_t (&q)[kChunks][16]) {
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      q[c][j] = pack2(__uint_as_float(r[c][2 * j]), __uint_as_float(r[c][2 * j + 1]), static_cast<OutT*>(nullptr));
}

// Forward: h = act(G) * U from the fp32 accumulators, and G and U themselves
// when they are kept. Backward (GRAD): dG and dU from G, U and dH, and h when
// it is wanted again. A warp takes the same BN/4 columns of G and of U, read
// from TMEM at once and handed back before the arithmetic. In the 256-column
// tile these are 128 registers of a thread's 168 and the packed columns 32 more:
// the forward form spills 244 bytes a thread (432 read back), GRAD, which takes
// 32 columns at a time, 12 (16). What that costs is not measured; with it the
// large product takes 1.03 of its MMAs' cycles.
template <typename OutT, bool GRAD>
struct GateEpi {
  using MapC = GateMaps;
  using Params = GateParams;
  template <int BN>
  struct Pre {};
  template <int BN>
  __device__ __forceinline__ static void prefetch(Pre<BN>&, int, int, const GateParams&, int) {}

  template <int ACT, int kChunks>
  __device__ __forceinline__ static void product(const uint32_t (&g)[kChunks][32], const uint32_t (&u)[kChunks][32],
                                                 uint32_t (&q)[kChunks][16]) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        q[c][j] = pack2(act_value<ACT>(__uint_as_float(g[c][2 * j])) * __uint_as_float(u[c][2 * j]),
                        act_value<ACT>(__uint_as_float(g[c][2 * j + 1])) * __uint_as_float(u[c][2 * j + 1]),
                        static_cast<OutT*>(nullptr));
  }

  // 32 columns of dG, dU and h, packed, from G, U and dH (packed in d).
  template <int ACT>
  __device__ __forceinline__ static void gradient(const uint32_t (&g)[32], const uint32_t (&u)[32],
                                                  const uint32_t (&d)[16], uint32_t (&gq)[16], uint32_t (&uq)[16],
                                                  uint32_t (&hq)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float dh[2], dg[2], du[2], h[2];
      unpack2(d[j], dh[0], dh[1], static_cast<OutT*>(nullptr));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float uu = __uint_as_float(u[2 * j + e]);
        float v, dv;
        act_value_slope<ACT>(__uint_as_float(g[2 * j + e]), v, dv);
        h[e] = v * uu;
        dg[e] = dh[e] * uu * dv;
        du[e] = dh[e] * v;
      }
      gq[j] = pack2(dg[0], dg[1], static_cast<OutT*>(nullptr));
      uq[j] = pack2(du[0], du[1], static_cast<OutT*>(nullptr));
      hq[j] = pack2(h[0], h[1], static_cast<OutT*>(nullptr));
    }
  }

  template <int BN, typename Release>
  __device__ __forceinline__ static void run(uint32_t tacc, int nb, int col_half, int row0, int, const GateParams& p,
                                             const GateMaps* maps, uint32_t stage_buf, int lane, const Pre<BN>&,
                                             Release&& release) {
    constexpr int kCols = BN / 4;
    constexpr int kChunks = kCols / 32;
    const int h0 = nb * (BN / 2) + col_half * kCols;
    if (row0 >= p.m || h0 >= p.n) {
      release();
      return;
    }
    uint32_t g[kChunks][32], u[kChunks][32], q[kChunks][16];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      tmem_ld_32x32b_x32(tacc + col_half * kCols + c * 32, g[c]);
      tmem_ld_32x32b_x32(tacc + BN / 2 + col_half * kCols + c * 32, u[c]);
    }
    tmem_wait_ld();
    release();
    if constexpr (!GRAD) {
      if (p.out1 != nullptr) {
        gate_pack<kChunks, OutT>(g, q);
        gate_store<kCols, OutT>(q, &maps->m[1], p.tma12 != 0, p.vec12 != 0, p.out1, p.ld12, h0, row0, p.m, p.n,
                                stage_buf, lane);
        gate_pack<kChunks, OutT>(u, q);
        gate_store<kCols, OutT>(q, &maps->m[2], p.tma12 != 0, p.vec12 != 0, p.out2, p.ld12, h0, row0, p.m, p.n,
                                stage_buf, lane);
      }
      switch (p.act) {
        case CHOREO_ACT_SILU: product<CHOREO_ACT_SILU>(g, u, q); break;
        case CHOREO_ACT_GELU: product<CHOREO_ACT_GELU>(g, u, q); break;
        case CHOREO_ACT_GELU_TANH: product<CHOREO_ACT_GELU_TANH>(g, u, q); break;
        default: product<CHOREO_ACT_RELU>(g, u, q); break;
      }
      gate_store<kCols, OutT>(q, &maps->m[0], p.c_tma != 0, p.c_vec_ok != 0, p.c, p.ldc, h0, row0, p.m, p.n, stage_buf,
                              lane);
    } else {
      uint32_t gq[kChunks][16], uq[kChunks][16];
      const int row = row0 + lane;
      const uint16_t* src =
          static_cast<const uint16_t*>(p.dh) + static_cast<int64_t>(row < p.m ? row : row0) * p.ld_dh + h0;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        uint32_t d[16];
        if (p.dh_vec && h0 + c * 32 + 32 <= p.n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 v = reinterpret_cast<const uint4*>(src + c * 32)[j];
            d[4 * j] = v.x;
            d[4 * j + 1] = v.y;
            d[4 * j + 2] = v.z;
            d[4 * j + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint32_t lo = h0 + c * 32 + 2 * j < p.n ? src[c * 32 + 2 * j] : 0u;
            const uint32_t hi = h0 + c * 32 + 2 * j + 1 < p.n ? src[c * 32 + 2 * j + 1] : 0u;
            d[j] = lo | (hi << 16);
          }
        }
        switch (p.act) {
          case CHOREO_ACT_SILU: gradient<CHOREO_ACT_SILU>(g[c], u[c], d, gq[c], uq[c], q[c]); break;
          case CHOREO_ACT_GELU: gradient<CHOREO_ACT_GELU>(g[c], u[c], d, gq[c], uq[c], q[c]); break;
          case CHOREO_ACT_GELU_TANH: gradient<CHOREO_ACT_GELU_TANH>(g[c], u[c], d, gq[c], uq[c], q[c]); break;
          default: gradient<CHOREO_ACT_RELU>(g[c], u[c], d, gq[c], uq[c], q[c]); break;
        }
      }
      if (p.c != nullptr)
        gate_store<kCols, OutT>(q, &maps->m[0], p.c_tma != 0, p.c_vec_ok != 0, p.c, p.ldc, h0, row0, p.m, p.n,
                                stage_buf, lane);
      gate_store<kCols, OutT>(gq, &maps->m[1], p.tma12 != 0, p.vec12 != 0, p.out1, p.ld12, h0, row0, p.m, p.n,
                              stage_buf, lane);
      gate_store<kCols, OutT>(uq, &maps->m[2], p.tma12 != 0, p.vec12 != 0, p.out2, p.ld12, h0, row0, p.m, p.n,
                              stage_buf, lane);
    }
  }
};

}  // namespace choreo_sm100
