// skinny.cuh — products with few rows of X (tokens of a decode batch): bound by
// reading the weights once, so the kernel is built around their stream.
//
// The weights are the MMA's 128-row operand and the tokens its NT columns
// (NT = 16, 32, 64, 96 or 128), so little tensor work goes to absent rows. One CTA streams
// 128 weight rows x 128 bytes per k-block; `split` CTAs of a cluster each take
// a range of the k-blocks of one tile, so that a few tiles still keep every SM
// loading, and add their partial sums through distributed shared memory in a
// fixed order. Two CTAs share an SM (at most 113 KB of shared memory each), so
// one streams while the other starts or finishes.
//
//   warp 0      TMA producer
//   warp 1      MMA issuer
//   warps 2..5  read the accumulators; thread = weight row (warp % 4 = TMEM
//               lane quarter)
// All six warps reduce the partial sums and write the output.
//
// kGate: rows 0..63 of the tile are 64 columns of Wg, rows 64..127 the same of
// Wu; the accumulator sums over the CTA's whole range and the output is
// act(G) * U. kBlock: e4m3 weights and tokens with scales; as in the large
// tiles every k-block is one scale block with an accumulator of its own, added
// to fp32 sums in registers.
//
// Measured: 1 x 4096 x 10240 bf16 gate, weights N x K, 29.6 us = 0.86 of the
// copy bandwidth (K x N: 27.2 us = 0.94); 77 x 2056 x 5461 f16 gate 16.1 us for
// 7 us of bytes, 16 x 10240 x 4096 in 8 bits 13.4 us for 6.5, the rest the start
// of ten k-blocks a CTA and the reduction over the cluster. kBlock with 128
// tokens holds 128 sums a thread and spills 72 bytes.
#pragma once
#include <algorithm>

#include "gated_ffn.cuh"
#include "internal.h"

namespace choreo_sm100 {

enum SkinnyKind { kGateRows = 0, kGateCols = 1, kBlock = 2 };  // weights N x K, K x N; 8-bit

constexpr int kSkinnyThreads = 192;

struct SkinnyParams : TcParams {
  int32_t split;
  // kGate*
  int32_t act;
  void* out1;
  void* out2;
  int64_t ld12;
  // kBlock
  int32_t dtype_c;
  int32_t block_b;
  const float* sa;
  int64_t sa_row, sa_blk;
  const float* sb;
  int64_t sb_row, sb_blk;
  const void* d;
  int64_t ldd;
};

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// Sums of the SPLIT CTAs' partial values at shared address `off` (and, for
// gate tiles, of U's, 64 rows on), in rank order.
template <int SPLIT, bool GATE>
__device__ __forceinline__ void add_partials(uint32_t off, float (&v)[4], float (&u)[4]) {
  float4 a[SPLIT], b[SPLIT];
#pragma unroll
  for (int s = 0; s < SPLIT; ++s) {
    const uint32_t at = SPLIT > 1 ? mapa_shared(off, static_cast<uint32_t>(s)) : off;
    a[s] = ld_cluster_v4(at);
    if constexpr (GATE) b[s] = ld_cluster_v4(at + 256u);
  }
#pragma unroll
  for (int s = 0; s < SPLIT; ++s) {
    v[0] += a[s].x, v[1] += a[s].y, v[2] += a[s].z, v[3] += a[s].w;
    if constexpr (GATE) u[0] += b[s].x, u[1] += b[s].y, u[2] += b[s].z, u[3] += b[s].w;
  }
}
__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dt) {
  if (dt == CHOREO_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dt == CHOREO_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int64_t i, int dt, float v) {
  if (dt == CHOREO_DTYPE_F32)
    static_cast<float*>(p)[i] = v;
  else if (dt == CHOREO_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// Up to four neighbouring elements; one 8- or 16-byte store where it is legal.
__device__ __forceinline__ void store_quad(void* p, int64_t i, int dt, const float (&v)[4], int left) {
  if (left >= 4) {
    if (dt == CHOREO_DTYPE_F32) {
      float* q = static_cast<float*>(p) + i;
      if ((reinterpret_cast<uintptr_t>(q) & 15u) == 0) {
        *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
        return;
      }
    } else {
      uint16_t* q = static_cast<uint16_t*>(p) + i;
      if ((reinterpret_cast<uintptr_t>(q) & 7u) == 0) {
        *reinterpret_cast<uint2*>(q) =
            dt == CHOREO_DTYPE_BF16
                ? make_uint2(pack2(v[0], v[1], static_cast<__nv_bfloat16*>(nullptr)),
                             pack2(v[2], v[3], static_cast<__nv_bfloat16*>(nullptr)))
                : make_uint2(pack2(v[0], v[1], static_cast<__half*>(nullptr)),
                             pack2(v[2], v[3], static_cast<__half*>(nullptr)));
        return;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) store_from_f32(p, i + e, dt, v[e]);
}
template <int ACT>
__device__ __forceinline__ void act_quad_of(float (&g)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) g[e] = act_value<ACT>(g[e]);
}
__device__ __forceinline__ void act_quad(int act, float (&g)[4]) {
  switch (act) {
    case CHOREO_ACT_SILU: act_quad_of<CHOREO_ACT_SILU>(g); break;
    case CHOREO_ACT_GELU: act_quad_of<CHOREO_ACT_GELU>(g); break;
    case CHOREO_ACT_GELU_TANH: act_quad_of<CHOREO_ACT_GELU_TANH>(g); break;
    default: act_quad_of<CHOREO_ACT_RELU>(g);
  }
}

constexpr uint32_t skinny_tmem_cols(int used) { return used <= 32 ? 32 : (used <= 64 ? 64 : (used <= 128 ? 128 : 256)); }

template <int NT>
struct SkinnyShape {
  static constexpr uint32_t kWStage = 128 * 128;  // bytes: 128 rows x 128 bytes of K
  static constexpr uint32_t kXStage = NT * 128;
  static constexpr int kStages = NT <= 16 ? 6 : (NT <= 32 ? 5 : (NT <= 64 ? 4 : 3));
  static constexpr int kBufs = NT <= 64 ? 4 : 2;  // kBlock: accumulators; two CTAs share the SM's 512 columns
  static constexpr uint32_t kRing = kStages * (kWStage + kXStage);
  static constexpr int kSmem = static_cast<int>(kRing) + 1024 + 256;
  static_assert(NT * 128 * 4 <= kRing, "the partial sums reuse the ring");
  // kBlock: the epilogue follows a stage's barrier by its parity. The issuer runs
  // at most kBufs k-blocks ahead of it, so the barrier may not come round sooner.
  static_assert(kStages >= kBufs, "a stage's barrier would complete twice before the epilogue looks");
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
};

template <int STAGES>
struct alignas(8) SkinnyBarriers {
  uint64_t full[STAGES];
  uint64_t empty[STAGES];     // the stage's MMAs are done
  uint64_t tmem_empty[4];     // kBlock: an accumulator has been read
  uint64_t done;              // every MMA of the CTA is done
  uint32_t tmem_base;
  int32_t abort;
};

template <int KIND, int NT>
__global__ void __launch_bounds__(kSkinnyThreads, 2)
    skinny_kernel(const __grid_constant__ TwoMaps tma_w, const __grid_constant__ CUtensorMap tma_x,
                  const SkinnyParams p) {
  using S = SkinnyShape<NT>;
  constexpr int STAGES = S::kStages;
  constexpr bool kGate = KIND != kBlock;
  constexpr int kElemsK = kGate ? 64 : 128;  // elements of K in a k-block (128 bytes)
  constexpr int kBufs = kGate ? 1 : S::kBufs;
  constexpr uint32_t kTmemCols = skinny_tmem_cols(kBufs * NT);
  constexpr int kOutCols = kGate ? 64 : 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint8_t* s_w = smem;
  uint8_t* s_x = smem + STAGES * S::kWStage;
  auto* bars = reinterpret_cast<SkinnyBarriers<STAGES>*>(smem + S::kRing);
  __shared__ alignas(16) float s_scale[kGate ? 1 : 4][kGate ? 1 : NT];  // kBlock: one k-block's token scales, per warp
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int col0 = static_cast<int>(blockIdx.x / split) * kOutCols;  // first output column of the tile
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.num_k_blocks) * rank / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.num_k_blocks) * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&bars->tmem_empty[i]), 4);
    mbar_init(smem_u32(&bars->done), 1);
    bars->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tma_w.m[0]);
    if constexpr (kGate) tma_prefetch_desc(&tma_w.m[1]);
    tma_prefetch_desc(&tma_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  const WaitCtx wctx{p.status, p.timeout_ns, &bars->abort};
  griddep_wait();

  bool ok = true;
  float* part = reinterpret_cast<float*>(smem);  // [token][weight row], once the ring is idle
  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------- producer
      const uint64_t pol_w = l2_policy_evict_normal();
      const uint64_t pol_x = l2_policy_evict_last();  // every CTA reads the tokens again
      uint32_t stage = 0, phase = 0, issued = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&bars->empty[stage]), phase ^ 1, wctx, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&bars->full[stage]);
        mbar_arrive_expect_tx(bar, S::kWStage + S::kXStage);
        const uint32_t dst = smem_u32(s_w + stage * S::kWStage);
        const int k0 = kb * kElemsK;
        if constexpr (KIND == kBlock) {
          tma_load_3d(dst, &tma_w.m[0], bar, k0, col0, 0, pol_w);
        } else if constexpr (KIND == kGateRows) {
          tma_load_3d(dst, &tma_w.m[0], bar, k0, col0, 0, pol_w);
          tma_load_3d(dst + 8192, &tma_w.m[1], bar, k0, col0, 0, pol_w);
        } else {
          tma_load_3d(dst, &tma_w.m[0], bar, col0, k0, 0, pol_w);
          tma_load_3d(dst + 8192, &tma_w.m[1], bar, col0, k0, 0, pol_w);
        }
        tma_load_3d(smem_u32(s_x + stage * S::kXStage), &tma_x, bar, k0, 0, 0, pol_x);
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      griddep_launch_dependents();
      if (!ok) {
        const uint32_t inflight = issued < STAGES ? issued : STAGES;
        uint32_t s = stage, ph = phase;
        for (uint32_t i = 0; i < inflight; ++i) {
          if (s == 0) { s = STAGES - 1; ph ^= 1; } else { --s; }
          mbar_wait(smem_u32(&bars->full[s]), ph, wctx, kStatusTimeoutDrain, false);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    const uint32_t idesc = kGate ? idesc_f16(128, NT, p.ab_bf16 != 0, KIND == kGateCols, false) : idesc_e4m3(128, NT);
    constexpr bool kAMn = KIND == kGateCols;
    const uint64_t desc_w = kAMn ? smem_desc_sw128(smem_u32(s_w), 8192, 1024) : smem_desc_sw128(smem_u32(s_w), 16, 1024);
    const uint64_t desc_x = smem_desc_sw128(smem_u32(s_x), 16, 1024);
    uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 1;
    for (int kb = kb0; kb < kb1; ++kb) {
      bool ready = mbar_wait(smem_u32(&bars->full[stage]), phase, wctx, kStatusTimeoutMma);
      if constexpr (!kGate)
        ready = ready && mbar_wait(smem_u32(&bars->tmem_empty[buf]), buf_phase, wctx, kStatusTimeoutMma);
      if (!__all_sync(0xffffffffu, ready)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t wd = smem_desc_advance(desc_w, stage * S::kWStage);
      const uint64_t xd = smem_desc_advance(desc_x, stage * S::kXStage);
      if (elect_one()) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          const uint64_t a = smem_desc_advance(wd, kAMn ? k * 2048 : k * 32);
          const uint64_t b = smem_desc_advance(xd, k * 32);
          if constexpr (kGate)
            umma_f16(tmem_base, a, b, idesc, (kb != kb0 || k != 0) ? 1u : 0u);
          else
            umma_f8(tmem_base + buf * NT, a, b, idesc, k != 0 ? 1u : 0u);
        }
        umma_commit(smem_u32(&bars->empty[stage]));
      }
      __syncwarp();
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
      if constexpr (!kGate)
        if (++buf == kBufs) { buf = 0; buf_phase ^= 1; }
    }
    if (elect_one()) umma_commit(smem_u32(&bars->done));
    // Also when the loop gave up: no MMA may read the ring or write TMEM later.
    mbar_wait(smem_u32(&bars->done), 0, wctx, kStatusTimeoutDrain, false);
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // weight row of the tile
    const uint32_t tmem_warp = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    if constexpr (kGate) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->done), 0, wctx, kStatusTimeoutEpilogue));
      if (ok) {
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < NT / 16; ++c) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(tmem_warp + c * 16, r);
          tmem_wait_ld(r);
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(c * 16 + j) * 128 + row] = __uint_as_float(r[j]);
        }
      }
    } else {
      const int n = min(col0 + row, p.n - 1);
      const float* sb = p.sb + static_cast<int64_t>(n / p.block_b) * p.sb_row + static_cast<int64_t>(kb0) * p.sb_blk;
      constexpr int kSa = (NT + 31) / 32;  // token scales a lane loads
      const float* sa[kSa];
#pragma unroll
      for (int c = 0; c < kSa; ++c)
        sa[c] = p.sa + static_cast<int64_t>(min(32 * c + lane, p.m - 1)) * p.sa_row + static_cast<int64_t>(kb0) * p.sa_blk;
      float next_b = 0.f, next_a[kSa] = {};
      if (kb0 < kb1) {
        next_b = ldg_early(sb);
#pragma unroll
        for (int c = 0; c < kSa; ++c) next_a[c] = ldg_early(sa[c]);
      }
      float acc[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[j] = 0.f;
      float* warp_scale = s_scale[quarter];
      uint32_t stage = 0, phase = 0, buf = 0;
#pragma unroll 1
      for (int kb = kb0; kb < kb1; ++kb) {
        const float b = next_b;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kSa; ++c)
          if (NT % 32 == 0 || 32 * c + lane < NT) warp_scale[32 * c + lane] = next_a[c];
        __syncwarp();
        if (kb + 1 < kb1) {
          sb += p.sb_blk;
          next_b = ldg_early(sb);
#pragma unroll
          for (int c = 0; c < kSa; ++c) {
            sa[c] += p.sa_blk;
            next_a[c] = ldg_early(sa[c]);
          }
        }
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->empty[stage]), phase, wctx, kStatusTimeoutEpilogue))) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < NT / 16; ++c) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(tmem_warp + buf * NT + c * 16, r);
          tmem_wait_ld(r);
          if (c + 1 == NT / 16) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->tmem_empty[buf]));
          }
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(warp_scale + c * 16 + j);
            acc[c * 16 + j] = fmaf(__uint_as_float(r[j]), s.x * b, acc[c * 16 + j]);
            acc[c * 16 + j + 1] = fmaf(__uint_as_float(r[j + 1]), s.y * b, acc[c * 16 + j + 1]);
            acc[c * 16 + j + 2] = fmaf(__uint_as_float(r[j + 2]), s.z * b, acc[c * 16 + j + 2]);
            acc[c * 16 + j + 3] = fmaf(__uint_as_float(r[j + 3]), s.w * b, acc[c * 16 + j + 3]);
          }
        }
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        if (++buf == kBufs) buf = 0;
      }
      // The ring is idle once the last MMA is done.
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->done), 0, wctx, kStatusTimeoutEpilogue))) ok = false;
      if (ok) {
#pragma unroll
        for (int j = 0; j < NT; ++j) part[j * 128 + row] = acc[j];
      }
    }
  }

  // A CTA that gave up leaves the cluster's outputs unwritten (the status word
  // says so); the barriers below are met all the same.
  const bool cta_ok = __syncthreads_and(ok ? 1 : 0) != 0;
  __shared__ int s_ok;
  if (threadIdx.x == 0) s_ok = cta_ok ? 1 : 0;
  tc_fence_before();
  if (split > 1) cluster_sync(); else __syncthreads();
  bool all_ok = cta_ok;
  if (split > 1) {
    all_ok = true;
    for (int s = 0; s < split; ++s) {
      uint32_t v;
      asm volatile("ld.shared::cluster.u32 %0, [%1];"
                   : "=r"(v)
                   : "r"(mapa_shared(smem_u32(&s_ok), static_cast<uint32_t>(s)))
                   : "memory");
      all_ok = all_ok && v != 0;
    }
  }
  if (all_ok) {
    // CTA `rank` adds up and writes the tokens rank, rank + split, ...; a
    // thread takes four columns of one, all its loads in flight at once.
    const uint32_t part_addr = smem_u32(part);
    constexpr int kQuads = kOutCols / 4;
    const int tokens = (p.m - rank + split - 1) / split;
    for (int i = threadIdx.x; i < tokens * kQuads; i += kSkinnyThreads) {
      const int64_t t = rank + (i / kQuads) * split;
      const int c = i % kQuads * 4;
      const int left = p.n - col0 - c;  // columns of the quad inside the matrix
      if (left <= 0) continue;
      const uint32_t off = part_addr + static_cast<uint32_t>(t * 128 + c) * 4u;
      float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
      switch (split) {
        case 1: add_partials<1, kGate>(off, v, u); break;
        case 2: add_partials<2, kGate>(off, v, u); break;
        case 3: add_partials<3, kGate>(off, v, u); break;
        case 4: add_partials<4, kGate>(off, v, u); break;
        case 5: add_partials<5, kGate>(off, v, u); break;
        case 6: add_partials<6, kGate>(off, v, u); break;
        case 7: add_partials<7, kGate>(off, v, u); break;
        default: add_partials<8, kGate>(off, v, u);
      }
      if constexpr (kGate) {
        const int dt = p.ab_bf16 ? CHOREO_DTYPE_BF16 : CHOREO_DTYPE_F16;
        if (p.out1 != nullptr) {
          store_quad(p.out1, t * p.ld12 + col0 + c, dt, v, left);
          store_quad(p.out2, t * p.ld12 + col0 + c, dt, u, left);
        }
        act_quad(p.act, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= u[e];
        store_quad(p.c, t * p.ldc + col0 + c, dt, v, left);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] *= p.alpha;
          if (e < left) {
            if (p.beta != 0.f) v[e] += p.beta * load_as_f32(p.d, t * p.ldd + col0 + c + e, p.dtype_c);
            if (p.bias != nullptr) v[e] += load_bias(p.bias, p.dtype_bias, col0 + c + e);
          }
          if (p.relu) v[e] = v[e] < 0.f ? 0.f : v[e];  // NaN passes
        }
        store_quad(p.c, t * p.ldc + col0 + c, p.dtype_c, v, left);
      }
    }
  }
  if (split > 1) cluster_sync();  // no CTA leaves while others read its partial sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace choreo_sm100

namespace choreo_impl {

// Rows of X up to which the skinny kernel is used, and its token tile.
constexpr int64_t kSkinnyRows = 128;
inline int skinny_tokens(int64_t m) { return m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : (m <= 96 ? 96 : 128))); }

// CTAs per tile: the most (at most a portable cluster) whose grid is resident at
// once, with at least four k-blocks each. More pieces spread the weights more
// evenly over the SMs and keep more loads in flight; a second wave costs as much
// as the first. An SM holds two CTAs, but a cluster has to lie within one group
// of SMs, which leaves places unused: measured on a B200, clusters of 3 and 4
// still fit at 15/16 of the places, of 5 to 8 at 7/8 (weights in L2, 3 CTAs a
// tile: 92 tiles 15.0 us, 95 tiles 23.3, in 2 18.9; 8 a tile: 32 tiles 7.2, 34
// tiles 11.7). Weights from HBM, fewest against most pieces: 77 x 2056 x 5461
// gate 19.8 us in 1, 16.1 in 3; 16 x 4096 x 4096 19.8 in 1, 15.1 in 4; 16 x
// 10240 x 4096 in 8 bits 15.7 in 4, 13.4 in 8; 1 x 2048 x 5632 gate alike in 1
// and 3 (11.5, 11.1; in L2 10.5, 8.4); the worst for the rule 6.5 in 4, 6.8 in 8
// (1 x 2048 x 2048).
inline int skinny_split(int64_t tiles, int64_t k_blocks, int sms) {
  for (int split = 8; split > 1; --split) {
    const int sixteenths = split > 4 ? 14 : (split > 2 ? 15 : 16);
    if (tiles * split * 16 <= 2 * static_cast<int64_t>(sms) * sixteenths && k_blocks / split >= 4) return split;
  }
  return 1;
}

template <int NT>
void skinny_shape_nt(bool gate, choreo_launch_config* out) {
  using S = choreo_sm100::SkinnyShape<NT>;
  out->stages = S::kStages;
  out->smem_bytes = S::kSmem;
  out->tmem_cols = static_cast<int32_t>(choreo_sm100::skinny_tmem_cols(NT * (gate ? 1 : S::kBufs)));
}
// What a query reports of the kernel for `nt` tokens.
inline void skinny_shape(int nt, bool gate, choreo_launch_config* out) {
  switch (nt) {
    case 16: return skinny_shape_nt<16>(gate, out);
    case 32: return skinny_shape_nt<32>(gate, out);
    case 64: return skinny_shape_nt<64>(gate, out);
    case 96: return skinny_shape_nt<96>(gate, out);
    default: return skinny_shape_nt<128>(gate, out);
  }
}

template <int KIND, int NT>
int launch_skinny_nt(const choreo_sm100::TwoMaps& tw, const CUtensorMap& tx, const choreo_sm100::SkinnyParams& kp,
                     int64_t tiles, cudaStream_t stream) {
  using namespace choreo_sm100;
  auto kern = skinny_kernel<KIND, NT>;
  constexpr int smem = SkinnyShape<NT>::kSmem;
  static std::atomic<uint64_t> done{0};
  if (int rc = set_smem_limit_once(kern, smem, done, "cudaFuncSetAttribute(skinny)")) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * kp.split));
  cfg.blockDim = dim3(kSkinnyThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {static_cast<unsigned>(kp.split), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = kp.split > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw, tx, kp);
  return e == cudaSuccess ? CHOREO_OK : cuda_fail(e, "skinny product launch");
}

template <int KIND>
int launch_skinny(const choreo_sm100::TwoMaps& tw, const CUtensorMap& tx, const choreo_sm100::SkinnyParams& kp,
                  int64_t tiles, cudaStream_t stream) {
  switch (skinny_tokens(kp.m)) {
    case 16: return launch_skinny_nt<KIND, 16>(tw, tx, kp, tiles, stream);
    case 32: return launch_skinny_nt<KIND, 32>(tw, tx, kp, tiles, stream);
    case 64: return launch_skinny_nt<KIND, 64>(tw, tx, kp, tiles, stream);
    case 96: return launch_skinny_nt<KIND, 96>(tw, tx, kp, tiles, stream);
    default: return launch_skinny_nt<KIND, 128>(tw, tx, kp, tiles, stream);
  }
}

}  // namespace choreo_impl
