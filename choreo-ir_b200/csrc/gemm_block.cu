// gemm_block.cu — C = act(alpha * S + beta * D + bias) for e4m3 operands with
// an fp32 scale for each block of 128 along K:
//   S[i,j] = sum_t sa(i,t) sb(j,t) * P_t[i,j],  P_t = A_t B_t^T over block t.
//
// The tensor cores sum one block: a k-block of the pipeline is exactly one
// scale block (128 e4m3 = 128 bytes per row), so each starts a fresh
// accumulator in TMEM. The epilogue warps read it out, multiply by the two
// scales and add it to the tile's fp32 sum, which stays in their registers for
// the whole tile; the next block runs meanwhile in the other accumulator.
//
// Bound by the fp32 sums of the epilogue, not by the MMAs: a 256 x 256 tile's
// k-block takes 512 cycles of MMAs and 729 in all (1334 with a scale per column,
// which doubles the arithmetic: a product of the two scales and the sum for
// every element), and on long calls by the 1 kW cap: 8192^3 with bf16 output
// 536-546 us = 2.0 PFLOP/s, 4096^3 80 us, the f32 weight gradient 4096 x 8192 x
// 10240 with both scales per row 566-586 us. That form spills 46 bytes a thread
// (108 read back); the one with a scale per 128 rows does not.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>

#include "internal.h"
#include "skinny.cuh"
#include "tc_kernel.cuh"

namespace choreo_sm100 {

constexpr int kBlockThreads = 384;  // warpgroup 0: producer, MMA issuer, scales; warpgroups 1 and 2: epilogue
constexpr int kBlockK = 128;        // e4m3 elements (bytes) per k-block

struct BlockParams : TcParams {
  const float* sa;
  int64_t sa_row, sa_blk;
  const float* sb;
  int64_t sb_row, sb_blk;
  const void* d;        // addend
  int64_t ldd;
  int32_t d_vec;
};

template <int STAGES, int BUFS>
struct alignas(8) BlockBarriers {
  uint64_t half[STAGES];      // tiles in halves: the first half's MMAs are done, its accumulator is full
  uint64_t full[STAGES];      // the stage's tiles have landed
  uint64_t empty[STAGES];     // all its MMAs are done: the stage is free, the (other half's) accumulator is full
  uint64_t tmem_empty[BUFS];  // the epilogue has read the accumulator
  uint64_t scale_full[4];     // a block's scales are in their slot
  uint64_t scale_empty[4];    // the epilogue has read them
  uint64_t drain;
  uint64_t probe[2];
  uint32_t tmem_base;
  int32_t abort;
};

template <bool PAIR, int BN>
struct BlockShape {
  static constexpr int kBRows = PAIR ? BN / 2 : BN;  // B rows one CTA stages
  static constexpr uint32_t kAStage = kBM * kBlockK;
  static constexpr uint32_t kBStage = kBRows * kBlockK;
  static constexpr int kStages = 6;
  static constexpr int kBufs = 512 / BN;  // block accumulators in TMEM
  // The epilogue follows a stage's barrier by its parity. The issuer runs at most
  // kBufs k-blocks ahead of it, so the barrier may not come round sooner.
  static_assert(kStages >= kBufs, "a stage's barrier would complete twice before the epilogue looks");
  // 256-column tiles are two MMAs of 128 columns with an accumulator each: half
  // h is 64 columns of each CTA's B rows, tile columns 64 h .. and 128 + 64 h ..
  // The two epilogue warps of an SM sub-partition take one half each, so they
  // work half a k-block apart, one's waits under the other's arithmetic (848 ->
  // 729 cycles a k-block, 8192^3 638 -> 539 us).
  static constexpr int kHalves = PAIR && BN == 256 ? 2 : 1;
  using Barriers = BlockBarriers<kStages, kBufs * kHalves>;
  static constexpr uint32_t kStaging = kEpiWarps * 2048;             // 32 rows x 64 bytes a warp
  static constexpr int kSlots = 4;                                   // scale slots
  static constexpr uint32_t kSlotFloats = 128 + (BN > 128 ? BN : 128);  // rows', then columns' (see the scale warps)
  static constexpr int kSmem = kStages * static_cast<int>(kAStage + kBStage) + static_cast<int>(kStaging) +
                               kSlots * static_cast<int>(kSlotFloats) * 4 + 1024 + static_cast<int>(sizeof(Barriers));
  // 128 sums a thread and two 32-column reads in flight need more registers
  // than an even share of the SM's
  static constexpr bool kMoveRegs = BN == 256;
  static constexpr int kEpiRegs = 224, kOtherRegs = 56;
};
static_assert(BlockShape<true, 256>::kEpiRegs * 256 + BlockShape<true, 256>::kOtherRegs * 128 <= 168 * kBlockThreads,
              "the warpgroups' shares must fit the registers of the launch");

__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
// d += (a0, a1) * s on packed pairs, one rounding per element.
__device__ __forceinline__ void fma2_acc(uint64_t& d, uint32_t a0, uint32_t a1, uint64_t s) {
  uint64_t a;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "r"(a0), "r"(a1));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(s));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void ld_shared_2x64(uint32_t addr, uint64_t& a, uint64_t& b) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(addr));
}

// Writes one warp's 32 rows x kCols columns of sums, 32 columns at a time:
// through its 2 KB staging buffer (32 rows of 64 bytes in the 64-byte swizzle:
// 16-byte chunk j of row r at j ^ (r / 2 % 4)) and bulk tensor stores, or
// element by element where those are not legal.
template <int kCols, typename OutT>
__device__ __forceinline__ void block_output(const uint64_t (&acc)[kCols / 2], int n_first, int n_second, int row0,
                                             const BlockParams& p, const CUtensorMap* tma_c, uint32_t stage_buf,
                                             int lane) {
  constexpr int E = 64 / static_cast<int>(sizeof(OutT));  // columns per staging row
  const int row = row0 + lane;
  const bool row_ok = row < p.m;
  const OutT* drow = static_cast<const OutT*>(p.d) + static_cast<int64_t>(row_ok ? row : 0) * p.ldd;
  OutT* crow = static_cast<OutT*>(p.c) + static_cast<int64_t>(row_ok ? row : 0) * p.ldc;
  TcParams pd = p;
  pd.c_vec_ok = p.d_vec;
  const uint32_t row_addr = stage_buf + static_cast<uint32_t>(lane) * 64u;
  const int sw = (lane >> 1) & 3;
#pragma unroll
  for (int c = 0; c < kCols / 32; ++c) {
    // the warp's first 64 columns start at n_first, the others at n_second
    const int n_base = c < 2 ? n_first + c * 32 : n_second + (c - 2) * 32;
    if (n_base >= p.n) continue;  // warp-uniform
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      asm("mov.b64 {%0, %1}, %2;" : "=r"(r[2 * i]), "=r"(r[2 * i + 1]) : "l"(acc[c * 16 + i]));
    float v[32];
    epilogue_values<OutT>(r, v, drow, n_base, pd, row_ok, lane);
    // A bulk tensor store clips columns in whole 16 bytes: a ragged last group
    // that ends inside 16 bytes is stored element by element.
    if (p.c_tma != 0 && (n_base + 32 <= p.n || p.n * static_cast<int>(sizeof(OutT)) % 16 == 0)) {
#pragma unroll
      for (int g = 0; g < 32 / E; ++g) {
        if (n_base + g * E >= p.n) break;  // warp-uniform
        if (lane == 0) bulk_wait_read_all();  // the warp's previous store has read the buffer
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t at = row_addr + static_cast<uint32_t>((j ^ sw) << 4);
          if constexpr (sizeof(OutT) == 2)
            st_shared_v4(at, pack2(v[8 * j], v[8 * j + 1], static_cast<OutT*>(nullptr)),
                         pack2(v[8 * j + 2], v[8 * j + 3], static_cast<OutT*>(nullptr)),
                         pack2(v[8 * j + 4], v[8 * j + 5], static_cast<OutT*>(nullptr)),
                         pack2(v[8 * j + 6], v[8 * j + 7], static_cast<OutT*>(nullptr)));
          else
            st_shared_v4(at, __float_as_uint(v[g * 16 + 4 * j]), __float_as_uint(v[g * 16 + 4 * j + 1]),
                         __float_as_uint(v[g * 16 + 4 * j + 2]), __float_as_uint(v[g * 16 + 4 * j + 3]));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(tma_c, stage_buf, n_base + g * E, row0, 0);
          bulk_commit_group();
        }
      }
    } else if (row_ok) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (n_base + i < p.n) crow[n_base + i] = from_f32<OutT>(v[i]);
    }
  }
}

// BVEC: a scale per row of B (1 x 128 blocks), else one per 128 rows.
template <bool PAIR, int BN, bool BVEC, typename OutT>
__device__ __forceinline__ void block_body(const CUtensorMap* tma_a, const CUtensorMap* tma_b, const CUtensorMap* tma_c,
                                           const BlockParams& p) {
  using S = BlockShape<PAIR, BN>;
  constexpr int STAGES = S::kStages;
  constexpr int kCols = BN / 2;  // columns of one epilogue warp
  constexpr uint32_t kTmemCols = 512;
  constexpr int kBufs = S::kBufs;
  constexpr int kHalves = S::kHalves;
  constexpr int kHalfN = BN / kHalves;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint8_t* s_a = smem;
  uint8_t* s_b = smem + STAGES * S::kAStage;
  uint8_t* s_stage = s_b + STAGES * S::kBStage;
  float* s_scale = reinterpret_cast<float*>(s_stage + S::kStaging);
  auto* bars = reinterpret_cast<typename S::Barriers*>(s_scale + S::kSlots * S::kSlotFloats);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const int64_t first = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  const int64_t step = PAIR ? gridDim.x >> 1 : gridDim.x;
  constexpr int kTileM = PAIR ? 2 * kBM : kBM;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), 1);
      mbar_init(smem_u32(&bars->half[s]), 1);
    }
    for (int i = 0; i < kBufs * kHalves; ++i)
      mbar_init(smem_u32(&bars->tmem_empty[i]), (PAIR ? 2 : 1) * kEpiWarps / kHalves);
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(smem_u32(&bars->scale_full[i]), 2);
      mbar_init(smem_u32(&bars->scale_empty[i]), kEpiWarps);
    }
    mbar_init(smem_u32(&bars->drain), 1);
    bars->abort = 0;
    probe_start(p, bars->probe);
    fence_mbar_init();
    tma_prefetch_desc(tma_a);
    tma_prefetch_desc(tma_b);
    if (p.c_tma) tma_prefetch_desc(tma_c);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(&bars->tmem_base), kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  const WaitCtx wctx{p.status, p.timeout_ns, &bars->abort};

  if (warp < 4) {
    if constexpr (S::kMoveRegs) regs_dec<S::kOtherRegs>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- producer
      griddep_wait();
      const uint64_t pol_a = l2_policy(p.l2_policy_a);
      const uint64_t pol_b = l2_policy(p.l2_policy_b);
      uint32_t stage = 0, phase = 0, issued = 0;
      bool ok = true;
      for (int64_t t = first; t < p.num_tiles && ok; t += step) {
        int b, mb, nb;
        tile_coords(t, p, b, mb, nb);
        const int m0 = mb * kTileM + static_cast<int>(rank) * kBM;
        const int n0 = nb * BN + static_cast<int>(rank) * S::kBRows;
        for (int kb = 0; kb < p.num_k_blocks; ++kb) {
          if (!mbar_wait(smem_u32(&bars->empty[stage]), phase ^ 1, wctx, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&bars->full[stage]);
          if (leader) mbar_arrive_expect_tx(fb, (PAIR ? 2 : 1) * (S::kAStage + S::kBStage));
          const uint32_t bar = PAIR ? mapa_shared(fb, 0) : fb;
          load3<PAIR>(smem_u32(s_a + stage * S::kAStage), tma_a, bar, kb * kBlockK, m0, 0, pol_a);
          load3<PAIR>(smem_u32(s_b + stage * S::kBStage), tma_b, bar, kb * kBlockK, n0, 0, pol_b);
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      griddep_launch_dependents();
      if (!ok) {
        if (leader) {
          const uint32_t inflight = issued < STAGES ? issued : STAGES;
          uint32_t s = stage, ph = phase;
          for (uint32_t i = 0; i < inflight; ++i) {
            if (s == 0) { s = STAGES - 1; ph ^= 1; } else { --s; }
            mbar_wait(smem_u32(&bars->full[s]), ph, wctx, kStatusTimeoutDrain, false);
          }
        } else {
          // The peer's loads count on the leader's barriers: give them time to land.
          const uint64_t t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 200000ull) {
          }
        }
      }
    } else if (warp == 1 && leader) {
      // ---------------------------------------------------------- MMA issuer
      // The whole warp runs the loop and one lane issues: operands that are the
      // same in every lane stay in uniform registers, where the MMA wants them.
      // Its chain of dependent instructions is what a short k-block waits for,
      // so it holds little: descriptors and barrier addresses advance by
      // additions, and a k-block's last commit tells the producer that the
      // stage is free and the epilogue that its accumulator is full.
      constexpr uint32_t idesc = idesc_e4m3(kTileM, kHalfN);
      const uint64_t desc_a = smem_desc_sw128(smem_u32(s_a), 16, 1024);
      const uint64_t desc_b = smem_desc_sw128(smem_u32(s_b), 16, 1024);
      const uint32_t bar_full = smem_u32(&bars->full[0]), bar_done = smem_u32(&bars->empty[0]);
      const uint32_t bar_half = smem_u32(&bars->half[0]);
      const uint32_t bar_free = smem_u32(&bars->tmem_empty[0]);
      uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 1;
      const int64_t blocks = (p.num_tiles - first + step - 1) / step * p.num_k_blocks;
      for (int64_t i = 0; i < blocks; ++i) {
        if (!mbar_wait_warp2(bar_full + 8 * stage, phase, bar_free + 8 * kHalves * buf, buf_phase, wctx,
                             kStatusTimeoutMma))
          break;
        tc_fence_after();
        const uint64_t ad = smem_desc_advance(desc_a, stage * S::kAStage);
        bool ok = true;
#pragma unroll
        for (uint32_t h = 0; h < kHalves; ++h) {
          if (h > 0) {
            ok = mbar_wait_warp(bar_free + 8 * (kHalves * buf + h), buf_phase, wctx, kStatusTimeoutMma);
            if (!ok) break;
            tc_fence_after();
          }
          const uint64_t bd = smem_desc_advance(desc_b, stage * S::kBStage + h * (S::kBStage / kHalves));
          const uint32_t d = tmem_base + buf * BN + h * kHalfN;
          if (elect_one()) {
#pragma unroll
            for (uint32_t k = 0; k < kBlockK / 32; ++k) {
              if constexpr (PAIR)
                umma_f8_pair(d, smem_desc_advance(ad, k * 32), smem_desc_advance(bd, k * 32), idesc, k != 0 ? 1u : 0u);
              else
                umma_f8(d, smem_desc_advance(ad, k * 32), smem_desc_advance(bd, k * 32), idesc, k != 0 ? 1u : 0u);
            }
            const uint32_t done = (h + 1 == kHalves ? bar_done : bar_half) + 8 * stage;
            if constexpr (PAIR) umma_commit_pair_both(done); else umma_commit(done);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        if (++buf == kBufs) { buf = 0; buf_phase ^= 1; }
      }
      if (elect_one()) {
        if constexpr (PAIR) umma_commit_pair(smem_u32(&bars->drain)); else umma_commit(smem_u32(&bars->drain));
      }
      mbar_wait(smem_u32(&bars->drain), 0, wctx, kStatusTimeoutDrain, false);
      __syncwarp();
    } else if (warp >= 2) {
      // ------------------------------------------------------- scale warps
      // Each k-block's scales go through a ring of shared-memory slots, so the
      // epilogue neither addresses nor waits for global memory: with one scale
      // per 128 rows of B the products sa(row) sb(128 columns), 2 x 128; else
      // the 128 row scales and the BN column scales. The two warps take half
      // of the rows and of the columns each, loaded kAhead blocks ahead.
      griddep_wait();
      constexpr int kAhead = 4;
      constexpr int kSb = BVEC ? BN / 64 : 2;  // column values a lane holds
      const int half = warp - 2;
      uint32_t slot = 0, phase = 0;
      bool ok = true;
      for (int64_t t = first; t < p.num_tiles && ok; t += step) {
        int b, mb, nb;
        tile_coords(t, p, b, mb, nb);
        const int r0 = mb * kTileM + static_cast<int>(rank) * kBM + half * 64 + lane;
        const float* sa[2];
        const float* sb[kSb];
#pragma unroll
        for (int i = 0; i < 2; ++i) sa[i] = p.sa + static_cast<int64_t>(min(r0 + 32 * i, p.m - 1)) * p.sa_row;
#pragma unroll
        for (int i = 0; i < kSb; ++i) {
          const int n = BVEC ? nb * BN + half * (BN / 2) + 32 * i + lane : nb * BN + i * (BN / 2);
          sb[i] = p.sb + static_cast<int64_t>(min(n, p.n - 1) / (BVEC ? 1 : 128)) * p.sb_row;
        }
        float qa[kAhead][2], qb[kAhead][kSb];
        auto load = [&](int kb, float (&va)[2], float (&vb)[kSb]) {
          if (kb >= p.num_k_blocks) return;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            va[i] = ldg_early(sa[i]);
            sa[i] += p.sa_blk;
          }
#pragma unroll
          for (int i = 0; i < kSb; ++i) {
            vb[i] = ldg_early(sb[i]);
            sb[i] += p.sb_blk;
          }
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(i, qa[i], qb[i]);
        // Unrolled by kAhead: each queue entry is registers of its own (moving
        // a value that is still in flight would wait for it).
#pragma unroll 1
        for (int kb0 = 0; kb0 < p.num_k_blocks && ok; kb0 += kAhead) {
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            if (kb0 + u >= p.num_k_blocks) break;
            if (!mbar_wait_warp(smem_u32(&bars->scale_empty[slot]), phase ^ 1, wctx, kStatusTimeoutProducer)) {
              ok = false;
              break;
            }
            float* rows = s_scale + slot * S::kSlotFloats + half * 64 + lane;
            if constexpr (BVEC) {
              float* cols = s_scale + slot * S::kSlotFloats + 128 + half * (BN / 2) + lane;
#pragma unroll
              for (int i = 0; i < 2; ++i) rows[32 * i] = qa[u][i];
#pragma unroll
              for (int i = 0; i < kSb; ++i) cols[32 * i] = qb[u][i];
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) rows[h * 128 + 32 * i] = qa[u][i] * qb[u][h];
            }
            __syncwarp();
            mbar_arrive_lane0(smem_u32(&bars->scale_full[slot]), lane);
            load(kb0 + u + kAhead, qa[u], qb[u]);
            if (++slot == S::kSlots) { slot = 0; phase ^= 1; }
          }
        }
      }
    }
  } else {
    if constexpr (S::kMoveRegs) regs_inc<S::kEpiRegs>();
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;
    const int col_half = (warp - 4) >> 2;
    const uint32_t stage_buf = smem_u32(s_stage) + static_cast<uint32_t>(warp - 4) * 2048u;
    const uint32_t tmem_warp = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + col_half * kCols;
    // its accumulator: half col_half of the tile (halves), or the tile's
    const int half = kHalves == 2 ? col_half : 0;
    const uint32_t bar_done = smem_u32(kHalves == 2 && half == 0 ? &bars->half[0] : &bars->empty[0]);
    const uint32_t own_free = smem_u32(&bars->tmem_empty[half]);
    const uint32_t bar_free = PAIR ? mapa_shared(own_free, 0) : own_free;
    // first columns of its first and second 64 within the tile
    const int seg0 = kHalves == 2 ? 64 * half : col_half * kCols;
    const int seg1 = kHalves == 2 ? 128 + 64 * half : seg0 + 64;
    const uint32_t scale_full = smem_u32(&bars->scale_full[0]), scale_empty = smem_u32(&bars->scale_empty[0]);
    // this lane's row scale, and the warp's column scales, in slot 0
    const uint32_t scale_row =
        smem_u32(s_scale) +
        static_cast<uint32_t>((BVEC || kHalves == 2 ? 0 : col_half * 128) + quarter * 32 + lane) * 4u;
    const uint32_t scale_col = smem_u32(s_scale) + 128u * 4u;
    griddep_wait();
    uint32_t stage = 0, phase = 0, buf = 0, slot = 0, slot_phase = 0;
    bool ok = true;
    for (int64_t t = first; t < p.num_tiles && ok; t += step) {
      int b, mb, nb;
      tile_coords(t, p, b, mb, nb);
      const int row0 = mb * kTileM + static_cast<int>(rank) * kBM + quarter * 32;
      const int n_first = nb * BN + seg0;
      const bool active = row0 < p.m && n_first < p.n;
      uint64_t acc[kCols / 2];  // the warp's sums, in pairs of columns
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) acc[i] = 0;
#pragma unroll 1
      for (int kb = 0; kb < p.num_k_blocks; ++kb) {
        if (!mbar_wait_warp2(scale_full + 8 * slot, slot_phase, bar_done + 8 * stage, phase, wctx,
                             kStatusTimeoutEpilogue)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem_warp + buf * BN;
        // Two 32-column reads of TMEM alternate: one is in flight while the
        // other is used. Warps past the matrix's edge add up zeros rather than
        // branch: without branches the warp stays converged and the chunks in
        // one piece of code (866 -> 848 cycles a k-block, with column scales 1559
        // -> 1342).
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(taddr, r[0]);
        const float s = ld_shared_f32(scale_row + slot * (S::kSlotFloats * 4));
        const uint32_t cols = scale_col + slot * (S::kSlotFloats * 4);
        const uint64_t s2 = pack_f32x2(s, s);
        // halves: the second 64 columns lie in B's next 128 rows
        uint64_t s2_second = s2;
        if constexpr (kHalves == 2 && !BVEC) {
          const float second = ld_shared_f32(scale_row + slot * (S::kSlotFloats * 4) + 512u);
          s2_second = pack_f32x2(second, second);
        }
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if constexpr (PAIR)
            mbar_arrive_cluster_lane0(bar_free + 8 * kHalves * buf, lane);
          else
            mbar_arrive_lane0(bar_free + 8 * kHalves * buf, lane);
        };
        tmem_wait_ld(r[0]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          if (c + 1 < kCols / 32) tmem_ld_32x32b_x32(taddr + (c + 1) * 32, r[(c + 1) & 1]); else release();
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            uint64_t c0 = c < 2 ? s2 : s2_second, c1 = c0;
            if constexpr (BVEC) {
              const int col = (c < 2 ? seg0 + c * 32 : seg1 + (c - 2) * 32) + 2 * j;
              ld_shared_2x64(cols + static_cast<uint32_t>(col) * 4u, c0, c1);
              c0 = mul2(s2, c0);
              c1 = mul2(s2, c1);
            }
            fma2_acc(acc[c * 16 + j], r[c & 1][2 * j], r[c & 1][2 * j + 1], c0);
            fma2_acc(acc[c * 16 + j + 1], r[c & 1][2 * j + 2], r[c & 1][2 * j + 3], c1);
          }
          if (c + 1 < kCols / 32) tmem_wait_ld(r[(c + 1) & 1]);
        }
        // Every lane has read its column scales (the row scale was read before release()).
        if constexpr (BVEC) __syncwarp();
        mbar_arrive_lane0(scale_empty + 8 * slot, lane);
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        if (++buf == kBufs) buf = 0;
        if (++slot == S::kSlots) { slot = 0; slot_phase ^= 1; }
      }
      if (ok && active) block_output<kCols, OutT>(acc, n_first, nb * BN + seg1, row0, p, tma_c, stage_buf, lane);
    }
    if (lane == 0) bulk_wait_read_all();
    __syncwarp();
  }

  tc_fence_before();
  if constexpr (PAIR) cluster_sync(); else __syncthreads();
  probe_end(p, bars->probe);
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, kTmemCols); else tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int BN, bool BVEC, typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kBlockThreads, 1)
    block_pair_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                      const __grid_constant__ CUtensorMap tma_c, const BlockParams p) {
  block_body<true, BN, BVEC, OutT>(&tma_a, &tma_b, &tma_c, p);
}
template <int BN, bool BVEC, typename OutT>
__global__ void __launch_bounds__(kBlockThreads, 1)
    block_single_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                        const __grid_constant__ CUtensorMap tma_c, const BlockParams p) {
  block_body<false, BN, BVEC, OutT>(&tma_a, &tma_b, &tma_c, p);
}

}  // namespace choreo_sm100

namespace choreo_impl {
using namespace choreo_sm100;

namespace {

struct BlockConfig {
  bool pair;
  int bn;
};

BlockConfig select_block_config(int64_t m, int64_t n) {
  const int sms = current_sm_count();
  // 128 x 128 tiles on single CTAs while they fit one wave, else 256 x 256 tiles
  // on CTA pairs (four of the small ones). 512 x 4096 x 4096, 128 small tiles:
  // 13.2 us against 17.8 in pairs; 1031 x 2053 x 1999, 153 of them: 15.8 against
  // 12.6; 2048^3, 256: 14.2 against 12.7. With a scale per column 18.3 / 28.6,
  // 19.0 / 18.1 and 19.5 / 18.0.
  const int64_t singles = ((m + 127) / 128) * ((n + 127) / 128);
  return singles > sms ? BlockConfig{true, 256} : BlockConfig{false, 128};
}

template <typename Kern>
int launch_block(Kern kern, int smem, bool move_regs, std::atomic<uint64_t>& attr_done, const CUtensorMap& ta,
                 const CUtensorMap& tb, const CUtensorMap& tc, const BlockParams& kp, int grid, cudaStream_t s) {
  if (int rc = set_smem_limit_once(kern, smem, attr_done, "cudaFuncSetAttribute(block-scaled GEMM)")) return rc;
  if (move_regs) {
    // The epilogue's larger share comes out of the launch's registers: it must be there.
    cudaFuncAttributes fa{};
    const cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes(block-scaled GEMM)");
    if (fa.numRegs < 168)
      return fail(CHOREO_ERR_UNSUPPORTED, "block-scaled GEMM: built with %d registers per thread, needs 168", fa.numRegs);
  }
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kBlockThreads), smem, s, ta, tb, tc, kp);
  return e == cudaSuccess ? CHOREO_OK : cuda_fail(e, "block-scaled GEMM launch");
}

template <bool BVEC, typename OutT>
int dispatch_block(const BlockConfig& c, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                   const BlockParams& kp, int grid, cudaStream_t s) {
  if (c.pair) {
    using S = BlockShape<true, 256>;
    static std::atomic<uint64_t> done{0};
    return launch_block(block_pair_kernel<256, BVEC, OutT>, S::kSmem, S::kMoveRegs, done, ta, tb, tc, kp, grid, s);
  }
  using S = BlockShape<false, 128>;
  static std::atomic<uint64_t> done{0};
  return launch_block(block_single_kernel<128, BVEC, OutT>, S::kSmem, S::kMoveRegs, done, ta, tb, tc, kp, grid, s);
}

int encode_e4m3(CUtensorMap* map, const void* p, int64_t rows, int64_t k, int64_t ld, uint32_t box_rows) {
  if (rows == 1) ld = round_up(k, 16);  // never stepped over, but a map's stride has to be whole 16 bytes
  const uint64_t dims[3] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld), static_cast<uint64_t>(rows) * static_cast<uint64_t>(ld)};
  const uint32_t box[3] = {kBlockK, box_rows, 1};
  return encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int validate_block(const choreo_gemm_block_desc* d) {
  const char* what = "block-scaled GEMM";
  if (d == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "%s: null descriptor", what);
  if (d->m <= 0 || d->n <= 0 || d->k <= 0)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: Invalid matrix dimensions: M=%lld, N=%lld, K=%lld", what, (long long)d->m,
                (long long)d->n, (long long)d->k);
  if (d->m > INT32_MAX / 2 || d->n > INT32_MAX / 2 || d->k > INT32_MAX / 2)
    return fail(CHOREO_ERR_UNSUPPORTED, "%s: dimensions above 2^30-1 are not supported", what);
  if (d->a == nullptr || d->b == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "%s: an operand has null data pointer", what);
  if (d->scale_a == nullptr || d->scale_b == nullptr)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: a scale has null data pointer", what);
  if (d->c == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "%s: Output tensor C has null data pointer", what);
  if (!is_float_type(d->dtype_c)) return fail(CHOREO_ERR_UNSUPPORTED, "%s: unsupported output dtype %d", what, d->dtype_c);
  if (d->block_b != 1 && d->block_b != 128)
    return fail(CHOREO_ERR_UNSUPPORTED, "%s: block_b %d is neither 1 nor 128", what, d->block_b);
  if (d->lda < d->k || d->ldb < d->k)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: lda=%lld or ldb=%lld smaller than K=%lld", what, (long long)d->lda,
                (long long)d->ldb, (long long)d->k);
  // (a single row has no leading dimension to speak of)
  if ((d->m > 1 && d->lda % 16 != 0) || (d->n > 1 && d->ldb % 16 != 0) || (reinterpret_cast<uintptr_t>(d->a) & 15u) != 0 ||
      (reinterpret_cast<uintptr_t>(d->b) & 15u) != 0)
    return fail(CHOREO_ERR_INVALID_ARG,
                "%s: A, B and their leading dimensions must be multiples of 16 bytes (lda=%lld, ldb=%lld)", what,
                (long long)d->lda, (long long)d->ldb);
  if (d->ldc < d->n)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: ldc=%lld smaller than N=%lld", what, (long long)d->ldc, (long long)d->n);
  if (d->scale_a_row < 0 || d->scale_a_blk < 0 || d->scale_b_row < 0 || d->scale_b_blk < 0)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: negative scale stride", what);
  if (d->addend && d->ld_addend < d->n)
    return fail(CHOREO_ERR_INVALID_ARG, "%s: ld_addend=%lld smaller than N=%lld", what, (long long)d->ld_addend,
                (long long)d->n);
  if (d->bias && !is_float_type(d->dtype_bias))
    return fail(CHOREO_ERR_UNSUPPORTED, "%s: unsupported bias dtype %d", what, d->dtype_bias);
  const struct {
    const void* p;
    const char* name;
  } ptrs[] = {{d->a, "block-scaled GEMM A"},           {d->b, "block-scaled GEMM B"},
              {d->scale_a, "block-scaled GEMM scale A"}, {d->scale_b, "block-scaled GEMM scale B"},
              {d->c, "block-scaled GEMM C"},           {d->beta != 0.f ? d->addend : nullptr, "block-scaled GEMM addend"},
              {d->bias, "block-scaled GEMM bias"}};
  for (const auto& q : ptrs)
    if (q.p)
      if (int rc = check_device_ptr(q.p, q.name)) return rc;
  return CHOREO_OK;
}

int64_t block_tiles(const choreo_gemm_block_desc& d, const BlockConfig& c) {
  const int64_t rows = c.pair ? 256 : 128;
  return ((d.m + rows - 1) / rows) * ((d.n + c.bn - 1) / c.bn);
}
int block_grid(int64_t tiles, const BlockConfig& c) {
  const int sms = current_sm_count();
  return static_cast<int>(c.pair ? 2 * std::min<int64_t>(tiles, sms / 2) : std::min<int64_t>(tiles, sms));
}

constexpr int kSkinnyCols = 128;  // columns of C in a skinny tile

int launch_block_skinny(const choreo_gemm_block_desc& d, cudaStream_t stream) {
  CUtensorMap tx;
  TwoMaps tw;
  int rc = encode_e4m3(&tx, d.a, d.m, d.k, d.lda, static_cast<uint32_t>(skinny_tokens(d.m)));
  if (rc) return rc;
  if ((rc = encode_e4m3(&tw.m[0], d.b, d.n, d.k, d.ldb, 128))) return rc;
  tw.m[1] = tw.m[0];
  SkinnyParams kp;
  std::memset(&kp, 0, sizeof(kp));
  kp.m = static_cast<int32_t>(d.m);
  kp.n = static_cast<int32_t>(d.n);
  kp.num_k_blocks = static_cast<int32_t>((d.k + kBlockK - 1) / kBlockK);
  const int64_t tiles = (d.n + kSkinnyCols - 1) / kSkinnyCols;
  kp.split = skinny_split(tiles, kp.num_k_blocks, current_sm_count());
  kp.c = d.c;
  kp.ldc = d.ldc;
  kp.alpha = d.alpha;
  kp.beta = d.beta;
  kp.bias = d.bias;
  kp.dtype_bias = d.dtype_bias;
  kp.relu = d.relu;
  kp.dtype_c = d.dtype_c;
  kp.block_b = d.block_b;
  kp.sa = d.scale_a;
  kp.sa_row = d.scale_a_row;
  kp.sa_blk = d.scale_a_blk;
  kp.sb = d.scale_b;
  kp.sb_row = d.scale_b_row;
  kp.sb_blk = d.scale_b_blk;
  kp.d = d.addend ? d.addend : d.c;
  kp.ldd = d.addend ? d.ld_addend : d.ldc;
  kp.status = status_word();
  kp.timeout_ns = wait_timeout_ns();
  if (kp.status == nullptr) return CHOREO_ERR_CUDA;
  return launch_skinny<kBlock>(tw, tx, kp, tiles, stream);
}

}  // namespace
}  // namespace choreo_impl

using namespace choreo_impl;

extern "C" {

int choreo_gemm_block_scaled_query(const choreo_gemm_block_desc* d, choreo_launch_config* out) {
  int rc = validate_block(d);
  if (rc) return rc;
  if (out == nullptr) return fail(CHOREO_ERR_INVALID_ARG, "block-scaled GEMM query: null output");
  std::memset(out, 0, sizeof(*out));
  out->kernel = 5;
  out->tile_k = kBlockK;
  out->grid_y = out->grid_z = 1;
  out->split_k = 1;
  if (d->m <= kSkinnyRows) {
    const int nt = skinny_tokens(d->m);
    out->tile_m = nt;
    out->tile_n = kSkinnyCols;
    out->tiles = (d->n + kSkinnyCols - 1) / kSkinnyCols;
    out->split_k = skinny_split(out->tiles, (d->k + kBlockK - 1) / kBlockK, current_sm_count());
    out->cluster_m = static_cast<int32_t>(out->split_k);
    out->tiles *= out->split_k;
    out->grid_x = static_cast<int32_t>(out->tiles);
    out->block_x = kSkinnyThreads;
    skinny_shape(nt, false, out);
    return ok();
  }
  const BlockConfig c = select_block_config(d->m, d->n);
  out->tile_m = c.pair ? 256 : 128;
  out->tile_n = c.bn;
  out->stages = c.pair ? BlockShape<true, 256>::kStages : BlockShape<false, 128>::kStages;
  out->cluster_m = c.pair ? 2 : 1;
  out->tiles = block_tiles(*d, c);
  out->grid_x = block_grid(out->tiles, c);
  out->block_x = kBlockThreads;
  out->smem_bytes = c.pair ? BlockShape<true, 256>::kSmem : BlockShape<false, 128>::kSmem;
  out->tmem_cols = 512;
  return ok();
}

int choreo_gemm_block_scaled(const choreo_gemm_block_desc* d, void* stream) {
  int rc = validate_block(d);
  if (rc) return rc;
  if (d->m <= kSkinnyRows) {
    rc = launch_block_skinny(*d, static_cast<cudaStream_t>(stream));
    return rc ? rc : ok();
  }
  const BlockConfig c = select_block_config(d->m, d->n);
  CUtensorMap ta, tb, tc;
  if ((rc = encode_e4m3(&ta, d->a, d->m, d->k, d->lda, 128))) return rc;
  if ((rc = encode_e4m3(&tb, d->b, d->n, d->k, d->ldb, static_cast<uint32_t>(c.pair ? c.bn / 2 : c.bn)))) return rc;
  BlockParams kp;
  std::memset(&kp, 0, sizeof(kp));
  kp.m = static_cast<int32_t>(d->m);
  kp.n = static_cast<int32_t>(d->n);
  kp.num_k_blocks = static_cast<int32_t>((d->k + kBlockK - 1) / kBlockK);
  const int rows = c.pair ? 256 : 128;
  kp.num_m_blocks = static_cast<int32_t>((d->m + rows - 1) / rows);
  kp.num_n_blocks = static_cast<int32_t>((d->n + c.bn - 1) / c.bn);
  kp.batch = 1;
  kp.num_tiles = block_tiles(*d, c);
  const L2Plan l2 = l2_plan();
  kp.group_m = group_tiles(l2, rows, kp.num_m_blocks);
  kp.l2_policy_a = l2.policy_a;
  kp.l2_policy_b = l2.policy_b;
  kp.c = d->c;
  kp.ldc = d->ldc;
  kp.alpha = d->alpha;
  kp.beta = d->beta;
  kp.bias = d->bias;
  kp.dtype_bias = d->dtype_bias;
  kp.relu = d->relu;
  kp.sa = d->scale_a;
  kp.sa_row = d->scale_a_row;
  kp.sa_blk = d->scale_a_blk;
  kp.sb = d->scale_b;
  kp.sb_row = d->scale_b_row;
  kp.sb_blk = d->scale_b_blk;
  kp.d = d->addend ? d->addend : d->c;
  kp.ldd = d->addend ? d->ld_addend : d->ldc;
  const int eb = dtype_bytes(d->dtype_c);
  kp.d_vec = ((reinterpret_cast<uintptr_t>(kp.d) | static_cast<uintptr_t>(kp.ldd * eb)) & 15u) == 0;
  std::memset(&tc, 0, sizeof(tc));
  kp.c_vec_ok = kp.c_tma = ((reinterpret_cast<uintptr_t>(d->c) | static_cast<uintptr_t>(d->ldc * eb)) & 15u) == 0;
  if (kp.c_tma) {
    const uint64_t dims[3] = {static_cast<uint64_t>(d->n), static_cast<uint64_t>(d->m), 1};
    const uint64_t strides[2] = {static_cast<uint64_t>(d->ldc) * eb, static_cast<uint64_t>(d->m) * d->ldc * eb};
    const uint32_t box[3] = {static_cast<uint32_t>(64 / eb), 32, 1};
    const CUtensorMapDataType dt = d->dtype_c == CHOREO_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : d->dtype_c == CHOREO_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if ((rc = encode_tmap(&tc, dt, 3, d->c, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B))) return rc;
  }
  kp.status = status_word();
  kp.timeout_ns = wait_timeout_ns();
  kp.clock_probe = clock_probe();
  if (kp.status == nullptr) return CHOREO_ERR_CUDA;
  const int grid = block_grid(kp.num_tiles, c);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool vec = d->block_b == 1;
  switch (d->dtype_c) {
    case CHOREO_DTYPE_F16:
      rc = vec ? dispatch_block<true, __half>(c, ta, tb, tc, kp, grid, s)
               : dispatch_block<false, __half>(c, ta, tb, tc, kp, grid, s);
      break;
    case CHOREO_DTYPE_BF16:
      rc = vec ? dispatch_block<true, __nv_bfloat16>(c, ta, tb, tc, kp, grid, s)
               : dispatch_block<false, __nv_bfloat16>(c, ta, tb, tc, kp, grid, s);
      break;
    default:
      rc = vec ? dispatch_block<true, float>(c, ta, tb, tc, kp, grid, s)
               : dispatch_block<false, float>(c, ta, tb, tc, kp, grid, s);
  }
  return rc ? rc : ok();
}

}  // extern "C"
