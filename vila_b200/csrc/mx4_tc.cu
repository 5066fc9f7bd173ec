// Products of two microscaled 4-bit matrices on the tensor cores: tcgen05.mma kind::mxf4 with block scales.
//
//   D[p, q] = sum over blocks of 2^(sp + sq) * (32 products of 4-bit numbers), p the 128 TMEM lanes of a tile, q its columns.
//
// The instruction takes K = 64 columns (32 bytes) of both operands from shared memory and two scales a row from TMEM (a row's
// scales are one 32-bit word per 128 columns: lane r % 32 of column r / 32, the same in the four lane quarters, which is what
// tcgen05.cp.32x128b.warpx4 makes of 512 bytes in the tiled order of mx4.cuh).  No number is unpacked or rounded on the way.
//
//   TMA warp        a stage: 256 columns (128 bytes) of the tile's rows of P and of Q, 128-byte swizzle, and their scale tiles
//   MMA warp        TMEM allocation; scales to TMEM, then four tcgen05.mma a stage, into one of two accumulator sets
//   8 epilogue warps: bias, activation, gated unit, bf16 out, under the products of the next tile
//
// kSwap false: P = tokens, Q = weight rows (a lane writes 16 consecutive outputs of its token); true: P = weight rows, Q = tokens,
// for few tokens, whose number is then a multiple of 16 or so and not of 128.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "mx4.cuh"
#include "mx4_epi.cuh"

namespace vb {
namespace {

constexpr int kP = 128, kDepth = 256;                 // rows of P, columns of a stage
constexpr int kEpi = 8, kTma = kEpi, kMma = kEpi + 1, kThreads = 32 * (kEpi + 2);

template <int BN> struct Shape {
  static constexpr int kQTiles = (BN + 127) / 128;    // scale tiles of 128 rows; a tile begins with one
  static constexpr int kPBytes = kP * 128, kQBytes = BN * 128;
  static constexpr int kScales = 1024 * (1 + kQTiles);
  static constexpr int kStage = kPBytes + kQBytes + kScales;
  static constexpr int kStages = BN == 64 ? 4 : (BN == 128 ? 6 : 5);
  static constexpr int kPerSm = BN > 64 ? 1 : 2;
  static constexpr int kScaleCols = 8 * (1 + kQTiles);          // TMEM columns of a stage's scales
  static constexpr int kCols = 2 * BN + kStages * kScaleCols <= 256 ? 256 : 512;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStage + 256;
  static_assert(2 * BN + kStages * kScaleCols <= kCols, "TMEM");
  static_assert(kCols * kPerSm <= 512, "TMEM of an SM");
  static_assert(kSmem * kPerSm <= 227 * 1024, "shared memory");
};

// kind::mxf4: [4,6) scale index of B  [7,10) A = E2M1 (1)  [10,12) B = E2M1 (1)  [17,23) N >> 3  [23] scales are UE8M0
// [27,29) M >> 7  [29,31) scale index of A.  The scale index is the byte of the scale word at which the instruction's two begin.
__host__ __device__ constexpr uint32_t idesc_mx4(uint32_t M, uint32_t N, uint32_t scale_byte) {
  return (scale_byte << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 7) << 27) | (scale_byte << 29);
}
__device__ __forceinline__ void umma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}
// 512 bytes (32 rows of 16) -> 4 TMEM columns, in each of the four lane quarters
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int BN, bool kSwap>
__global__ void __launch_bounds__(kThreads, Shape<BN>::kPerSm)
mx4_tc_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const vila_mx4_linear_params p,
              const vila_glinear_ext x, const WaitLimit limit, volatile unsigned int* failed) {
  using S = Shape<BN>;
  constexpr int ST = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + ST * S::kStage);
  uint64_t* empty_bar = full_bar + ST;
  uint64_t* acc_full = empty_bar + ST;   // [2]
  uint64_t* acc_free = acc_full + 2;     // [2]
  uint64_t* drain_bar = acc_free + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* gave_up = reinterpret_cast<int*>(tmem_ptr + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P = kSwap ? p.N : p.M, Q = kSwap ? p.M : p.N;
  const int p_tiles = (P + kP - 1) / kP, q_tiles = (Q + BN - 1) / BN, total = p_tiles * q_tiles;
  const int nkb = (p.K + kDepth - 1) / kDepth, kts = 2 * nkb;
  auto tile_at = [&](int it, int& p0, int& q0) {     // the tiles that run together share their rows of Q (few of them)
    const int qt = it / p_tiles;
    p0 = (it - qt * p_tiles) * kP;
    q0 = qt * BN;
  };

  if (tid == 0) {
    tma_prefetch_desc(&tmap_p);
    tma_prefetch_desc(&tmap_q);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], kEpi);
    }
    mbar_init(drain_bar, 1);
    *gave_up = 0;
    fence_barrier_init();
  }
  if (warp == kMma) tmem_alloc<S::kCols>(tmem_ptr);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  bool ok = true;
  if (limit.quits >= 0) {
    ok = limit.quits != (warp == kTma ? 0 : warp == kMma ? 1 : 3);
    if (!ok) *gave_up = 1;
  }

  if (warp == kTma) {
    if (lane == 0) {
      const uint8_t *sp = kSwap ? p.w_scales : p.a_scales, *sq = kSwap ? p.a_scales : p.w_scales;
      const int q_row_tiles = (Q + 127) / 128;
      int s = 0, rounds = 0;              // rounds: through all the stages
      uint32_t ph = 1;                    // parity to wait for on an empty barrier: the first round passes
      for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
        int p0, q0;
        tile_at(it, p0, q0);
        const int qt0 = q0 >> 7, qts = min(S::kQTiles, q_row_tiles - qt0);
        const uint32_t bytes = S::kPBytes + S::kQBytes + 1024 * (1 + qts);
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_limited(&empty_bar[s], ph, gave_up, limit.tries);
          if (!ok) break;
          uint8_t* st = smem + s * S::kStage;
          mbar_arrive_expect_tx(&full_bar[s], bytes);
          tma_load_2d(st, &tmap_p, &full_bar[s], kb * 128, p0);
          tma_load_2d(st + S::kPBytes, &tmap_q, &full_bar[s], kb * 128, q0);
          uint8_t* sc = st + S::kPBytes + S::kQBytes;
          mx4_bulk_load(sc, sp + (static_cast<size_t>(p0 >> 7) * kts + 2 * kb) * 512, 1024, &full_bar[s]);
          for (int q = 0; q < qts; ++q)
            mx4_bulk_load(sc + 1024 * (1 + q), sq + (static_cast<size_t>(qt0 + q) * kts + 2 * kb) * 512, 1024, &full_bar[s]);
          if (++s == ST) {
            s = 0;
            ph ^= 1;
            ++rounds;
          }
        }
      }
      // what was asked for lands before the CTA's memory is given back, whichever warp gave up
      for (int i = 0; i < ST; ++i) {
        const int round = i < s ? rounds : rounds - 1;
        if (round >= 0) mbar_drain(&full_bar[i], round & 1);
      }
    }
  } else if (warp == kMma) {
    // The whole warp walks the loop and one lane issues: what the instructions are given stays in uniform registers.
    const bool one = elect_one();
    const uint64_t ad0 = make_smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128), bd0 = make_smem_desc(smem_u32(smem) + S::kPBytes, 16, 1024, kLayoutSW128);
    const uint64_t sd0 = make_smem_desc(smem_u32(smem) + S::kPBytes + S::kQBytes, 16, 128, kLayoutNone);
    int s = 0, k = 0;
    uint32_t ph = 0;
    for (int it = blockIdx.x; it < total && ok; it += gridDim.x, ++k) {
      int p0, q0;
      tile_at(it, p0, q0);
      const uint32_t n = kSwap ? min(BN, (Q - q0 + 15) & ~15) : BN, acc = tmem + (k & 1) * BN;
      const uint32_t idesc = idesc_mx4(kP, n, 0), idesc2 = idesc_mx4(kP, n, 2);
      ok = mx4_warp_wait(&acc_free[k & 1], ((k >> 1) & 1) ^ 1, gave_up, limit.tries);
      uint32_t here = mx4_test(&full_bar[s], ph);
      for (int kb = 0; kb < nkb && ok; ++kb) {
        if (!__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&full_bar[s], ph, gave_up, limit.tries);
        if (!ok) break;
        tc_fence_after();
        // Every stage has TMEM columns of its own for its scales: P's 128 columns twice, then Q's by column tile.  They are free
        // when the stage's shared memory is, which full_bar has said.
        const uint32_t ts = tmem + 2 * BN + s * S::kScaleCols, tq = ts + 8;
        const uint64_t ad = ad0 + s * (S::kStage >> 4), bd = bd0 + s * (S::kStage >> 4), sd = sd0 + s * (S::kStage >> 4);
        uint64_t* done = &empty_bar[s];
        if (++s == ST) {
          s = 0;
          ph ^= 1;
        }
        here = mx4_test(&full_bar[s], ph);
        if (one) {      // columns past K are zeros on both sides
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            scales_to_tmem(ts + 4 * h, sd + 32 * h);
#pragma unroll
            for (int q = 0; q < S::kQTiles; ++q) scales_to_tmem(tq + 4 * (S::kQTiles * h + q), sd + 64 * (1 + q) + 32 * h);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            umma_mx4(acc, ad + 2 * j, bd + 2 * j, j & 1 ? idesc2 : idesc, ts + 4 * (j >> 1), tq + 4 * S::kQTiles * (j >> 1), (kb | j) != 0);
          umma_commit(done);
        }
        __syncwarp();
      }
      if (ok && one) umma_commit(&acc_full[k & 1]);
      __syncwarp();
    }
    if (one) umma_commit(drain_bar);             // products under way end before TMEM and the CTA's memory are given back, too
    if (lane == 0) mbar_drain(drain_bar, 0);
    __syncwarp();
  } else {
    const int quad = warp & 3, half = warp >> 2;
    const bool wide = reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.ldo % 16 == 0;
    int k = 0;
    for (int it = blockIdx.x; it < total && ok; it += gridDim.x, ++k) {
      int p0, q0;
      tile_at(it, p0, q0);
      // all lanes or none: the TMEM loads need the whole warp
      ok = mx4_warp_wait(&acc_full[k & 1], (k >> 1) & 1, gave_up, limit.tries);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16) + (k & 1) * BN;
      const int row = p0 + quad * 32 + lane, cols = min(BN, Q - q0);
      const float bias = kSwap && p.bias && row < p.N ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[row]) : 0.f;
      mx4_with_epilogue(p, [&](auto epi) {
        constexpr int EPI = decltype(epi)::value;
        constexpr int kChunk = kSwap ? 16 : 32;
#pragma unroll 1
        for (int c = kChunk * half; c < cols; c += 2 * kChunk) {
          float r[kChunk];
          if constexpr (kSwap) tmem_ld_32x32b_x16(acc + c, reinterpret_cast<uint32_t*>(r));
          else tmem_ld_32x32b_x32(acc + c, reinterpret_cast<uint32_t*>(r));
          tmem_ld_wait();
          if constexpr (kSwap) mx4_store_col<EPI>(p, x, r, q0 + c, p.M, row, bias);
          else mx4_store_row<EPI>(p, x, r, row, q0 + c, wide);
        }
      });
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_free[k & 1]);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc<S::kCols>(tmem);
  }
  if (tid == 0 && *gave_up) {
    *failed = 1u;
    __threadfence_system();
  }
}

// ---- many tokens: tiles of 256 tokens x 256 weight rows by CTA pairs (cta_group::2) ----
// A single CTA's tile of 128 x 128 asks for 128 bytes of operands per clock of products, more than an SM takes in; the pair's, of
// which each CTA stages half the tokens and half the weight rows, for 64.  Each CTA's TMEM holds the sums of its 128 tokens for all 256
// weight rows, the scales of its tokens, and those of all the weight rows.
//
// TMEM has room for two accumulators of 256 columns, but not for the scales beside them.  So the two share kShared columns: the
// epilogue takes those first and says so, and the next tile's products begin then, under the rest of the epilogue.  Every stage
// has columns of its own for its scales, which are free when its shared memory is: with fewer places and a wait for the products
// that read one last, 8192 x 8192 x 8192 took 236 us instead of 198.
namespace pair {
constexpr int kN = 256, kStages = 5, kShared = 128;
constexpr int kPBytes = 128 * 128, kQBytes = 128 * 128, kScales = 1024 + 2048, kStage = kPBytes + kQBytes + kScales;
constexpr int kAcc1 = kN - kShared, kScaleCol = 2 * kN - kShared, kScaleCols = 24;
constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStage + 256;
static_assert(kScaleCol + kStages * kScaleCols <= 512 && kShared % 32 == 0 && kSmem <= 227 * 1024, "");

__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}
// in both CTAs, each from its own shared memory
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
mx4_pair_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_sp,
                const __grid_constant__ CUtensorMap tmap_sq, const vila_mx4_linear_params p, const vila_glinear_ext x, const WaitLimit limit,
                volatile unsigned int* failed) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kStages * kStage);   // the first CTA's: both CTAs' loads
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* acc_full = empty_bar + kStages;   // [2]
  uint64_t* shared_free = acc_full + 2;       // the first CTA's: the columns that the accumulators share, in both CTAs
  uint64_t* drain_bar = shared_free + 1;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* gave_up = reinterpret_cast<int*>(tmem_ptr + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = static_cast<int>(cluster_ctarank());
  const int p_tiles = (p.M + 255) / 256, q_tiles = (p.N + kN - 1) / kN, total = p_tiles * q_tiles;
  const int worker = blockIdx.x >> 1, workers = gridDim.x >> 1, nkb = (p.K + kDepth - 1) / kDepth;
  auto tile_at = [&](int it, int& p0, int& q0) {
    const int qt = it / p_tiles;
    p0 = (it - qt * p_tiles) * 256 + rank * 128;
    q0 = qt * kN;
  };

  if (tid == 0) {
    tma_prefetch_desc(&tmap_p);
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_sp);
    tma_prefetch_desc(&tmap_sq);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    mbar_init(&acc_full[0], 1);
    mbar_init(&acc_full[1], 1);
    mbar_init(shared_free, 2 * kEpi);
    mbar_init(drain_bar, 1);
    *gave_up = 0;
    fence_barrier_init();
  }
  if (warp == kMma) tmem_alloc_pair<512>(tmem_ptr);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  // a warp that gives up tells the other CTA, too
  auto tell = [&] {
    *gave_up = 1;
    st_dsmem_u32(mapa_u32(smem_u32(const_cast<int*>(gave_up)), rank ^ 1), 1u);
  };
  bool ok = true;
  if (limit.quits >= 0) ok = limit.quits != (warp == kTma ? 0 : warp == kMma ? 1 : 3);

  if (warp == kTma) {
    if (lane == 0) {
      int s = 0, rounds = 0;
      uint32_t ph = 1;
      for (int it = worker; it < total && ok; it += workers) {
        int p0, q0;
        tile_at(it, p0, q0);
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait_limited(&empty_bar[s], ph, gave_up, limit.tries);
          if (!ok) break;
          uint8_t* st = smem + s * kStage;
          const uint32_t bar = mapa_u32(smem_u32(&full_bar[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * kStage);
          tma_load_2d_pair(st, &tmap_p, bar, kb * 128, p0);
          tma_load_2d_pair(st + kPBytes, &tmap_q, bar, kb * 128, q0 + rank * 128);
          tma_load_3d_pair(st + kPBytes + kQBytes, &tmap_sp, bar, 0, 2 * kb, p0 >> 7);
          tma_load_3d_pair(st + kPBytes + kQBytes + 1024, &tmap_sq, bar, 0, 2 * kb, q0 >> 7);
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
            ++rounds;
          }
        }
      }
      if (!ok) tell();
      // what was asked for lands before the CTAs' memory is given back (their loads report to the first one)
      if (rank == 0)
        for (int i = 0; i < kStages; ++i) {
          const int round = i < s ? rounds : rounds - 1;
          if (round >= 0) mbar_drain(&full_bar[i], round & 1);
        }
    }
  } else if (warp == kMma) {
    if (rank == 0) {
      // The whole warp walks the loop and one lane issues: what the instructions are given stays in uniform registers.
      const bool one = elect_one();
      const uint64_t ad0 = make_smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128), bd0 = make_smem_desc(smem_u32(smem) + kPBytes, 16, 1024, kLayoutSW128);
      const uint64_t sd0 = make_smem_desc(smem_u32(smem) + kPBytes + kQBytes, 16, 128, kLayoutNone);
      int k = 0, s = 0;                   // tiles so far, stage
      uint32_t ph = 0;
      for (int it = worker; it < total && ok; it += workers, ++k) {
        const uint32_t acc = tmem + (k & 1) * kAcc1;
        if (k > 0) ok = mx4_warp_wait(shared_free, (k - 1) & 1, gave_up, limit.tries);
        uint32_t here = mx4_test(&full_bar[s], ph);
        for (int kb = 0; kb < nkb && ok; ++kb) {
          if (!__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&full_bar[s], ph, gave_up, limit.tries);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ts = tmem + kScaleCol + s * kScaleCols, tq = ts + 8;
          const uint64_t ad = ad0 + s * (kStage >> 4), bd = bd0 + s * (kStage >> 4), sd = sd0 + s * (kStage >> 4);
          uint64_t* done = &empty_bar[s];
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
          here = mx4_test(&full_bar[s], ph);
          if (one) {      // columns past K are zeros on both sides
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              scales_to_tmem_pair(ts + 4 * h, sd + 32 * h);
              scales_to_tmem_pair(tq + 8 * h, sd + 64 + 32 * h);
              scales_to_tmem_pair(tq + 8 * h + 4, sd + 128 + 32 * h);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              umma(acc, ad + 2 * i, bd + 2 * i, idesc_mx4(256, kN, 2 * (i & 1)), ts + 4 * (i >> 1), tq + 8 * (i >> 1), (kb | i) != 0);
            umma_commit_pair(done);
          }
          __syncwarp();
        }
        if (ok && one) umma_commit_pair(&acc_full[k & 1]);
        __syncwarp();
      }
      if (!ok && lane == 0) tell();
      if (one) umma_commit_pair(drain_bar);      // reports to both CTAs
    }
    // products under way, and what they report to this CTA, end before TMEM and the CTA's memory are given back
    if (lane == 0 && !mbar_wait_limited(drain_bar, 0, gave_up, limit.tries)) mbar_drain(drain_bar, 0);
    __syncwarp();
  } else {
    const int quad = warp & 3, half = warp >> 2;
    const bool wide = reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.ldo % 16 == 0;
    const uint32_t free_bar = mapa_u32(smem_u32(shared_free), 0);
    int k = 0;
    for (int it = worker; it < total && ok; it += workers, ++k) {
      int p0, q0;
      tile_at(it, p0, q0);
      ok = mx4_warp_wait(&acc_full[k & 1], (k >> 1) & 1, gave_up, limit.tries);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16) + (k & 1) * kAcc1;
      const int row = p0 + quad * 32 + lane, first = k & 1 ? 0 : kN - kShared;
      mx4_with_epilogue(p, [&](auto epi) {
        constexpr int EPI = decltype(epi)::value;
#pragma unroll 1
        for (int i = half; i < kN / 32; i += 2) {
          const int c = (first + 32 * i) & (kN - 1);      // the shared columns first
          float r[32];
          tmem_ld_32x32b_x32(acc + c, reinterpret_cast<uint32_t*>(r));
          tmem_ld_wait();
          if (i + 2 >= kShared / 32 && i < kShared / 32) {      // this warp's last one of them
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && it + workers < total) mbar_arrive_cluster_relaxed(free_bar);      // someone waits for it
          }
          if (q0 + c < p.N) mx4_store_row<EPI>(p, x, r, row, q0 + c, wide);
        }
      });
    }
    if (!ok && lane == 0) tell();
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync_all();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc_pair<512>(tmem);
  }
  if (tid == 0 && *gave_up) {
    *failed = 1u;
    __threadfence_system();
  }
}

int launch(const vila_mx4_linear_params& p, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  static PerDeviceOnce once;
  if (once.first()) VB_CUDA(cudaFuncSetAttribute(mx4_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem)));
  const int pitch = mx4_pitch(p.K), kts = mx4_ktiles(p.K);
  CUtensorMap tp, tq, sp, sq;
  if (int rc = make_tmap_2d_u8(&tp, p.a_codes, p.M, pitch, pitch, 128, 128, 128)) return rc;
  if (int rc = make_tmap_2d_u8(&tq, p.w_codes, p.N, pitch, pitch, 128, 128, 128)) return rc;
  if (int rc = make_tmap_3d_u32(&sp, p.a_scales, 128, kts, (p.M + 127) / 128, 2, 1)) return rc;
  if (int rc = make_tmap_3d_u32(&sq, p.w_scales, 128, kts, (p.N + 127) / 128, 2, 2)) return rc;
  const long long tiles = static_cast<long long>((p.M + 255) / 256) * ((p.N + kN - 1) / kN), most = num_sms() / 2;
  VB_CHECK(tiles < (1LL << 30), "mx4_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  VB_CUDA(launch_serial(mx4_pair_kernel, dim3(static_cast<unsigned>(2 * (tiles < most ? tiles : most))), dim3(kThreads), kSmem, stream, tp, tq, sp, sq, p, x,
                        wait_limit(tries), failed_word()));
  return 0;
}
}  // namespace pair

template <int BN, bool kSwap>
int launch(const vila_mx4_linear_params& p, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  using S = Shape<BN>;
  static PerDeviceOnce once;
  if (once.first())
    VB_CUDA(cudaFuncSetAttribute(mx4_tc_kernel<BN, kSwap>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem)));
  const int pitch = mx4_pitch(p.K);
  const uint8_t *pc = kSwap ? p.w_codes : p.a_codes, *qc = kSwap ? p.a_codes : p.w_codes;
  const int P = kSwap ? p.N : p.M, Q = kSwap ? p.M : p.N;
  CUtensorMap tp, tq;
  if (int rc = make_tmap_2d_u8(&tp, pc, P, pitch, pitch, kP, 128, 128)) return rc;
  if (int rc = make_tmap_2d_u8(&tq, qc, Q, pitch, pitch, BN, 128, 128)) return rc;
  const long long tiles = static_cast<long long>((P + kP - 1) / kP) * ((Q + BN - 1) / BN);
  VB_CHECK(tiles < (1LL << 31), "mx4_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  const long long most = static_cast<long long>(S::kPerSm) * num_sms();
  VB_CUDA(launch_serial(mx4_tc_kernel<BN, kSwap>, dim3(static_cast<unsigned>(tiles < most ? tiles : most)), dim3(kThreads), S::kSmem, stream, tp, tq, p, x,
                        wait_limit(tries), failed_word()));
  return 0;
}

}  // namespace

int mx4_tc(const vila_mx4_linear_params& p, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "mx4_linear: no pinned host memory for the status word");
  if (p.M <= 32) return launch<32, true>(p, x, tries, stream);
  if (p.M <= 64) return launch<64, true>(p, x, tries, stream);
  if (p.M <= 128) return launch<128, true>(p, x, tries, stream);
  if (p.M > 512) return pair::launch(p, x, tries, stream);
  return launch<128, false>(p, x, tries, stream);
}

}  // namespace vb
