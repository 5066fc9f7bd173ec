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
// kSwap false: P = tokens, Q = weight rows (a lane writes 32 consecutive outputs of its token); true: P = weight rows, Q = tokens,
// for few tokens, whose number is then a multiple of 16 and not of 128, and K is split over a cluster of up to 8 CTAs where the weight
// rows' tiles leave SMs idle (the parts are added in rank order through distributed shared memory).
//
// kPieces: few bf16 tokens on 4-bit weights, by the same products.  A token is cut into 16 rows of 4-bit numbers that add up to it
// (mx4_pieces): a block's numbers in units u_0 = 2^(floor(log2 max) - 2) are below 8, the nearest 4-bit number leaves at most 2, which are
// at most 8 of the next row's units u_1 = u_0 / 4, and so on; what 16 rows leave is under 2^-31 of the block's largest magnitude, and of
// bf16's 8 bits nothing at all where a number is above 2^-22 of it.  That holds for small blocks, too, as the rows' scales are 2^kPieceUnits too
// large: scale bytes end at 2^-127, units at 2^-135.  bf16 numbers are multiples of 2^-133; in the last unit but one, 2^-132 or 2^-133, what is left
// is a multiple of a half and below 8, its nearest 4-bit number leaves 0, 1/2, 1 or 3/2, and the last row holds four times that.  Blocks
// of 2^122 and more have no scale.  The 16 columns of a token are added in fp32, and the 2^kPieceUnits taken out; a sum that is not finite
// (a block without a scale reads as NaN) is taken again from the token itself (sum_again).  The tensor core has
// that to spare (128 weight rows x 16 columns x 256: about 60 clocks, their codes take 300 to arrive), while unpacking weights
// to f16 is bound by integer instructions: mx4_rows.cu takes 22.0 us for one token on 37888 x 3584, this 15.9.
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
  static constexpr int kCols = 2 * BN + kStages * kScaleCols <= 128 ? 128 : (2 * BN + kStages * kScaleCols <= 256 ? 256 : 512);
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
constexpr int kPieceRows = 16, kPieceUnits = 8;
// One sum term by term, where the cut rows' came out infinite or NaN: of a block with an infinity or a NaN they know no more than that (its first
// row reads as NaN), and one row's part of a sum may leave fp32's range alone.  x: the token's row, n: the weight row.
__device__ __noinline__ float sum_again(const __nv_bfloat16* x, const uint8_t* codes, const uint8_t* scales, int n, int K) {
  const int pitch = mx4_pitch(K), kts = mx4_ktiles(K);
  float s = 0.f;
  for (int k = 0; k < K && s == s; k += 32) {
    const uint4 c4 = __ldg(reinterpret_cast<const uint4*>(codes + static_cast<size_t>(n) * pitch + k / 2));
    const float unit = mx4_scale(__ldg(scales + mx4_scale_at(n, k >> 7, kts) + (k >> 5 & 3)));
    const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
    for (int i = 0; i < 32 && k + i < K; ++i) s = fmaf(__bfloat162float(x[k + i]), mx4_number(c[i >> 3] >> (4 * (i & 7)) & 15u) * unit, s);
  }
  return s;
}
template <int BN, bool kSwap, bool kPieces>
__global__ void __launch_bounds__(kThreads, Shape<BN>::kPerSm)
mx4_tc_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const vila_mx4_linear_params p,
              const vila_glinear_ext x, const int split, const WaitLimit limit, volatile unsigned int* failed) {
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
  const int P = kSwap ? p.N : p.M, Q = kSwap ? (kPieces ? kPieceRows * p.M : p.M) : p.N;
  const int p_tiles = (P + kP - 1) / kP, q_tiles = (Q + BN - 1) / BN, total = p_tiles * q_tiles;
  const int nkb = (p.K + kDepth - 1) / kDepth, kts = 2 * nkb;
  // a cluster's CTAs share a tile and cut K; without clusters split is 1
  const int rank = static_cast<int>(blockIdx.x) % split, it0 = static_cast<int>(blockIdx.x) / split, it_step = static_cast<int>(gridDim.x) / split;
  const int kb0 = static_cast<int>(static_cast<long long>(nkb) * rank / split), kb1 = static_cast<int>(static_cast<long long>(nkb) * (rank + 1) / split);
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
    const bool one = elect_one();
    const uint8_t *sp = kSwap ? p.w_scales : p.a_scales, *sq = kSwap ? p.a_scales : p.w_scales;
    const int q_row_tiles = (Q + 127) / 128;
    int s = 0, rounds = 0;                // stage, rounds through all of them
    uint32_t ph = 1, here = 1;            // parity to wait for on an empty barrier: the first round passes
    for (int it = it0; it < total && ok; it += it_step) {
      int p0, q0;
      tile_at(it, p0, q0);
      const int qt0 = q0 >> 7, qts = min(S::kQTiles, q_row_tiles - qt0);
      const uint32_t bytes = S::kPBytes + S::kQBytes + 1024 * (1 + qts);
      const uint8_t *scale_p = sp + static_cast<size_t>(p0 >> 7) * kts * 512, *scale_q = sq + static_cast<size_t>(qt0) * kts * 512;
      auto load_p = [&](uint8_t* st, uint64_t* full, int kb) {
        mbar_arrive_expect_tx(full, bytes);
        tma_load_2d(st, &tmap_p, full, kb * 128, p0);
        mx4_bulk_load(st + S::kPBytes + S::kQBytes, scale_p + kb * 1024, 1024, full);
      };
      auto load_q = [&](uint8_t* st, uint64_t* full, int kb) {
        tma_load_2d(st + S::kPBytes, &tmap_q, full, kb * 128, q0);
        for (int q = 0; q < qts; ++q)
          mx4_bulk_load(st + S::kPBytes + S::kQBytes + 1024 * (1 + q), scale_q + static_cast<size_t>(q) * kts * 512 + kb * 1024, 1024, full);
      };
      int ahead = 0;
      if (kPieces && it == it0) {      // the first weights are asked for while the kernel before cuts the tokens
        ahead = min(ST, kb1 - kb0);
        if (one)
          for (int i = 0; i < ahead; ++i) load_p(smem + i * S::kStage, &full_bar[i], kb0 + i);
        __syncwarp();
        griddep_wait();
      }
      for (int kb = kb0; kb < kb1; ++kb) {
        const bool first = kb - kb0 < ahead;      // in the first round: nothing to wait for
        if (!__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&empty_bar[s], ph, gave_up, limit.tries);
        if (!ok) break;
        uint8_t* st = smem + s * S::kStage;
        uint64_t* full = &full_bar[s];
        if (++s == ST) {
          s = 0;
          ph ^= 1;
          ++rounds;
        }
        here = mx4_test(&empty_bar[s], ph);
        if (one) {
          if (!first) load_p(st, full, kb);
          load_q(st, full, kb);
        }
        __syncwarp();
      }
    }
    if (kPieces) griddep_wait();      // whatever became of the loads: this kernel does not end before the one before it
    // what was asked for lands before the CTA's memory is given back, whichever warp gave up
    if (lane == 0)
      for (int i = 0; i < ST; ++i) {
        const int round = i < s ? rounds : rounds - 1;
        if (round >= 0) mbar_drain(&full_bar[i], round & 1);
      }
    __syncwarp();
  } else if (warp == kMma) {
    // The whole warp walks the loop and one lane issues: what the instructions are given stays in uniform registers.
    const bool one = elect_one();
    const uint64_t ad0 = make_smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128), bd0 = make_smem_desc(smem_u32(smem) + S::kPBytes, 16, 1024, kLayoutSW128);
    const uint64_t sd0 = make_smem_desc(smem_u32(smem) + S::kPBytes + S::kQBytes, 16, 128, kLayoutNone);
    int s = 0, k = 0;
    uint32_t ph = 0;
    for (int it = it0; it < total && ok; it += it_step, ++k) {
      int p0, q0;
      tile_at(it, p0, q0);
      const uint32_t n = kSwap ? min(BN, (Q - q0 + 15) & ~15) : BN, acc = tmem + (k & 1) * BN;
      const uint32_t idesc = idesc_mx4(kP, n, 0), idesc2 = idesc_mx4(kP, n, 2);
      ok = mx4_warp_wait(&acc_free[k & 1], ((k >> 1) & 1) ^ 1, gave_up, limit.tries);
      uint32_t here = mx4_test(&full_bar[s], ph);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
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
            umma_mx4(acc, ad + 2 * j, bd + 2 * j, j & 1 ? idesc2 : idesc, ts + 4 * (j >> 1), tq + 4 * S::kQTiles * (j >> 1), (kb - kb0) | j ? 1u : 0u);
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
    for (int it = it0; it < total && ok; it += it_step, ++k) {
      int p0, q0;
      tile_at(it, p0, q0);
      // all lanes or none: the TMEM loads need the whole warp
      ok = mx4_warp_wait(&acc_full[k & 1], (k >> 1) & 1, gave_up, limit.tries);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16) + (k & 1) * BN;
      const int row = p0 + quad * 32 + lane, cols = min(BN, Q - q0);
      float* red = reinterpret_cast<float*>(smem);      // [column][128]; a part of a tile is all its CTA has: the stages are done with
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
          if constexpr (!kSwap) {
            mx4_store_row<EPI>(p, x, r, row, q0 + c, wide);
          } else if constexpr (kPieces) {
            float v = r[kPieceRows - 1];      // the smallest first
#pragma unroll
            for (int i = kPieceRows - 2; i >= 0; --i) v += r[i];
            v *= 1.f / (1 << kPieceUnits);
            if (split > 1) {
              red[(c / kPieceRows) * kP + quad * 32 + lane] = v;
            } else {
              const int m = (q0 + c) / kPieceRows;
              if (!isfinite(v) && row < p.N) v = sum_again(static_cast<const __nv_bfloat16*>(p.x) + static_cast<size_t>(m) * p.ldx, p.w_codes, p.w_scales, row, p.K);
              __syncwarp();      // the next TMEM load needs the whole warp
              mx4_store_one<EPI>(p, x, v, m, row, bias);
            }
          } else {
            if (split > 1) {
#pragma unroll
              for (int i = 0; i < 16; ++i) red[(c + i) * kP + quad * 32 + lane] = r[i];
            } else {
              mx4_store_col<EPI>(p, x, r, q0 + c, p.M, row, bias);
            }
          }
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
  if (kSwap && split > 1) {      // every CTA of the cluster adds the parts of its share of the weight rows
    cluster_sync_all();
    int p0, q0;
    tile_at(it0, p0, q0);
    const int cols = kPieces ? min(BN, Q - q0) / kPieceRows : min(BN, Q - q0), m0 = kPieces ? q0 / kPieceRows : q0;
    const bool gated = (p.flags & kGluFlags) != 0;
    const int f0 = kP / 4 * rank / split, f1 = kP / 4 * (rank + 1) / split;      // its rows, by fours
    const uint32_t red = smem_u32(smem);
    const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
    for (int i = tid; i < cols * (f1 - f0); i += kThreads) {
      const int c = i / (f1 - f0), r = 4 * (f0 + i - c * (f1 - f0)), n = p0 + r;
      float4 part[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < split) part[q] = ld_dsmem_v4f(mapa_u32(red + (c * kP + r) * 4, q));
      float z[4] = {part[0].x, part[0].y, part[0].z, part[0].w};
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q < split) {
          z[0] += part[q].x;
          z[1] += part[q].y;
          z[2] += part[q].z;
          z[3] += part[q].w;
        }
      if constexpr (kPieces) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!isfinite(z[j]) && n + j < p.N)
            z[j] = sum_again(static_cast<const __nv_bfloat16*>(p.x) + static_cast<size_t>(m0 + c) * p.ldx, p.w_codes, p.w_scales, n + j, p.K);
      }
      const size_t o = static_cast<size_t>(m0 + c) * p.ldo;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (bias != nullptr && n + j < p.N) z[j] += __bfloat162float(bias[n + j]);
      if (gated) {
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          if (n + j < p.N) out[o + (n + j) / 2] = __float2bfloat16_rn(glu(z[j], z[j + 1], p.flags, x));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) out[o + n + j] = __float2bfloat16_rn(activate(z[j], p.act, x));
      }
    }
    __syncwarp();
    cluster_sync_all();      // the others still read this CTA's parts
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
  volatile int* asked = gave_up + 1;          // [2]: stages whose loads this CTA asked for; in the first one also: the second did

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
  bool ok = !mx4_pair_quits(limit, warp == kTma ? 0 : warp == kMma ? 1 : 3, rank);

  if (warp == kTma) {
    const bool one = elect_one();
    int s = 0, rounds = 0;
    uint32_t ph = 1, here = 1;      // the first round passes
    for (int it = worker; it < total && ok; it += workers) {
      int p0, q0;
      tile_at(it, p0, q0);
      for (int kb = 0; kb < nkb; ++kb) {
        if (!__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&empty_bar[s], ph, gave_up, limit.tries);
        if (!ok) break;
        uint8_t* st = smem + s * kStage;
        uint64_t* full = &full_bar[s];
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
          ++rounds;
        }
        here = mx4_test(&empty_bar[s], ph);
        if (one) {
          const uint32_t bar = mapa_u32(smem_u32(full), 0);
          if (rank == 0) mbar_arrive_expect_tx(full, 2 * kStage);
          tma_load_2d_pair(st, &tmap_p, bar, kb * 128, p0);
          tma_load_2d_pair(st + kPBytes, &tmap_q, bar, kb * 128, q0 + rank * 128);
          tma_load_3d_pair(st + kPBytes + kQBytes, &tmap_sp, bar, 0, 2 * kb, p0 >> 7);
          tma_load_3d_pair(st + kPBytes + kQBytes + 1024, &tmap_sq, bar, 0, 2 * kb, q0 >> 7);
        }
        __syncwarp();
      }
    }
    if (lane == 0) {
      if (!ok) tell();
      asked[0] = rounds * kStages + s;
    }
    __syncwarp();
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
  if (tid == 0) {
    if (rank == 1) st_dsmem_u32(mapa_u32(smem_u32(const_cast<int*>(asked + 1)), 0), asked[0]);
    if (*gave_up) tell();      // both CTAs take the branch below, or neither does
  }
  __syncwarp();
  cluster_sync_all();
  if (*gave_up) {      // otherwise the products have consumed what was asked for, and the epilogues the products
    if (tid == 0) {
      if (rank == 0) mx4_settle_pair(full_bar, kStages, asked[0], asked[1], kStage);
      mbar_drain(drain_bar, 0);
    }
    __syncthreads();
    cluster_sync_all();
  }
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
  VB_ALLOW_SMEM(once, mx4_pair_kernel, static_cast<int>(kSmem));
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

// ---- bf16 tokens to 16 rows of 4-bit numbers each ----
// A warp takes 256 columns of a token, a lane 8.  v is what is left, in units of the row at hand; all steps are exact in fp32.
constexpr int kPieceWarps = 4;
__global__ void __launch_bounds__(32 * kPieceWarps)
mx4_pieces_kernel(const __nv_bfloat16* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int M, int K) {
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, pitch = mx4_pitch(K), kts = mx4_ktiles(K), chunks = kts / 2;
  const int it = blockIdx.x * kPieceWarps + (threadIdx.x >> 5), m = it / chunks, ch = it - m * chunks;
  const int rows = kPieceRows * M, padded = (rows + 127) / 128 * 128;
  if (m * kPieceRows >= padded) return;
  const int c0 = ch * 256 + lane * 8, at = ch * 128 + lane * 4;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (m < M) {
    const __nv_bfloat16* row = x + static_cast<size_t>(m) * ldx;
    if (c0 + 8 <= K && ((reinterpret_cast<uintptr_t>(x) | (ldx * 2)) & 15) == 0) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c0));
      v[0] = bf_lo(a.x); v[1] = bf_hi(a.x); v[2] = bf_lo(a.y); v[3] = bf_hi(a.y);
      v[4] = bf_lo(a.z); v[5] = bf_hi(a.z); v[6] = bf_lo(a.w); v[7] = bf_hi(a.w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c0 + i < K ? __bfloat162float(row[c0 + i]) : 0.f;
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const uint32_t e = top >> 23, unit = e > 2 ? e - 2 : 0u;
  const bool held = unit + kPieceUnits < 255u;
  const uint32_t first = held ? unit + kPieceUnits : 255u;
  const float inv = __uint_as_float((254u - (held ? unit : 0u)) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = held ? v[i] * inv : 0.f;
#pragma unroll 1
  for (int i = 0; i < kPieceRows; ++i) {
    const int r = m * kPieceRows + i;
    // the first row of a block without a scale says so; bytes below 0 do not exist, nor do rows of them
    const uint32_t byte = i == 0 ? first : (held && first >= 2u * i ? first - 2u * i : 0u);
    const bool rest = i == 0 || (held && first >= 2u * i);
    const uint32_t c = rest && m < M ? mx4_encode8(v) : 0u;
    const uint32_t h[4] = {mx4_pair_f16<0>(c), mx4_pair_f16<1>(c), mx4_pair_f16<2>(c), mx4_pair_f16<3>(c)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      v[2 * j] = (v[2 * j] - f.x) * 4.f;
      v[2 * j + 1] = (v[2 * j + 1] - f.y) * 4.f;
    }
    if (m < M && at < pitch) *reinterpret_cast<uint32_t*>(codes + static_cast<size_t>(r) * pitch + at) = c;
    uint32_t word = m < M ? byte << (8 * ((lane >> 2) & 3)) : 0u;
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(r, 2 * ch + (lane >> 4), kts)) = word;
  }
}

template <int BN, bool kSwap, bool kPieces>
int launch(const vila_mx4_linear_params& p, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  using S = Shape<BN>;
  static PerDeviceOnce once;
  VB_ALLOW_SMEM(once, mx4_tc_kernel<BN, kSwap, kPieces>, static_cast<int>(S::kSmem));
  const int pitch = mx4_pitch(p.K), tokens = kPieces ? kPieceRows * p.M : p.M;
  const uint8_t *pc = kSwap ? p.w_codes : p.a_codes, *qc = kSwap ? p.a_codes : p.w_codes;
  const int P = kSwap ? p.N : tokens, Q = kSwap ? tokens : p.N;
  CUtensorMap tp, tq;
  if (int rc = make_tmap_2d_u8(&tp, pc, P, pitch, pitch, kP, 128, 128)) return rc;
  if (int rc = make_tmap_2d_u8(&tq, qc, Q, pitch, pitch, BN, 128, 128)) return rc;
  const long long tiles = static_cast<long long>((P + kP - 1) / kP) * ((Q + BN - 1) / BN), most = static_cast<long long>(S::kPerSm) * num_sms();
  VB_CHECK(tiles < (1LL << 28), "mx4_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  // K over a cluster where the tiles leave SMs idle and K is long: of 14 stages (K = 3584) the cluster's joint end cost what it saved
  static Mx4Clusters clusters;
  const int split = kSwap ? clusters.split(mx4_tc_kernel<BN, kSwap, kPieces>, kThreads, S::kSmem, tiles, (p.K + kDepth - 1) / kDepth / 8) : 1;
  const dim3 grid(static_cast<unsigned>(split > 1 ? tiles * split : (tiles < most ? tiles : most)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (kPieces && pdl_enabled()) {      // behind mx4_pieces_kernel, which lets it begin
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  VB_CUDA(cudaLaunchKernelEx(&cfg, mx4_tc_kernel<BN, kSwap, kPieces>, tp, tq, p, x, split, wait_limit(tries), failed_word()));
  return 0;
}

}  // namespace

int mx4_tc(const vila_mx4_linear_params& p, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "mx4_linear: no pinned host memory for the status word");
  if (p.M <= 16) return launch<16, true, false>(p, x, tries, stream);
  if (p.M <= 32) return launch<32, true, false>(p, x, tries, stream);
  if (p.M <= 64) return launch<64, true, false>(p, x, tries, stream);
  if (p.M <= 128) return launch<128, true, false>(p, x, tries, stream);
  if (p.M > 512) return pair::launch(p, x, tries, stream);
  return launch<128, false, false>(p, x, tries, stream);
}

size_t mx4_pieces_bytes(int M, int K) {
  return static_cast<size_t>(kPieceRows) * M * mx4_pitch(K) + mx4_scale_bytes(kPieceRows * M, K);
}
int mx4_pieces(const vila_mx4_linear_params& given, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "mx4_linear: no pinned host memory for the status word");
  vila_mx4_linear_params p = given;
  uint8_t* codes = static_cast<uint8_t*>(p.scratch);
  uint8_t* scales = codes + static_cast<size_t>(kPieceRows) * p.M * mx4_pitch(p.K);
  const long long items = static_cast<long long>((kPieceRows * p.M + 127) / 128 * 128 / kPieceRows) * (mx4_ktiles(p.K) / 2);
  VB_CUDA(launch_serial(mx4_pieces_kernel, dim3(static_cast<unsigned>((items + kPieceWarps - 1) / kPieceWarps)), dim3(32 * kPieceWarps), 0, stream,
                        static_cast<const __nv_bfloat16*>(p.x), p.ldx, codes, scales, p.M, p.K));
  p.a_codes = codes;
  p.a_scales = scales;
  const int rows = kPieceRows * p.M;
  if (rows <= 16) return launch<16, true, true>(p, x, tries, stream);
  if (rows <= 32) return launch<32, true, true>(p, x, tries, stream);
  if (rows <= 64) return launch<64, true, true>(p, x, tries, stream);
  return launch<128, true, true>(p, x, tries, stream);
}

}  // namespace vb
