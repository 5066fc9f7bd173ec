// Linear layers on 8-bit rows with a scale per block of 128 columns (fp8.cuh), on the tensor cores: tcgen05.mma kind::f8f6f4.
//
//   z[m, n] = sum over blocks b of sa[m, b] sw[n / 128, b] * (sum over the block's 128 columns of a[m, k] w[n, k])
//
// A block's products are summed by the tensor core into an accumulator of their own in TMEM; the epilogue warps fetch it, multiply by
// both scales and add to their sums in registers, in fp32, while the tensor core is at the next blocks.
//
//   TMA warp        a stage: one block (128 bytes) of the tile's weight rows and of its tokens, 128-byte swizzle
//   MMA warp        TMEM allocation; four tcgen05.mma of 32 columns a stage, into one of four accumulators
//   scale warp      the products of both scales, a group of blocks at a time, into shared memory
//   epilogue warps  two blocks at a time: scales times accumulators, added up; behind the last: bias, activation, gated unit, result
//
// Weight rows are the 128 lanes of a tile, tokens its columns (at most BN): few tokens cost few columns.  A tile's weight rows are one block
// row, so that sw is one number a block; the products are one number a column.  What an epilogue warp does one after another for
// a block is the bound where tokens are many (a wait takes it 150 - 250 clocks even if it is over, 16 columns of TMEM 70, so that it
// waits once for two blocks and finds the scales ready made); where they are few it is memory.  Where the tiles leave SMs idle K is
// split over a cluster of up to 8 CTAs, whose sums are added in rank order through distributed shared memory.
//
// A launch may begin before the one before it has ended: the first weights are asked for while that one ends, everything else comes behind
// griddepcontrol.wait.  (Weights come from launches that do not let others begin early.)
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "fp8.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"
#include "mx4.cuh"
#include "mx4_epi.cuh"

namespace vb {
namespace {

constexpr int kRows = 128;                    // weight rows of a tile
constexpr int kAcc = 4, kVisit = 2;            // accumulators in TMEM, and how many of them change hands together
constexpr int kTogether = 8;                  // blocks whose scales change hands together
static_assert(kTogether % kVisit == 0 && kAcc == 2 * kVisit, "");

__device__ __forceinline__ void umma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
template <int BN> struct Shape {
  static constexpr int kEpi = BN > 64 ? 8 : 4;                  // epilogue warps: a quarter of the lanes each; two share a quarter's columns
  static constexpr int kTma = kEpi, kMma = kEpi + 1, kScale = kEpi + 2, kThreads = 32 * (kEpi + 3);
  static constexpr int kColumns = BN > 64 ? BN / 2 : BN;        // columns of a thread
  static constexpr int kPBytes = kRows * 128, kQBytes = BN * 128, kStage = kPBytes + kQBytes;
  static constexpr int kStages = BN == 16 ? 6 : (BN == 32 ? 5 : (BN == 64 ? 4 : 6));
  static constexpr int kPerSm = BN > 64 ? 1 : 2;
  static constexpr int kCols = kAcc * BN;                        // of TMEM
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStage + 2 * kTogether * BN * 4 + 256;
  static_assert(kCols == 64 || kCols == 128 || kCols == 256 || kCols == 512, "TMEM");
  static_assert(kCols * kPerSm <= 512, "TMEM of an SM");
  static_assert((kSmem + 1024) * kPerSm <= 228 * 1024, "shared memory");
  static_assert(kRows * BN * 4 <= kStages * kStage, "the sums of a cluster's CTA");
};

// What becomes of the sums of one weight row n (a lane's), tokens m .. m + 15 below `end`.  All lanes call it.  out32: unrounded, rows of
// ld32 columns.
template <int EPI>
__device__ __forceinline__ void store_col(const vila_fp8_linear_params& p, const vila_glinear_ext& x, float* out32, int ld32, const float* r, int m, int end,
                                          int n, float bias) {
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  auto put = [&](int row, int col, float v) {
    if (out32 != nullptr) out32[static_cast<size_t>(row) * ld32 + col] = v;
    else out[static_cast<size_t>(row) * p.ldo + col] = __float2bfloat16_rn(v);
  };
  if constexpr (EPI >= kMx4Gated) {
    const bool odd = (n & 1) != 0;      // the lanes of a pair hold gate and up: of two tokens each lane finishes one
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float za = r[i] + bias, zb = r[i + 1] + bias, other = __shfl_xor_sync(0xffffffffu, odd ? za : zb, 1);
      const int row = m + i + (odd ? 1 : 0);
      if (n < p.N && row < end) put(row, n / 2, mx4_glu<EPI>(odd ? other : za, odd ? zb : other, x));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n < p.N && m + i < end) put(m + i, n, mx4_act<EPI>(r[i] + bias, x));
  }
}

// bn: tokens of a tile, a multiple of 16, at most BN.  split: CTAs of a cluster, which share a tile and cut K.
template <int BN>
__global__ void __launch_bounds__(Shape<BN>::kThreads, Shape<BN>::kPerSm)
fp8_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a, const vila_fp8_linear_params p, const vila_glinear_ext x,
           float* out32, const int bn, const int split, const WaitLimit limit, volatile unsigned int* failed) {
  using S = Shape<BN>;
  constexpr int ST = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* scales = reinterpret_cast<float*>(smem + ST * S::kStage);      // [2][kTogether][BN]: both scales of a token's block
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(scales + 2 * kTogether * BN);
  uint64_t* empty_bar = full_bar + ST;
  uint64_t* acc_full = empty_bar + ST;   // [2]: of up to kVisit blocks
  uint64_t* acc_free = acc_full + 2;     // [2]
  uint64_t* scale_full = acc_free + 2;   // [2]: of up to kTogether blocks
  uint64_t* scale_free = scale_full + 2; // [2]
  uint64_t* drain_bar = scale_free + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* gave_up = reinterpret_cast<int*>(tmem_ptr + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int p_tiles = (p.N + kRows - 1) / kRows, q_tiles = (p.M + bn - 1) / bn, total = p_tiles * q_tiles;
  const int nkb = fp8_blocks(p.K);
  const int rank = static_cast<int>(blockIdx.x) % split, it0 = static_cast<int>(blockIdx.x) / split, it_step = static_cast<int>(gridDim.x) / split;
  const int kb0 = static_cast<int>(static_cast<long long>(nkb) * rank / split), kb1 = static_cast<int>(static_cast<long long>(nkb) * (rank + 1) / split);
  auto tile_at = [&](int it, int& p0, int& q0) {     // the tiles that run together share their tokens
    const int qt = it / p_tiles;
    p0 = (it - qt * p_tiles) * kRows;
    q0 = qt * bn;
  };

  griddep_launch_dependents();
  if (tid == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_a);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], S::kEpi);
      mbar_init(&scale_full[i], 1);
      mbar_init(&scale_free[i], S::kEpi);
    }
    mbar_init(drain_bar, 1);
    *gave_up = 0;
    fence_barrier_init();
  }
  if (warp == S::kMma) tmem_alloc<S::kCols>(tmem_ptr);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  bool ok = true;
  if (limit.quits >= 0) {
    ok = limit.quits != (warp == S::kTma ? 0 : warp == S::kMma ? 1 : warp == S::kScale ? 2 : 3);
    if (!ok) *gave_up = 1;
  }

  if (warp == S::kTma) {
    const bool one = elect_one();
    int s = 0, rounds = 0;                // stage, rounds through all of them
    uint32_t ph = 1;                      // parity to wait for on an empty barrier: the first round passes
    const uint32_t bytes = S::kPBytes + bn * 128;
    int ahead = 0;                        // stages of the first tile whose weights are asked for before the launch before has ended
    if (ok && it0 < total) {
      int p0, q0;
      tile_at(it0, p0, q0);
      ahead = min(ST, kb1 - kb0);
      if (one)
        for (int i = 0; i < ahead; ++i) {
          mbar_arrive_expect_tx(&full_bar[i], bytes);
          tma_load_2d(smem + i * S::kStage, &tmap_w, &full_bar[i], (kb0 + i) * 128, p0);
        }
      __syncwarp();
    }
    griddep_wait();
    for (int it = it0; it < total && ok; it += it_step) {
      int p0, q0;
      tile_at(it, p0, q0);
      for (int kb = kb0; kb < kb1; ++kb) {
        const bool first = it == it0 && kb - kb0 < ahead;      // in the first round: nothing to wait for
        if (!first) ok = mx4_warp_wait(&empty_bar[s], ph, gave_up, limit.tries);
        if (!ok) break;
        if (one) {
          uint8_t* st = smem + s * S::kStage;
          if (!first) {
            mbar_arrive_expect_tx(&full_bar[s], bytes);
            tma_load_2d(st, &tmap_w, &full_bar[s], kb * 128, p0);
          }
          tma_load_2d(st + S::kPBytes, &tmap_a, &full_bar[s], kb * 128, q0);
        }
        __syncwarp();
        if (++s == ST) {
          s = 0;
          ph ^= 1;
          ++rounds;
        }
      }
    }
    // what was asked for lands before the CTA's memory is given back, whichever warp gave up
    if (lane == 0)
      for (int i = 0; i < ST; ++i) {
        const int round = i < s ? rounds : rounds - 1;
        if (round >= 0) mbar_drain(&full_bar[i], round & 1);
      }
    __syncwarp();
  } else if (warp == S::kMma) {
    // The whole warp walks the loop and one lane issues: what the instructions are given stays in uniform registers.
    const bool one = elect_one();
    const uint64_t pd0 = make_smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128), qd0 = make_smem_desc(smem_u32(smem) + S::kPBytes, 16, 1024, kLayoutSW128);
    const uint32_t idesc = fp8_idesc(kRows, bn);
    int s = 0, v = 0;                     // stage, visits of the epilogue warps so far
    uint32_t ph = 0;
    for (int it = it0; it < total && ok; it += it_step) {
      for (int kb = kb0; kb < kb1 && ok; kb += kVisit, ++v) {
        ok = mx4_warp_wait(&acc_free[v & 1], ((v >> 1) & 1) ^ 1, gave_up, limit.tries);      // the first two pass
        for (int i = 0; i < kVisit && kb + i < kb1 && ok; ++i) {
          ok = mx4_warp_wait(&full_bar[s], ph, gave_up, limit.tries);
          if (!ok) break;
          tc_fence_after();
          if (one) {      // columns past K are zeros on both sides
            const uint64_t pd = pd0 + s * (S::kStage >> 4), qd = qd0 + s * (S::kStage >> 4);
            const uint32_t acc = tmem + ((v & 1) * kVisit + i) * BN;
#pragma unroll
            for (int j = 0; j < 4; ++j) umma_fp8(acc, pd + 2 * j, qd + 2 * j, idesc, j != 0);
            umma_commit(&empty_bar[s]);
            if (i + 1 == kVisit || kb + i + 1 == kb1) umma_commit(&acc_full[v & 1]);
          }
          __syncwarp();
          if (++s == ST) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
    if (one) umma_commit(drain_bar);             // products under way end before TMEM and the CTA's memory are given back, too
    if (lane == 0) mbar_drain(drain_bar, 0);
    __syncwarp();
  } else if (warp == S::kScale) {
    griddep_wait();
    // a lane takes four tokens; a row of scales is a multiple of 4 long, and behind the last token nothing counts
    int g = 0;
    for (int it = it0; it < total && ok; it += it_step) {
      int p0, q0;
      tile_at(it, p0, q0);
      const bool there = lane * 4 < bn && q0 + lane * 4 < p.ld_as;
      const float* sa = p.a_scales + (there ? q0 + lane * 4 : 0);
      const float* sw = p.w_scales + (p0 / kRows) * p.ld_ws;
      for (int kb = kb0; kb < kb1; kb += kTogether, ++g) {
        float4 a[kTogether];
        float w[kTogether];
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          const bool in = there && kb + i < kb1;
          a[i] = in ? __ldg(reinterpret_cast<const float4*>(sa + (kb + i) * p.ld_as)) : make_float4(0.f, 0.f, 0.f, 0.f);
          w[i] = in ? __ldg(sw + kb + i) : 0.f;
        }
        ok = mx4_warp_wait(&scale_free[g & 1], ((g >> 1) & 1) ^ 1, gave_up, limit.tries);      // the first two pass
        if (!ok) break;
        if (lane * 4 < BN) {
#pragma unroll
          for (int i = 0; i < kTogether; ++i)
            *reinterpret_cast<float4*>(scales + ((g & 1) * kTogether + i) * BN + lane * 4) =
                make_float4(fp8_both_scales(a[i].x, w[i]), fp8_both_scales(a[i].y, w[i]), fp8_both_scales(a[i].z, w[i]), fp8_both_scales(a[i].w, w[i]));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&scale_full[g & 1]);
      }
    }
  } else {
    griddep_wait();
    const int quad = warp & 3, c0 = (warp >> 2) * S::kColumns;      // its lanes of TMEM, its columns
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16) + c0;
    const int ld32 = p.flags & kGluFlags ? p.N / 2 : p.N;
    constexpr int kChunks = S::kColumns / 16;
    int v = 0, g = 0;                     // visits, groups of blocks so far
    for (int it = it0; it < total && ok; it += it_step) {
      int p0, q0;
      tile_at(it, p0, q0);
      float sum[S::kColumns];
#pragma unroll
      for (int i = 0; i < S::kColumns; ++i) sum[i] = 0.f;
#pragma unroll 1
      for (int kb = kb0; kb < kb1; kb += kVisit, ++v) {
        const int in_group = (kb - kb0) % kTogether;
        if (in_group == 0) {
          if (kb > kb0) {      // all lanes have read the group before: the warp has met since
            if (lane == 0) mbar_arrive(&scale_free[g & 1]);
            ++g;
          }
          ok = mx4_warp_wait(&scale_full[g & 1], (g >> 1) & 1, gave_up, limit.tries);
          if (!ok) break;
        }
        ok = mx4_warp_wait(&acc_full[v & 1], (v >> 1) & 1, gave_up, limit.tries);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < kVisit; ++i) {
          if (kb + i < kb1) {
            const float4* both = reinterpret_cast<const float4*>(scales + ((g & 1) * kTogether + in_group + i) * BN + c0);
            const uint32_t from = lanes + ((v & 1) * kVisit + i) * BN;
            float r[2][16];
            tmem_ld_32x32b_x16(from, reinterpret_cast<uint32_t*>(r[0]));
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {      // a chunk is fetched under the sums of the one before
              tmem_ld_wait();
              if (c + 1 < kChunks) tmem_ld_32x32b_x16(from + 16 * (c + 1), reinterpret_cast<uint32_t*>(r[(c + 1) & 1]));
              float* z = sum + 16 * c;
              const float* n = r[c & 1];
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const float4 f = both[4 * c + j / 4];
                fp8_fma2(z[j], z[j + 1], n[j], n[j + 1], f.x, f.y);
                fp8_fma2(z[j + 2], z[j + 3], n[j + 2], n[j + 3], f.z, f.w);
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_free[v & 1]);
      }
      if (!ok) break;
      if (lane == 0) mbar_arrive(&scale_free[g & 1]);
      ++g;
      const int n = p0 + quad * 32 + lane;
      if (split > 1) {      // a part of a tile is all its CTA has: the stages are done with
        float* red = reinterpret_cast<float*>(smem);      // [column][128]
#pragma unroll
        for (int i = 0; i < S::kColumns; ++i) red[(c0 + i) * kRows + quad * 32 + lane] = sum[i];
      } else {
        const float bias = p.bias != nullptr && n < p.N ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]) : 0.f;
        const int end = min(p.M, q0 + bn);
        mx4_with_epilogue(p, [&](auto epi) {
          constexpr int EPI = decltype(epi)::value;
#pragma unroll
          for (int c = 0; c < S::kColumns; c += 16) store_col<EPI>(p, x, out32, ld32, sum + c, q0 + c0 + c, end, n, bias);
        });
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == S::kMma) {
    tc_fence_after();
    tmem_dealloc<S::kCols>(tmem);
  }
  if (split > 1) {      // every CTA of the cluster adds the parts of its share of the weight rows
    cluster_sync_all();
    int p0, q0;
    tile_at(it0, p0, q0);
    const int cols = min(bn, p.M - q0);
    const bool gated = (p.flags & kGluFlags) != 0;
    const int ld32 = gated ? p.N / 2 : p.N;
    const int f0 = kRows / 4 * rank / split, f1 = kRows / 4 * (rank + 1) / split;      // its rows, by fours
    const uint32_t red = smem_u32(smem);
    const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
    auto put = [&](int row, int col, float v) {
      if (out32 != nullptr) out32[static_cast<size_t>(row) * ld32 + col] = v;
      else out[static_cast<size_t>(row) * p.ldo + col] = __float2bfloat16_rn(v);
    };
    for (int i = tid; i < cols * (f1 - f0); i += S::kThreads) {
      const int c = i / (f1 - f0), r = 4 * (f0 + i - c * (f1 - f0)), n = p0 + r;
      float4 part[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < split) part[q] = ld_dsmem_v4f(mapa_u32(red + (c * kRows + r) * 4, q));
      float z[4] = {part[0].x, part[0].y, part[0].z, part[0].w};
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q < split) {
          z[0] += part[q].x;
          z[1] += part[q].y;
          z[2] += part[q].z;
          z[3] += part[q].w;
        }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (bias != nullptr && n + j < p.N) z[j] += __bfloat162float(bias[n + j]);
      if (gated) {
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          if (n + j < p.N) put(q0 + c, (n + j) / 2, glu(z[j], z[j + 1], p.flags, x));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) put(q0 + c, n + j, activate(z[j], p.act, x));
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

template <int BN>
int launch(const vila_fp8_linear_params& p, const vila_glinear_ext& x, float* out32, int tries, cudaStream_t stream) {
  using S = Shape<BN>;
  static PerDeviceOnce once;
  VB_ALLOW_SMEM(once, fp8_kernel<BN>, static_cast<int>(S::kSmem));
  // as many token tiles as BN makes, all as wide as the widest has to be
  const int q_tiles = (p.M + BN - 1) / BN, bn = ((p.M + q_tiles - 1) / q_tiles + 15) / 16 * 16;
  CUtensorMap tw, ta;
  if (int rc = make_tmap_2d_u8(&tw, p.w_codes, p.N, p.K, p.ldw, kRows, 128, 128)) return rc;
  if (int rc = make_tmap_2d_u8(&ta, p.a_codes, p.M, p.K, p.lda, bn, 128, 128)) return rc;
  const long long tiles = static_cast<long long>((p.N + kRows - 1) / kRows) * ((p.M + bn - 1) / bn), most = static_cast<long long>(S::kPerSm) * num_sms();
  VB_CHECK(tiles < (1LL << 28), "fp8_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  static Mx4Clusters clusters;
  const int split = clusters.split(fp8_kernel<BN>, S::kThreads, S::kSmem, tiles, fp8_blocks(p.K) / 4);
  const dim3 grid(static_cast<unsigned>(split > 1 ? tiles * split : (tiles < most ? tiles : most)));
  VB_CUDA(launch_pdl_cluster(fp8_kernel<BN>, grid, dim3(S::kThreads), S::kSmem, stream, dim3(split), tw, ta, p, x, out32, bn, split, wait_limit(tries),
                                failed_word()));
  return 0;
}

}  // namespace

int fp8_tc(const vila_fp8_linear_params& p, const vila_glinear_ext& ext, float* out32, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "fp8_linear: no pinned host memory for the status word");
  if (p.M <= 16) return launch<16>(p, ext, out32, tries, stream);
  if (p.M <= 32) return launch<32>(p, ext, out32, tries, stream);
  if (p.M <= 64) return launch<64>(p, ext, out32, tries, stream);
  return launch<128>(p, ext, out32, tries, stream);
}

}  // namespace vb
