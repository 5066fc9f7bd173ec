// Linear layers of many 8-bit rows (fp8.cuh): tiles of 256 tokens x 256 weight rows by CTA pairs (tcgen05.mma cta_group::2, kind::f8f6f4).
//
// A pair's CTAs stage half the tokens and half the weight rows each, 64 bytes of operands per clock of products, where a single CTA's tile
// of 128 x 128 asks for 128, which is all that shared memory gives.  Each CTA's TMEM holds two accumulators of its 128 tokens by 256
// columns: while the tensor core sums a block of 128 columns into one, eight epilogue warps fetch the other, multiply by the block's
// scales and add to their sums in registers: a lane is a token, a warp's 128 columns are one block of weight rows, so that a thread's scale is one
// number a block.  A block's products take 512 clocks at least, its 32768 sums a CTA 256 clocks of TMEM reads and as many of fp32
// instructions, and what a warp does for a block one after another some 900 - 1000: a wait 150 - 250 even if it is over, 16 columns of
// TMEM 70.
//
// 2048 x 37888 x 3584 runs at 1.71 PFLOP/s over seconds, 8192 x 8192 x 8192 at 1.84, both at some 1.5 - 1.6 GHz under the power limit (a copy that
// fetched no sums, for timing: 2.05 and 2.21, so that at most a fifth is left).  Tried and slower or even: registers moved to the
// epilogue (by 8 %), 16 epilogue warps, 32 columns a TMEM load, scales staged by warps of their own, lane 0 alone polling (116 us for 75).
//
// A result in 8 bits is made in the epilogue: a thread has 128 columns of a row, a block of it, or behind a gated unit half a block, and learns
// the other half's largest magnitude from the warp that has it.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "fp8.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"
#include "mx4.cuh"
#include "mx4_epi.cuh"

namespace vb {
namespace {

constexpr int kN = 256, kStages = 6;
constexpr int kEpi = 8, kTma = kEpi, kMma = kEpi + 1, kThreads = 32 * (kEpi + 2);
constexpr int kPBytes = 128 * 128, kQBytes = 128 * 128, kStage = kPBytes + kQBytes;
constexpr int kAhead = 4;                     // blocks that a token's scales are asked for ahead
constexpr int kGroup = 8;                     // token tiles that the pairs go through side by side
constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStage + 2 * kN * 4 + 256;
static_assert(kSmem <= 227 * 1024, "");

__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The tile that comes `it`-th.  Token tiles go in groups of kGroup, and within a group the tiles that run together share weight rows and
// tokens: 74 pairs at a time read some 8 token tiles and 9 of weight rows, which stay in L2, not all tokens for every weight tile.
__device__ __forceinline__ void tile_at(int it, int p_tiles, int q_tiles, int& pt, int& qt) {
  const int g = it / (kGroup * q_tiles), first = g * kGroup, size = min(kGroup, p_tiles - first), i = it - first * q_tiles;
  qt = i / size;
  pt = first + i - qt * size;
}

__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const vila_fp8_linear_params p,
                const vila_glinear_ext x, const WaitLimit limit, volatile unsigned int* failed) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint32_t* tops = reinterpret_cast<uint32_t*>(smem + kStages * kStage);      // [2][half][128]: largest magnitudes of half a block
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(tops + 2 * kN);            // the first CTA's: both CTAs' loads
  uint64_t* done_bar = full_bar + kStages;    // a stage's products are summed: it may be loaded anew, and the accumulator fetched
  uint64_t* acc_free = done_bar + kStages;    // [2], the first CTA's: fetched in both CTAs
  uint64_t* top_bar = acc_free + 2;           // [4]: both halves' magnitudes of 32 tokens are there
  uint64_t* drain_bar = top_bar + 4;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* gave_up = reinterpret_cast<int*>(tmem_ptr + 1);
  volatile int* asked = gave_up + 1;          // [2]: stages whose loads this CTA asked for; in the first one also: the second did

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = static_cast<int>(cluster_ctarank());
  const int p_tiles = (p.M + 255) / 256, q_tiles = (p.N + kN - 1) / kN, total = p_tiles * q_tiles;
  const int worker = blockIdx.x >> 1, workers = gridDim.x >> 1, nkb = fp8_blocks(p.K);

  if (tid == 0) {
    tma_prefetch_desc(&tmap_p);
    tma_prefetch_desc(&tmap_q);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&done_bar[i], 1);
    }
    mbar_init(&acc_free[0], 2 * kEpi);
    mbar_init(&acc_free[1], 2 * kEpi);
    for (int i = 0; i < 4; ++i) mbar_init(&top_bar[i], 2);
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
      int pt, qt;
      tile_at(it, p_tiles, q_tiles, pt, qt);
      const int p0 = pt * 256 + rank * 128, q0 = qt * kN + rank * 128;
      for (int kb = 0; kb < nkb; ++kb) {
        if (!__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&done_bar[s], ph, gave_up, limit.tries);
        if (!ok) break;
        uint8_t* st = smem + s * kStage;
        uint64_t* full = &full_bar[s];
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
          ++rounds;
        }
        here = mx4_test(&done_bar[s], ph);
        if (one) {
          const uint32_t bar = mapa_u32(smem_u32(full), 0);
          if (rank == 0) mbar_arrive_expect_tx(full, 2 * kStage);
          tma_load_2d_pair(st, &tmap_p, bar, kb * 128, p0);
          tma_load_2d_pair(st + kPBytes, &tmap_q, bar, kb * 128, q0);
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
      constexpr uint32_t idesc = fp8_idesc(256, kN);
      int s = 0, a = 0;
      uint32_t ph = 0, aph = 1;      // the first round of accumulators passes
      uint32_t here = 0, free = 1;
      for (int it = worker; it < total && ok; it += workers) {
        for (int kb = 0; kb < nkb; ++kb) {
          if (!__all_sync(0xffffffffu, free)) ok = mx4_warp_wait(&acc_free[a], aph, gave_up, limit.tries);
          if (ok && !__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&full_bar[s], ph, gave_up, limit.tries);
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = ad0 + s * (kStage >> 4), bd = bd0 + s * (kStage >> 4);
          const uint32_t acc = tmem + a * kN;
          uint64_t* done = &done_bar[s];
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
          if (++a == 2) {
            a = 0;
            aph ^= 1;
          }
          here = mx4_test(&full_bar[s], ph);
          free = mx4_test(&acc_free[a], aph);
          if (one) {      // columns past K are zeros on both sides
#pragma unroll
            for (int i = 0; i < 4; ++i) umma(acc, ad + 2 * i, bd + 2 * i, idesc, i != 0);
            umma_commit_pair(done);
          }
          __syncwarp();
        }
      }
      if (!ok && lane == 0) tell();
      if (one) umma_commit_pair(drain_bar);      // reports to both CTAs
    }
    // products under way, and what they report to this CTA, end before TMEM and the CTA's memory are given back
    if (lane == 0 && !mbar_wait_limited(drain_bar, 0, gave_up, limit.tries)) mbar_drain(drain_bar, 0);
    __syncwarp();
  } else {
    const int quad = warp & 3, half = warp >> 2;      // its lanes of TMEM, its 128 columns
    const bool wide = reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.ldo % 16 == 0;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * 128;
    const uint32_t free_bar = mapa_u32(smem_u32(acc_free), 0);
    const int w_blocks = fp8_blocks(p.N);
    int s = 0, a = 0, k = 0;
    uint32_t ph = 0;
    for (int it = worker; it < total && ok; it += workers, ++k) {
      int pt, qt;
      tile_at(it, p_tiles, q_tiles, pt, qt);
      const int m = pt * 256 + rank * 128 + quad * 32 + lane, n0 = qt * kN + half * 128;
      const float* sa = p.a_scales + (m < p.M ? m : 0);
      const float* sw = p.w_scales + min(n0 / kFp8Block, w_blocks - 1) * p.ld_ws;
      float z[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) z[i] = 0.f;
      float sa_now[kAhead], sa_next[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) sa_now[j] = j < nkb ? sa[j * p.ld_as] : 0.f;
      float w_now = lane < nkb ? sw[lane] : 0.f;      // of 32 blocks, one a lane
      // a block's factor, and whether any lane's is wide: made while the block before is fetched from TMEM (in line with it the test took 3 - 4 %)
      float both = fp8_both_scales(sa_now[0], __shfl_sync(0xffffffffu, w_now, 0));
      bool any_wide = __any_sync(0xffffffffu, fp8_is_wide(both));
#pragma unroll 1
      for (int kb = 0; kb < nkb && ok; kb += kAhead) {
        float w_next = w_now;
        if (((kb + kAhead) & 31) == 0) w_next = kb + kAhead + lane < nkb ? sw[kb + kAhead + lane] : 0.f;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) sa_next[j] = kb + kAhead + j < nkb ? sa[(kb + kAhead + j) * p.ld_as] : 0.f;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (kb + j < nkb && ok) {
            ok = mx4_warp_wait(&done_bar[s], ph, gave_up, limit.tries);
            if (ok) {
              tc_fence_after();
              if (any_wide) fp8_widen(lanes + a * kN, 128, [&](int) { return both; });
              float r[2][16];
              tmem_ld_32x32b_x16(lanes + a * kN, reinterpret_cast<uint32_t*>(r[0]));
              const float both_next = fp8_both_scales(j + 1 < kAhead ? sa_now[(j + 1) % kAhead] : sa_next[0],
                                                      __shfl_sync(0xffffffffu, j + 1 < kAhead ? w_now : w_next, (kb + j + 1) & 31));
              any_wide = __any_sync(0xffffffffu, fp8_is_wide(both_next));
#pragma unroll
              for (int c = 0; c < 8; ++c) {      // a chunk is fetched under the sums of the one before
                tmem_ld_wait();
                if (c < 7) tmem_ld_32x32b_x16(lanes + a * kN + 16 * (c + 1), reinterpret_cast<uint32_t*>(r[(c + 1) & 1]));
#pragma unroll
                for (int i = 0; i < 16; i += 2) fp8_fma2(z[16 * c + i], z[16 * c + i + 1], r[c & 1][i], r[c & 1][i + 1], both, both);
              }
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster_relaxed(free_bar + 8 * a);
              a ^= 1;
              if (++s == kStages) {
                s = 0;
                ph ^= 1;
              }
              both = both_next;
            }
          }
        }
        w_now = w_next;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) sa_now[j] = sa_next[j];
      }
      if (!ok) break;
      if (p.o_codes == nullptr) {
        mx4_with_epilogue(p, [&](auto epi) {
          constexpr int EPI = decltype(epi)::value;
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            float r[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = z[c + i];
            if (n0 + c < p.N) mx4_store_row<EPI>(p, x, r, m, n0 + c, wide);
          }
        });
      } else {
        if (p.bias != nullptr) {
          const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
#pragma unroll
          for (int i = 0; i < 128; ++i) z[i] += n0 + i < p.N ? __bfloat162float(bias[n0 + i]) : 0.f;
        }
        mx4_with_epilogue(p, [&](auto epi) {
          constexpr int EPI = decltype(epi)::value;
          constexpr bool kGated = EPI >= kMx4Gated;
          constexpr int kOut = kGated ? 64 : 128;
          const int cols = kGated ? p.N / 2 : p.N, o0 = kGated ? n0 / 2 : n0;      // of the result, this thread's first
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < kOut; ++i) {
            const float v = kGated ? mx4_glu<EPI>(z[2 * i % 128], z[(2 * i + 1) % 128], x) : mx4_act<EPI, true>(z[i], x);
            z[i] = o0 + i < cols ? v : 0.f;
            top = max(top, __float_as_uint(z[i]) & 0x7fffffffu);
          }
          if constexpr (kGated) {
            uint32_t* mine = tops + (k & 1) * kN + half * 128 + quad * 32 + lane;
            *mine = top;
            __syncwarp();
            if (lane == 0) mbar_arrive(&top_bar[quad]);
            ok = mx4_warp_wait(&top_bar[quad], k & 1, gave_up, limit.tries);
            top = max(top, tops[(k & 1) * kN + (half ^ 1) * 128 + quad * 32 + lane]);
          }
          const Fp8Scale e = fp8_scale(top);
          if (ok && m < p.M && o0 < cols) {
            uint8_t* to = static_cast<uint8_t*>(p.o_codes) + static_cast<int64_t>(m) * p.ld_oc + o0;
#pragma unroll
            for (int i = 0; i < kOut; i += 16) {
              float v[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = z[i + j];
              if (o0 + i < cols) stg_v4(to + i, fp8_encode16(v, e));      // a row's codes have room for whole chunks
            }
            if (!kGated || half == 0) p.o_scales[static_cast<int64_t>(o0 / kFp8Block) * p.ld_os + m] = e.scale;
          }
        });
      }
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

}  // namespace

// By rounds through the GPU, rows of padding counted as rows; measured at 3584 columns only.  There a round of pairs takes 17.5 us, one of single CTAs'
// tiles of 128 x 128 (fp8_tc.cu) 13.4, us against us:
// 600 rows of 1152 weight rows 19.6 and 11.6, 512 of 4608 20.5 and 14.7 (one round each), 600 of 4608 20.8 and 26.7 (one and two), 300 of 18944
// 39.3 and 43.5, 1536 of 3584 37.2 and 40.5 (two and three), 1024 of 18944 73.6 and 112.8.
bool fp8_pair_takes(const vila_fp8_linear_params& p) {
  if (p.M <= 128) return false;
  const long long sms = num_sms(), singles = ((p.M + 127ll) / 128 * ((p.N + 127) / 128) + sms - 1) / sms;
  const long long pairs = ((p.M + 255ll) / 256 * ((p.N + kN - 1) / kN) + sms / 2 - 1) / (sms / 2);
  return 4 * pairs < 3 * singles;
}

int fp8_pair(const vila_fp8_linear_params& p, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "fp8_linear: no pinned host memory for the status word");
  static PerDeviceOnce once;
  VB_ALLOW_SMEM(once, fp8_pair_kernel, static_cast<int>(kSmem));
  CUtensorMap ta, tw;
  if (int rc = make_tmap_2d_u8(&ta, p.a_codes, p.M, p.K, p.lda, 128, 128, 128)) return rc;
  if (int rc = make_tmap_2d_u8(&tw, p.w_codes, p.N, p.K, p.ldw, 128, 128, 128)) return rc;
  const long long tiles = static_cast<long long>((p.M + 255) / 256) * ((p.N + kN - 1) / kN), most = num_sms() / 2;
  VB_CHECK(tiles < (1LL << 27), "fp8_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  VB_CUDA(launch_serial(fp8_pair_kernel, dim3(static_cast<unsigned>(2 * (tiles < most ? tiles : most))), dim3(kThreads), kSmem, stream, ta, tw, p, x,
                        wait_limit(tries), failed_word()));
  return 0;
}

}  // namespace vb
