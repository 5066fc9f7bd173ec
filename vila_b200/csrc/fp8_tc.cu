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
//   epilogue warps  two blocks at a time: scales times accumulators, added up
//
// Up to 32 tokens (kSwap): weight rows are the 128 lanes of a tile, tokens its 16 or 32 columns; bound by the weights' bytes.  More tokens: these are the lanes, 64 or 128 weight rows the columns, so that a thread's scale is one number a block (as one a column
// it took four loads from shared memory per 16 columns, in line with the loads from TMEM: 0.43 us a block instead of 0.3).  There a block
// costs what an epilogue warp does for it one after another: a wait takes 150 - 250 clocks even if it is over, 16 columns of TMEM 70.
//
// A CTA takes one tile, or, where the tiles leave SMs idle, a share of its blocks: a cluster of up to 8 CTAs splits K, every CTA sends
// its sums to the CTAs that finish them, by rows, and these add them in rank order.
//
// A launch may begin before the one before it has ended: TMEM is asked for while that one ends, and so are the first weights where the caller says
// that the host has waited for what wrote them (VILA_FLAG_STATIC_W).  Everything else comes behind griddepcontrol.wait: that alone promises that
// what the launch before wrote can be seen, even where that one lets none begin before its own end.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "fp8.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"
#include "mx4.cuh"
#include "mx4_epi.cuh"

namespace vb {
namespace {

constexpr int kRows = 128;                    // lanes of a tile
constexpr int kAcc = 4, kVisit = 2;            // accumulators in TMEM, and how many of them change hands together
static_assert(kAcc == 2 * kVisit, "");

__device__ __forceinline__ void umma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void st_dsmem_f32(uint32_t cluster_addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <int BN, bool kSwap> struct Shape {
  static constexpr int kEpi = BN > 64 ? 16 : (BN > 32 ? 8 : 4);      // epilogue warps: a quarter of the lanes each; the others share its columns
  static constexpr int kTma = kEpi, kMma = kEpi + 1, kScale = kEpi + 2, kThreads = 32 * (kEpi + 3);
  static constexpr int kColumns = 4 * BN / kEpi;                 // columns of a thread
  static constexpr int kPBytes = kRows * 128, kQBytes = BN * 128, kStage = kPBytes + kQBytes;
  static constexpr int kStages = BN == 16 ? 5 : (BN == 64 ? 3 : 4);
  static constexpr int kTogether = BN == 64 ? 4 : 8;             // blocks whose scales change hands together
  static constexpr int kPerSm = BN > 64 ? 1 : 2;                 // two: a launch's first weights come while the one before it ends
  static constexpr int kCols = kAcc * BN;                        // of TMEM
  static constexpr int kTokens = kSwap ? BN : kRows;             // of a tile
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStage + (2 * kTogether * kTokens + BN * (kRows + (kSwap ? 0 : 8))) * 4 + 256;
  static_assert(kCols == 64 || kCols == 128 || kCols == 256 || kCols == 512, "TMEM");
  // Clusters of two launches, each with a CTA that holds TMEM and one that waits for what the other holds, would not end.  Those that fit on an SM
  // together never ask for more than 512 columns: kernels here whose CTAs wait for one another take over 128 KB of shared memory where they take 512.
  static_assert(kCols * kPerSm <= 512, "TMEM of an SM");
  static_assert((kSmem + 1024) * kPerSm <= 228 * 1024, "shared memory");
  static_assert(kTogether % kVisit == 0 && (kSwap || kColumns == 32), "");
  static_assert(kSwap || (kEpi * 1024 <= BN * kRows && kThreads / 32 * 4096 <= kStages * kStage), "slabs");
};

// kSwap: what becomes of the sums of token m, weight rows n .. n + 3 (n a multiple of 4).  out32: unrounded, rows of ld32 columns.  `wide`: four
// results of out lie on an 8-byte boundary.  The fast exponentials' error is under either rounding that follows (common.cuh has it).
template <int EPI>
__device__ __forceinline__ void finish(const vila_fp8_linear_params& p, const vila_glinear_ext& x, float* out32, int ld32, bool wide, int m, int n, float4 sums) {
  constexpr bool kGated = EPI >= kMx4Gated;
  constexpr int kOut = kGated ? 2 : 4;
  if (m >= p.M || n >= p.N) return;
  float z[4] = {sums.x, sums.y, sums.z, sums.w};
  if (p.bias != nullptr) {
    const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias) + n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) z[j] += __bfloat162float(bias[j]);
  }
#pragma unroll
  for (int j = 0; j < kOut; ++j) z[j] = kGated ? mx4_glu<EPI>(z[2 * j % 4], z[(2 * j + 1) % 4], x) : mx4_act<EPI, true>(z[j], x);
  const int cols = kGated ? p.N / 2 : p.N, o = kGated ? n / 2 : n;
  if (out32 != nullptr) {
#pragma unroll
    for (int j = 0; j < kOut; ++j)
      if (o + j < cols) out32[static_cast<size_t>(m) * ld32 + o + j] = z[j];
    return;
  }
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(m) * p.ldo + o;
  if (wide && o + kOut <= cols) {
    if (kGated) *reinterpret_cast<uint32_t*>(out) = pack_bf16(z[0], z[1]);
    else *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]));
  } else {
#pragma unroll
    for (int j = 0; j < kOut; ++j)
      if (o + j < cols) out[j] = __float2bfloat16_rn(z[j]);
  }
}
// Without kSwap: of 32 tokens, a lane's m, those below `end`, and weight rows n .. n + 31.  All lanes call it.  `wide`: rows of out lie on 32-byte
// boundaries, and a lane writes its own; other rows change hands in `slab` (32 x 32, of this warp), so that neighbouring lanes write
// neighbouring columns (77 rows of 1157 columns, one block: 8.9 us if each lane writes 2 bytes of a row of its own at a time).
__device__ __forceinline__ void finish_rows(const vila_fp8_linear_params& p, const vila_glinear_ext& x, float* out32, int ld32, bool wide, int m, int end, int n,
                                            float (&z)[32], float* slab) {
  if (n >= p.N) return;
  mx4_with_epilogue(p, [&](auto epi) {
    constexpr int EPI = decltype(epi)::value;
    constexpr bool kGated = EPI >= kMx4Gated;
    constexpr int kOut = kGated ? 16 : 32, kRowsAtOnce = 32 / kOut;
    const int cols = kGated ? p.N / 2 : p.N, o = kGated ? n / 2 : n, lane = threadIdx.x & 31;
    if (p.bias != nullptr) {
      const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
#pragma unroll
      for (int i = 0; i < 32; ++i) z[i] += n + i < p.N ? __bfloat162float(bias[n + i]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kOut; ++i) z[i] = kGated ? mx4_glu<EPI>(z[2 * i % 32], z[(2 * i + 1) % 32], x) : mx4_act<EPI, true>(z[i], x);
    if (out32 == nullptr && wide && o + kOut <= cols) {
      if (m < end) {
        uint32_t h[kOut / 2];
#pragma unroll
        for (int i = 0; i < kOut / 2; ++i) h[i] = pack_bf16(z[2 * i], z[2 * i + 1]);
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(m) * p.ldo + o;
#pragma unroll
        for (int i = 0; i < kOut; i += 16) mx4_stg32(out + i, h + i / 2);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kOut; ++i) slab[lane * 32 + (i ^ lane)] = z[i];
    __syncwarp();
    const int m0 = m - lane, c = lane % kOut;
#pragma unroll 4
    for (int r0 = 0; r0 < 32; r0 += kRowsAtOnce) {
      const int r = r0 + lane / kOut;
      const float v = slab[r * 32 + (c ^ r)];
      if (m0 + r < end && o + c < cols) {
        if (out32 != nullptr) out32[static_cast<size_t>(m0 + r) * ld32 + o + c] = v;
        else static_cast<__nv_bfloat16*>(p.out)[static_cast<size_t>(m0 + r) * p.ldo + o + c] = __float2bfloat16_rn(v);
      }
    }
    __syncwarp();
  });
}

// split: CTAs of a cluster, which share a tile and cut K.
template <int BN, bool kSwap>
__global__ void __launch_bounds__(Shape<BN, kSwap>::kThreads, Shape<BN, kSwap>::kPerSm)
fp8_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const vila_fp8_linear_params p, const vila_glinear_ext x,
           float* out32, const int split, const WaitLimit limit, volatile unsigned int* failed) {
  using S = Shape<BN, kSwap>;
  constexpr int ST = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* scales = reinterpret_cast<float*>(smem + ST * S::kStage);      // [2][kTogether][token]: both scales of a token's block
  float* sums = scales + 2 * S::kTogether * S::kTokens;      // of this CTA's share of the rows, by rank: [rank][column][row], without kSwap a column one longer
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sums + BN * (kRows + (kSwap ? 0 : 8)));
  uint64_t* empty_bar = full_bar + ST;
  uint64_t* acc_full = empty_bar + ST;   // [2]: of up to kVisit blocks
  uint64_t* acc_free = acc_full + 2;     // [2]
  uint64_t* scale_full = acc_free + 2;   // [2]: of up to kTogether blocks
  uint64_t* scale_free = scale_full + 2; // [2]
  uint64_t* drain_bar = scale_free + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* gave_up = reinterpret_cast<int*>(tmem_ptr + 1);
  int* wides = reinterpret_cast<int*>(tmem_ptr + 2);      // [2]: whether a token's scales in a group of blocks are fp8_is_wide

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int p_tiles = ((kSwap ? p.N : p.M) + kRows - 1) / kRows, nkb = fp8_blocks(p.K);
  const int tile = static_cast<int>(blockIdx.x) / split, rank = static_cast<int>(blockIdx.x) - tile * split;
  const int kb0 = static_cast<int>(static_cast<long long>(nkb) * rank / split), kb1 = static_cast<int>(static_cast<long long>(nkb) * (rank + 1) / split);
  const int qt = tile / p_tiles, p0 = (tile - qt * p_tiles) * kRows, q0 = qt * BN;      // tiles that run together share their columns' rows
  const int t0 = kSwap ? q0 : p0, n0 = kSwap ? p0 : q0;                                 // first token, first weight row

  if (split > 1) cluster_arrive();      // this CTA runs: others may write to its shared memory
  // stages whose weights are asked for before the launch before has ended
  const int ahead = (p.flags & VILA_FLAG_STATIC_W) == 0 || limit.quits == 0 ? 0 : min(ST, kb1 - kb0);
  if (warp == S::kTma) {
    if (lane == 0) {
      tma_prefetch_desc(&tmap_p);
      tma_prefetch_desc(&tmap_q);
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
      for (int i = 0; i < ahead; ++i) {
        mbar_arrive_expect_tx(&full_bar[i], S::kStage);
        tma_load_2d(smem + i * S::kStage + (kSwap ? 0 : S::kPBytes), kSwap ? &tmap_p : &tmap_q, &full_bar[i], (kb0 + i) * 128, n0);
      }
    }
    __syncwarp();
  }
  if (warp == S::kMma) tmem_alloc<S::kCols>(tmem_ptr);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Behind TMEM: the next launch's CTAs may ask for theirs and then wait for this one to end, on an SM that both fit on.  Were they there first,
  // both would wait for good.
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_ptr;
  const int ld32 = p.flags & kGluFlags ? p.N / 2 : p.N;
  const bool wide = kSwap ? reinterpret_cast<uintptr_t>(p.out) % 8 == 0 && p.ldo % 4 == 0 : reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.ldo % 16 == 0;
  bool ok = true;
  if (limit.quits >= 0) {
    ok = limit.quits != (warp == S::kTma ? 0 : warp == S::kMma ? 1 : warp == S::kScale ? 2 : 3);
    if (!ok) *gave_up = 1;
  }

  if (warp == S::kTma) {
    const bool one = elect_one();
    const CUtensorMap *tw = kSwap ? &tmap_p : &tmap_q, *ta = kSwap ? &tmap_q : &tmap_p;
    const int w_at = kSwap ? 0 : S::kPBytes, a_at = kSwap ? S::kPBytes : 0;
    griddep_wait();
    int s = 0, rounds = 0;                // stage, rounds through all of them
    uint32_t ph = 1;                      // parity to wait for on an empty barrier: the first round passes
    for (int kb = kb0; kb < kb1 && ok; ++kb) {
      const bool first = kb - kb0 < ahead;
      if (!first) ok = mx4_warp_wait(&empty_bar[s], ph, gave_up, limit.tries);
      if (!ok) break;
      if (one) {
        uint8_t* st = smem + s * S::kStage;
        if (!first) {
          mbar_arrive_expect_tx(&full_bar[s], S::kStage);
          tma_load_2d(st + w_at, tw, &full_bar[s], kb * 128, n0);
        }
        tma_load_2d(st + a_at, ta, &full_bar[s], kb * 128, t0);
      }
      __syncwarp();
      if (++s == ST) {
        s = 0;
        ph ^= 1;
        ++rounds;
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
    constexpr uint32_t idesc = fp8_idesc(kRows, BN);
    griddep_wait();                       // or the tries of the first wait would be spent on the launch before
    int s = 0, v = 0;                     // stage, visits of the epilogue warps so far
    uint32_t ph = 0;
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
    if (one) umma_commit(drain_bar);             // products under way end before TMEM and the CTA's memory are given back, too
    if (lane == 0) mbar_drain(drain_bar, 0);
    __syncwarp();
  } else if (warp == S::kScale) {
    griddep_wait();
    // a lane takes four tokens; a row of scales is a multiple of 4 long, and behind the last token nothing counts.  Plain loads: the launch before may
    // still write what this one reads, and the read-only path is for what no launch writes meanwhile.
    const bool there = lane * 4 < S::kTokens && t0 + lane * 4 < p.ld_as;
    const float* sa = p.a_scales + (there ? t0 + lane * 4 : 0);
    const float* sw = p.w_scales + (n0 / kFp8Block) * p.ld_ws;
    int g = 0;
    for (int kb = kb0; kb < kb1 && ok; kb += S::kTogether, ++g) {
      float4 a[S::kTogether];
      float w[S::kTogether];
#pragma unroll
      for (int i = 0; i < S::kTogether; ++i) {
        const bool in = there && kb + i < kb1;
        a[i] = in ? *reinterpret_cast<const float4*>(sa + (kb + i) * p.ld_as) : make_float4(0.f, 0.f, 0.f, 0.f);
        w[i] = in ? sw[kb + i] : 0.f;
      }
      ok = mx4_warp_wait(&scale_free[g & 1], ((g >> 1) & 1) ^ 1, gave_up, limit.tries);      // the first two pass
      if (!ok) break;
      bool wide_x = false, wide_y = false, wide_z = false, wide_w = false;
#pragma unroll
      for (int i = 0; i < S::kTogether; ++i) {
        const float4 f = make_float4(fp8_both_scales(a[i].x, w[i]), fp8_both_scales(a[i].y, w[i]), fp8_both_scales(a[i].z, w[i]), fp8_both_scales(a[i].w, w[i]));
        wide_x |= fp8_is_wide(f.x);
        wide_y |= fp8_is_wide(f.y);
        wide_z |= fp8_is_wide(f.z);
        wide_w |= fp8_is_wide(f.w);
        if (lane * 4 < S::kTokens) *reinterpret_cast<float4*>(scales + ((g & 1) * S::kTogether + i) * S::kTokens + lane * 4) = f;
      }
      __syncwarp();
      const int t = t0 + lane * 4;
      const bool any = __any_sync(0xffffffffu, (wide_x && t < p.M) || (wide_y && t + 1 < p.M) || (wide_z && t + 2 < p.M) || (wide_w && t + 3 < p.M));
      if (lane == 0) {
        wides[g & 1] = any;
        mbar_arrive(&scale_full[g & 1]);
      }
    }
  } else {
    griddep_wait();
    const int quad = warp & 3, row = quad * 32 + lane, c0 = (warp >> 2) * S::kColumns;      // its lane of TMEM, its columns
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16) + c0;
    constexpr int kChunks = S::kColumns / 16;
    int v = 0, g = 0;                     // visits, groups of blocks so far
    bool any_wide = false;
    float sum[S::kColumns];
#pragma unroll
    for (int i = 0; i < S::kColumns; ++i) sum[i] = 0.f;
#pragma unroll 1
    for (int kb = kb0; kb < kb1 && ok; kb += kVisit, ++v) {
      const int in_group = (kb - kb0) % S::kTogether;
      if (in_group == 0) {
        if (kb > kb0) {      // all lanes have read the group before: the warp has met since
          if (lane == 0) mbar_arrive(&scale_free[g & 1]);
          ++g;
        }
        ok = mx4_warp_wait(&scale_full[g & 1], (g >> 1) & 1, gave_up, limit.tries);
        if (!ok) break;
        any_wide = wides[g & 1] != 0;
      }
      const float* both = scales + ((g & 1) * S::kTogether + in_group) * S::kTokens + (kSwap ? c0 : row);
      float mine[kVisit];
#pragma unroll
      for (int i = 0; i < kVisit; ++i) mine[i] = kSwap ? 0.f : both[i * S::kTokens];      // ahead of the loads from TMEM, which they would queue behind
      ok = mx4_warp_wait(&acc_full[v & 1], (v >> 1) & 1, gave_up, limit.tries);
      if (!ok) break;
      tc_fence_after();
      if (any_wide) {      // ahead of the loop: between its blocks the branch alone would keep one's sums from the next one's loads
#pragma unroll 1
        for (int i = 0; i < kVisit && kb + i < kb1; ++i)
          fp8_widen(lanes + ((v & 1) * kVisit + i) * BN, S::kColumns, [&](int c) { return both[i * S::kTokens + (kSwap ? c : 0)]; });
      }
#pragma unroll
      for (int i = 0; i < kVisit; ++i) {
        if (kb + i < kb1) {
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
              const float4 f = kSwap ? *reinterpret_cast<const float4*>(both + i * S::kTokens + 16 * c + j) : make_float4(mine[i], mine[i], mine[i], mine[i]);
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
    tc_fence_before();
    if (split == 1) {      // a warp finishes what it has summed up
      if (ok) {
        if constexpr (kSwap) {      // by a short loop: written out for every register, what a launch of few blocks took was fetching the code
#pragma unroll
          for (int c = 0; c < S::kColumns; ++c) sums[(c0 + c) * kRows + row] = sum[c];
          __syncwarp();
          mx4_with_epilogue(p, [&](auto epi) {
#pragma unroll 1
            for (int i = lane; i < S::kColumns * 8; i += 32) {
              const int c = c0 + i / 8, r = quad * 32 + 4 * (i % 8);
              finish<decltype(epi)::value>(p, x, out32, ld32, wide, t0 + c, n0 + r, *reinterpret_cast<const float4*>(sums + c * kRows + r));
            }
          });
        } else {
          finish_rows(p, x, out32, ld32, wide, t0 + row, p.M, n0 + c0, sum, sums + warp * 1024);      // nobody else's sums are there
        }
      }
    } else {               // the rows' sums to the CTAs that finish them
      cluster_wait();
      const int share = kRows / split, owner = row / share, at = row - owner * share;
      const uint32_t to = mapa_u32(smem_u32(sums), owner);
      if (ok) {
#pragma unroll
        for (int c = 0; c < S::kColumns; ++c) st_dsmem_f32(to + ((rank * BN + c0 + c) * (share + (kSwap ? 0 : 1)) + at) * 4, sum[c]);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  if (warp == S::kMma) {
    tc_fence_after();
    tmem_dealloc<S::kCols>(tmem);
  }
  if (split > 1) {
    if (warp >= S::kEpi) cluster_wait();      // the one that the epilogue warps have waited for
    __syncwarp();
    cluster_arrive();                         // behind this CTA's sums
    cluster_wait();
    const int share = kRows / split;
    if constexpr (kSwap) {
      const int fours = share / 4, items = min(BN, p.M - q0) * fours;
      mx4_with_epilogue(p, [&](auto epi) {
#pragma unroll 1
        for (int i = tid; i < items; i += S::kThreads) {
          const int c = i / fours, r = 4 * (i - c * fours);
          float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int q = 0; q < split; ++q) {
            const float4 part = *reinterpret_cast<const float4*>(sums + (q * BN + c) * share + r);
            z = make_float4(z.x + part.x, z.y + part.y, z.z + part.z, z.w + part.w);
          }
          finish<decltype(epi)::value>(p, x, out32, ld32, wide, t0 + c, n0 + rank * share + r, z);
        }
      });
    } else if (wide && out32 == nullptr) {      // a warp takes 32 rows by 32 columns
      const int groups = (share + 31) / 32;
#pragma unroll 1
      for (int i = warp; i < groups * (BN / 32); i += S::kThreads / 32) {
        const int r = i % groups * 32 + lane, c = i / groups * 32;
        float z[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = 0.f;
#pragma unroll 1
        for (int q = 0; q < split && r < share; ++q) {
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] += sums[(q * BN + c + j) * (share + 1) + r];
        }
        __syncwarp();
        finish_rows(p, x, out32, ld32, wide, t0 + rank * share + r, min(p.M, t0 + (rank + 1) * share), n0 + c, z,
                    reinterpret_cast<float*>(smem) + warp * 1024);      // the stages are done with
      }
    } else {      // a warp takes 32 neighbouring results of a token at a time
      mx4_with_epilogue(p, [&](auto epi) {
        constexpr int EPI = decltype(epi)::value;
        constexpr bool kGated = EPI >= kMx4Gated;
        constexpr int kParts = kGated ? BN / 64 : BN / 32;
        const int cols = kGated ? p.N / 2 : p.N, rows = min(share, p.M - t0 - rank * share);
        const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
#pragma unroll 2
        for (int i = warp; i < rows * kParts; i += S::kThreads / 32) {
          const int r = i / kParts, c = (i - r * kParts) * 32 + lane, m = t0 + rank * share + r, o = (kGated ? n0 / 2 : n0) + c;
          float z[2] = {0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 8; ++q) {
#pragma unroll
            for (int j = 0; j < (kGated ? 2 : 1); ++j)
              if (q < split) z[j] += sums[(q * BN + (kGated ? 2 * c + j : c)) * (share + 1) + r];
          }
          if (o < cols) {
            if (bias != nullptr) {
#pragma unroll
              for (int j = 0; j < (kGated ? 2 : 1); ++j) z[j] += __bfloat162float(bias[kGated ? 2 * o + j : o]);
            }
            const float v = kGated ? mx4_glu<EPI>(z[0], z[1], x) : mx4_act<EPI, true>(z[0], x);
            if (out32 != nullptr) out32[static_cast<size_t>(m) * ld32 + o] = v;
            else static_cast<__nv_bfloat16*>(p.out)[static_cast<size_t>(m) * p.ldo + o] = __float2bfloat16_rn(v);
          }
        }
      });
    }
  }
  if (tid == 0 && *gave_up) {
    *failed = 1u;
    __threadfence_system();
  }
}

template <int BN, bool kSwap>
int launch(const vila_fp8_linear_params& p, const vila_glinear_ext& x, float* out32, int tries, cudaStream_t stream) {
  using S = Shape<BN, kSwap>;
  static PerDeviceOnce once;
  VB_ALLOW_SMEM(once, fp8_kernel<BN, kSwap>, static_cast<int>(S::kSmem));
  CUtensorMap tw, ta;
  if (int rc = make_tmap_2d_u8(&tw, p.w_codes, p.N, p.K, p.ldw, kSwap ? kRows : BN, 128, 128)) return rc;
  if (int rc = make_tmap_2d_u8(&ta, p.a_codes, p.M, p.K, p.lda, S::kTokens, 128, 128)) return rc;
  const long long tiles = kSwap ? (p.N + kRows - 1) / kRows : static_cast<long long>((p.N + BN - 1) / BN) * ((p.M + kRows - 1) / kRows);
  VB_CHECK(tiles < (1LL << 27), "fp8_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  static Mx4Clusters clusters;
  // As many CTAs a tile, a power of two up to 8, as the GPU holds clusters for at once.  The occupancy that CUDA reports counts one CTA an SM
  // where two fit (15 clusters of 8); the GPU holds both (64 rows of 3584 x 18944 by 4: 25.5 us, by 2, as reported, 33.6).
  // Of 4 blocks a cluster's joint end costs what it saves (77 rows of 1157 x 512: 7.2 us by two, 6.2 alone; x 1024 by 4 7.1, by 2 8.0).
  const int blocks = fp8_blocks(p.K), limit = blocks < 8 ? 1 : blocks / 2;
  int split = 1;
  for (int l = 1; l <= 3 && (1 << l) <= limit && tiles <= static_cast<long long>(S::kPerSm) * clusters.of(fp8_kernel<BN, kSwap>, l, S::kThreads, S::kSmem); ++l)
    split = 1 << l;
  VB_CUDA(launch_pdl_cluster(fp8_kernel<BN, kSwap>, dim3(static_cast<unsigned>(tiles * split)), dim3(S::kThreads), S::kSmem, stream, dim3(split),
                             kSwap ? tw : ta, kSwap ? ta : tw, p, x, out32, split, wait_limit(tries), failed_word()));
  return 0;
}

}  // namespace

int fp8_tc(const vila_fp8_linear_params& p, const vila_glinear_ext& ext, float* out32, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "fp8_linear: no pinned host memory for the status word");
  if (p.M <= 16) return launch<16, true>(p, ext, out32, tries, stream);
  if (p.M <= 32) return launch<32, true>(p, ext, out32, tries, stream);
  // fp8_pair_takes has the rule for tiles that are many.  Up to 128 tokens tiles of 64 weight rows, two CTAs an SM; beyond, tokens would be read too often.
  if (p.M <= 128) return launch<64, false>(p, ext, out32, tries, stream);
  return launch<128, false>(p, ext, out32, tries, stream);
}

}  // namespace vb
