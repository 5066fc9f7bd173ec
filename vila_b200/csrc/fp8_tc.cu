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
// Up to 32 tokens (kSwap): weight rows are the 128 lanes of a tile, tokens its columns, of which there are only as many as needed; bound by the
// weights' bytes.  More tokens: these are the lanes, 128 weight rows the columns, so that a thread's scale is one number a block (as one a column
// it took four loads from shared memory per 16 columns, in line with the loads from TMEM: 0.43 us a block instead of 0.3).  There a block
// costs what an epilogue warp does for it one after another: a wait takes 150 - 250 clocks even if it is over, 16 columns of TMEM 70.
//
// A CTA takes one tile, or, where the tiles leave SMs idle, a share of its blocks: a cluster of up to 8 CTAs splits K, every CTA sends
// its sums to the CTAs that finish them, by rows, and these add them in rank order.  Sums go through shared memory in any case, and a
// loop of few instructions finishes them (written out for every register of a thread, what a launch of few blocks took was fetching it).
//
// A launch may begin before the one before it has ended: the first weights are asked for while that one ends, everything else comes behind
// griddepcontrol.wait.  (Weights come from launches that do not let others begin early.)
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "fp8.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"
#include "mx4.cuh"

namespace vb {
namespace {

constexpr int kRows = 128;                    // lanes of a tile
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
__device__ __forceinline__ void st_dsmem_f32(uint32_t cluster_addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_dsmem_v4f(uint32_t cluster_addr, const float* v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(cluster_addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <int BN, bool kSwap> struct Shape {
  static constexpr int kEpi = BN > 64 ? 16 : 4;                 // epilogue warps: a quarter of the lanes each; four share a quarter's columns
  static constexpr int kTma = kEpi, kMma = kEpi + 1, kScale = kEpi + 2, kThreads = 32 * (kEpi + 3);
  static constexpr int kColumns = BN > 64 ? BN / 4 : BN;        // columns of a thread
  static constexpr int kPBytes = kRows * 128, kQBytes = BN * 128, kStage = kPBytes + kQBytes;
  static constexpr int kStages = BN == 16 ? 5 : 4;
  static constexpr int kPerSm = BN > 64 ? 1 : 2;
  static constexpr int kCols = kAcc * BN;                        // of TMEM
  static constexpr int kTokens = kSwap ? BN : kRows;             // of a tile
  static constexpr int kPitch = kSwap ? 0 : BN + 4;              // of a token's sums, so that lanes with a token each meet different banks
  static constexpr int kSums = kSwap ? BN * kRows : kRows * kPitch;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * kStage + (2 * kTogether * kTokens + kSums) * 4 + 256;
  static_assert(kCols == 64 || kCols == 128 || kCols == 256 || kCols == 512, "TMEM");
  static_assert(kCols * kPerSm <= 512, "TMEM of an SM");
  static_assert((kSmem + 1024) * kPerSm <= 228 * 1024, "shared memory");
};

// What becomes of the sums of token m, weight rows n .. n + 3 (n a multiple of 4).  out32: unrounded, rows of ld32 columns.  `wide`: four
// results of out lie on an 8-byte boundary.  The fast exponentials are off by some 2^-21, under either rounding that follows.
__device__ __forceinline__ void finish(const vila_fp8_linear_params& p, const vila_glinear_ext& x, float* out32, int ld32, bool wide, int m, int n, float4 sums) {
  if (m >= p.M || n >= p.N) return;
  float z[4] = {sums.x, sums.y, sums.z, sums.w};
  if (p.bias != nullptr) {
    const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias) + n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) z[j] += __bfloat162float(bias[j]);
  }
  const bool gated = (p.flags & kGluFlags) != 0;
  if (gated) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float g = z[2 * j], u = z[2 * j + 1];
      z[j] = p.flags & VILA_FLAG_GLU_CLAMP ? glu_clamp_fast_f(g, u, x.act_alpha, x.act_limit) : (p.flags & VILA_FLAG_GEGLU ? gelu_tanh_f(g) : silu_f(g)) * u;
    }
  } else if (p.act != VILA_ACT_NONE) {
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const float v = z[0];      // in turn, so that the activations are there once
      z[0] = z[1];
      z[1] = z[2];
      z[2] = z[3];
      z[3] = p.act == VILA_ACT_SILU ? silu_f(v) : (p.act == VILA_ACT_GELU_TANH ? gelu_tanh_f(v) : (p.act == VILA_ACT_XIELU ? xielu_fast_f(v, x.act_pos, x.act_neg) : activate(v, p.act, x)));
    }
  }
  const int cols = gated ? p.N / 2 : p.N, o = gated ? n / 2 : n, count = gated ? 2 : 4;
  if (out32 != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < count && o + j < cols) out32[static_cast<size_t>(m) * ld32 + o + j] = z[j];
    return;
  }
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(m) * p.ldo + o;
  if (wide && o + count <= cols) {
    if (gated) *reinterpret_cast<uint32_t*>(out) = pack_bf16(z[0], z[1]);
    else *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < count && o + j < cols) out[j] = __float2bfloat16_rn(z[j]);
  }
}

// bn: columns of a tile, with kSwap a multiple of 16, at most BN.  split: CTAs of a cluster, which share a tile and cut K.
template <int BN, bool kSwap>
__global__ void __launch_bounds__(Shape<BN, kSwap>::kThreads, Shape<BN, kSwap>::kPerSm)
fp8_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const vila_fp8_linear_params p, const vila_glinear_ext x,
           float* out32, const int bn, const int split, const WaitLimit limit, volatile unsigned int* failed) {
  using S = Shape<BN, kSwap>;
  constexpr int ST = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* scales = reinterpret_cast<float*>(smem + ST * S::kStage);      // [2][kTogether][token]: both scales of a token's block
  float* sums = scales + 2 * kTogether * S::kTokens;      // of this CTA's share of the rows, by rank: [rank][column][row], or [rank][row][column]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sums + S::kSums);
  uint64_t* empty_bar = full_bar + ST;
  uint64_t* acc_full = empty_bar + ST;   // [2]: of up to kVisit blocks
  uint64_t* acc_free = acc_full + 2;     // [2]
  uint64_t* scale_full = acc_free + 2;   // [2]: of up to kTogether blocks
  uint64_t* scale_free = scale_full + 2; // [2]
  uint64_t* drain_bar = scale_free + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* gave_up = reinterpret_cast<int*>(tmem_ptr + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int p_tiles = ((kSwap ? p.N : p.M) + kRows - 1) / kRows, nkb = fp8_blocks(p.K);
  const int tile = static_cast<int>(blockIdx.x) / split, rank = static_cast<int>(blockIdx.x) - tile * split;
  const int kb0 = static_cast<int>(static_cast<long long>(nkb) * rank / split), kb1 = static_cast<int>(static_cast<long long>(nkb) * (rank + 1) / split);
  const int qt = tile / p_tiles, p0 = (tile - qt * p_tiles) * kRows, q0 = qt * bn;      // tiles that run together share their columns' rows
  const int t0 = kSwap ? q0 : p0, n0 = kSwap ? p0 : q0;                                 // first token, first weight row

  griddep_launch_dependents();
  if (split > 1) cluster_arrive();      // this CTA runs: others may write to its shared memory
  if (tid == 0) {
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
  }
  if (warp == S::kMma) tmem_alloc<S::kCols>(tmem_ptr);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const int ld32 = p.flags & kGluFlags ? p.N / 2 : p.N;
  const bool wide = reinterpret_cast<uintptr_t>(p.out) % 8 == 0 && p.ldo % 4 == 0;
  bool ok = true;
  if (limit.quits >= 0) {
    ok = limit.quits != (warp == S::kTma ? 0 : warp == S::kMma ? 1 : warp == S::kScale ? 2 : 3);
    if (!ok) *gave_up = 1;
  }

  if (warp == S::kTma) {
    const bool one = elect_one();
    const CUtensorMap *tw = kSwap ? &tmap_p : &tmap_q, *ta = kSwap ? &tmap_q : &tmap_p;
    const int w_at = kSwap ? 0 : S::kPBytes, a_at = kSwap ? S::kPBytes : 0;
    const uint32_t bytes = S::kPBytes + bn * 128;
    const int ahead = ok ? min(ST, kb1 - kb0) : 0;      // stages whose weights are asked for before the launch before has ended
    if (one)
      for (int i = 0; i < ahead; ++i) {
        mbar_arrive_expect_tx(&full_bar[i], bytes);
        tma_load_2d(smem + i * S::kStage + w_at, tw, &full_bar[i], (kb0 + i) * 128, n0);
      }
    __syncwarp();
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
          mbar_arrive_expect_tx(&full_bar[s], bytes);
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
    const uint32_t idesc = fp8_idesc(kRows, bn);
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
    // a lane takes four tokens; a row of scales is a multiple of 4 long, and behind the last token nothing counts
    const int most = kSwap ? bn : kRows;
    const bool there = lane * 4 < most && t0 + lane * 4 < p.ld_as;
    const float* sa = p.a_scales + (there ? t0 + lane * 4 : 0);
    const float* sw = p.w_scales + (n0 / kFp8Block) * p.ld_ws;
    int g = 0;
    for (int kb = kb0; kb < kb1 && ok; kb += kTogether, ++g) {
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
      if (lane * 4 < S::kTokens) {
#pragma unroll
        for (int i = 0; i < kTogether; ++i)
          *reinterpret_cast<float4*>(scales + ((g & 1) * kTogether + i) * S::kTokens + lane * 4) =
              make_float4(fp8_both_scales(a[i].x, w[i]), fp8_both_scales(a[i].y, w[i]), fp8_both_scales(a[i].z, w[i]), fp8_both_scales(a[i].w, w[i]));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&scale_full[g & 1]);
    }
  } else {
    griddep_wait();
    const int quad = warp & 3, row = quad * 32 + lane, c0 = (warp >> 2) * S::kColumns;      // its lane of TMEM, its columns
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16) + c0;
    constexpr int kChunks = S::kColumns / 16;
    int v = 0, g = 0;                     // visits, groups of blocks so far
    float sum[S::kColumns];
#pragma unroll
    for (int i = 0; i < S::kColumns; ++i) sum[i] = 0.f;
#pragma unroll 1
    for (int kb = kb0; kb < kb1 && ok; kb += kVisit, ++v) {
      const int in_group = (kb - kb0) % kTogether;
      if (in_group == 0) {
        if (kb > kb0) {      // all lanes have read the group before: the warp has met since
          if (lane == 0) mbar_arrive(&scale_free[g & 1]);
          ++g;
        }
        ok = mx4_warp_wait(&scale_full[g & 1], (g >> 1) & 1, gave_up, limit.tries);
        if (!ok) break;
      }
      const float* both = scales + ((g & 1) * kTogether + in_group) * S::kTokens + (kSwap ? c0 : row);
      float mine[kVisit];
#pragma unroll
      for (int i = 0; i < kVisit; ++i) mine[i] = kSwap ? 0.f : both[i * S::kTokens];      // ahead of the loads from TMEM, which they would queue behind
      ok = mx4_warp_wait(&acc_full[v & 1], (v >> 1) & 1, gave_up, limit.tries);
      if (!ok) break;
      tc_fence_after();
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
        if constexpr (kSwap) {
#pragma unroll
          for (int c = 0; c < S::kColumns; ++c) sums[(c0 + c) * kRows + row] = sum[c];
          __syncwarp();
#pragma unroll 1
          for (int i = lane; i < S::kColumns * 8; i += 32) {
            const int c = c0 + i / 8, r = quad * 32 + 4 * (i % 8);
            if (c < bn) finish(p, x, out32, ld32, wide, t0 + c, n0 + r, *reinterpret_cast<const float4*>(sums + c * kRows + r));
          }
        } else {
#pragma unroll
          for (int c = 0; c < S::kColumns; c += 4) *reinterpret_cast<float4*>(sums + row * S::kPitch + c0 + c) = make_float4(sum[c], sum[c + 1], sum[c + 2], sum[c + 3]);
          __syncwarp();
#pragma unroll 1
          for (int i = lane; i < 32 * S::kColumns / 4; i += 32) {
            const int r = quad * 32 + i / (S::kColumns / 4), c = c0 + 4 * (i % (S::kColumns / 4));
            finish(p, x, out32, ld32, wide, t0 + r, n0 + c, *reinterpret_cast<const float4*>(sums + r * S::kPitch + c));
          }
        }
      }
    } else {               // the rows' sums to the CTAs that finish them
      cluster_wait();
      const int share = kRows / split, owner = row / share, at = row - owner * share;
      const uint32_t to = mapa_u32(smem_u32(sums), owner);
      if (ok) {
        if constexpr (kSwap) {
#pragma unroll
          for (int c = 0; c < S::kColumns; ++c) st_dsmem_f32(to + ((rank * BN + c0 + c) * share + at) * 4, sum[c]);
        } else {
#pragma unroll
          for (int c = 0; c < S::kColumns; c += 4) st_dsmem_v4f(to + ((rank * share + at) * S::kPitch + c0 + c) * 4, sum + c);
        }
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
    const int fours = (kSwap ? share : BN) / 4, lines = kSwap ? min(bn, p.M - q0) : share;
#pragma unroll 1
    for (int i = tid; i < lines * fours; i += S::kThreads) {
      const int l = i / fours, f = 4 * (i - l * fours);
      float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < split; ++q) {
        const float4 part = *reinterpret_cast<const float4*>(sums + (kSwap ? (q * BN + l) * share + f : (q * share + l) * S::kPitch + f));
        z = make_float4(z.x + part.x, z.y + part.y, z.z + part.z, z.w + part.w);
      }
      finish(p, x, out32, ld32, wide, kSwap ? t0 + l : t0 + rank * share + l, kSwap ? n0 + rank * share + f : n0 + f, z);
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
  const int bn = kSwap ? (p.M + 15) / 16 * 16 : BN;
  CUtensorMap tw, ta;
  if (int rc = make_tmap_2d_u8(&tw, p.w_codes, p.N, p.K, p.ldw, kSwap ? kRows : BN, 128, 128)) return rc;
  if (int rc = make_tmap_2d_u8(&ta, p.a_codes, p.M, p.K, p.lda, kSwap ? bn : kRows, 128, 128)) return rc;
  const long long tiles = static_cast<long long>((p.N + kRows - 1) / kRows) * (kSwap ? 1 : (p.M + kRows - 1) / kRows);
  VB_CHECK(tiles < (1LL << 27), "fp8_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  static Mx4Clusters clusters;
  const int split = clusters.split(fp8_kernel<BN, kSwap>, S::kThreads, S::kSmem, tiles, fp8_blocks(p.K) / 2);
  VB_CUDA(launch_pdl_cluster(fp8_kernel<BN, kSwap>, dim3(static_cast<unsigned>(tiles * split)), dim3(S::kThreads), S::kSmem, stream, dim3(split),
                             kSwap ? tw : ta, kSwap ? ta : tw, p, x, out32, bn, split, wait_limit(tries), failed_word()));
  return 0;
}

}  // namespace

int fp8_tc(const vila_fp8_linear_params& p, const vila_glinear_ext& ext, float* out32, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "fp8_linear: no pinned host memory for the status word");
  if (p.M <= 16) return launch<16, true>(p, ext, out32, tries, stream);
  if (p.M <= 32) return launch<32, true>(p, ext, out32, tries, stream);
  return launch<128, false>(p, ext, out32, tries, stream);
}

}  // namespace vb
