// Linear layers of bf16 rows on microscaled 4-bit weights, more rows than mx4_rows.cu is for: tcgen05.mma kind::f16 with the
// weights unpacked into TMEM.
//
// A weight is code * 2^e, which bf16 holds exactly, so the products are those of bf16 operands.  The unpacked weights never see
// memory: the M side of tcgen05.mma may lie in TMEM, lane = weight row, 32 columns = 64 weights of a row, which is what a thread that
// unpacks its own row writes with one tcgen05.st.  Shared memory then only serves the tokens, the N side.
//
//   2 TMA warps      codes and scales, 256 columns of 128 rows at a time; a stage of tokens (64 columns, 128 bytes, swizzled).  As the MMA
//                    warp they stay converged but for the branch that issues: one thread with both loops took 800 clocks a stage
//   unpack warps     two or three groups of four (a warp reaches the TMEM lanes of its quarter), which take the stages in turn: a byte of
//                    codes (two weights) is looked up in shared memory as a pair of bf16, then multiplied by the block's 2^e
//   MMA warp         TMEM allocation; tcgen05.mma of K = 16, four per 64 columns, into one of two accumulator sets
//   8 epilogue warps TMEM lane = weight row, column = token, under the next tile's products
//
// The table has 256 entries, one copy for each lane in a bank of its own, entry v of lane l at 65536 + 256 v + 4 l: one prmt makes the
// address, no two lanes meet in a bank.  Spreading the bits with integer instructions instead took 174 of them on the ALU per
// 64 weights of a row (counted by the profiler), 350 clocks of a scheduler at 16 lanes a clock, where the products of 128 tokens take 256.
// With the table and faster activations 2048 rows through 37888 x 3584, gated, went from 545 to 457 us; the two were not timed apart.
//
// Tiles of 128 weight rows x up to BT tokens; of many tokens by CTA pairs (cta_group::2), each CTA with 128 of 256 weight rows and half
// of 256 tokens in its shared memory: an SM takes in 54 bytes a clock, and 256 tokens of its own alone are 64 per clock of their
// products.  Tokens have a ring of their own, as deep as shared memory allows: from the end of a stage's products to the arrival of
// the tokens that replace it 1.6 us pass.  The pair's accumulators share kShared columns, which the epilogue takes first (there is no
// room for both beside the unpacked weights).
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "mx4.cuh"
#include "mx4_epi.cuh"

namespace vb {
namespace {

constexpr int kRowsW = 128, kDepth = 64, kCodeDepth = 256;
constexpr int kEpi = 8, kFirstUnpack = kEpi;
constexpr int kCodeBytes = kRowsW * 128, kCodeStage = kCodeBytes + 1024, kCodeStages = 3;
// Shared memory by addresses of the shared window: codes and barriers, the table from 64 KB on, tokens behind it
constexpr uint32_t kTable = 0x10000, kTokens = 0x20000, kTokensBytes = 96 * 1024, kBars = kCodeStages * kCodeStage, kLow = kBars + 1024;
constexpr uint32_t kSmemFrom = 1024;                  // where dynamic shared memory begins (the first 1 KB is the system's)
constexpr size_t kSmem = kTokens + kTokensBytes - kSmemFrom;
static_assert(kSmemFrom + kLow <= kTable && kSmem <= 227 * 1024, "");

template <int BT, bool kPair> struct Shape {
  static constexpr int kGroups = kPair ? 2 : 3;                 // of four unpack warps
  static constexpr int kUnpack = 4 * kGroups, kTma = kEpi + kUnpack, kCode = kTma + 1, kMma = kTma + 2, kThreads = 32 * (kMma + 1);
  // times 64 columns are a stage: of one, the issuing warp's 400 clocks a stage showed (17 rows, 3584 x 3584: 22.2 us, of two 19.1)
  static constexpr int kSub = kPair ? 1 : 2;
  static constexpr int kTokRows = kPair ? BT / 2 : BT;          // that a CTA holds
  static constexpr int kTokBytes = kSub * kTokRows * 128;
  static constexpr int kTok = kTokensBytes / kTokBytes;         // stages of tokens
  static constexpr int kW = 4;                                  // stages of unpacked weights
  static constexpr int kAcc1 = BT > 128 ? 128 : BT;             // the second accumulator's first column
  static constexpr int kShared = BT - kAcc1;
  static constexpr int kWeights = kAcc1 + BT;                   // first column of the unpacked weights
  static constexpr int kCols = 512;
  static_assert(kWeights + kW * kSub * 32 <= kCols && kShared % 16 == 0, "");
};

template <bool kPair>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (kPair)
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// eight codes -> four pairs of bf16 out of the table; here: this lane's column of it
__device__ __forceinline__ void look_up8(uint32_t w, uint32_t here, uint32_t (&y)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t at;      // bytes: here's 0, w's byte i, here's 2 and 3
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(at) : "r"(w), "r"(here), "r"(0x7604 | i << 4));
    asm("ld.shared.u32 %0, [%1];" : "=r"(y[i]) : "r"(at));
  }
}

// Token tiles of M rows: as few as tiles of BT allow, or more where that fills the SMs, of nearly equal size
struct Pieces {
  int n, per;     // tiles, rows of one (a multiple of 16, of 32 for pairs)
};

template <int BT, bool kPair>
__global__ void __launch_bounds__(Shape<BT, kPair>::kThreads, 1)
mx4_mixed_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const vila_mx4_linear_params p,
                 const vila_glinear_ext x, const Pieces pieces, const WaitLimit limit, volatile unsigned int* failed) {
  using S = Shape<BT, kPair>;
  constexpr int kUnpack = S::kUnpack, kTma = S::kTma, kCode = S::kCode, kMma = S::kMma;
  constexpr int kCtas = kPair ? 2 : 1, kSteps = kCodeDepth / (kDepth * S::kSub);      // stages of 256 columns
  extern __shared__ uint8_t smem_raw[];
  // where it lies in the shared window is known, as the kernel has no other; in a cluster the CTA's rank is in the upper bits.  (Were it
  // somewhere else, all CTAs would leave here, and the launch be reported as one that gave up.)
  const uint32_t window = smem_u32(smem_raw) - kSmemFrom;
  if ((window & 0xffffffu) != 0u) {
    if (threadIdx.x == 0) *failed = 1u;
    return;
  }
  uint8_t *codes_s = smem_raw, *smem = smem_raw + (kTokens - kSmemFrom);
  uint64_t* tok_full = reinterpret_cast<uint64_t*>(codes_s + kBars);   // a pair's: in the first CTA, of both
  uint64_t* tok_empty = tok_full + S::kTok;
  uint64_t* w_full = tok_empty + S::kTok;          // unpacked weights are in TMEM; a pair's: in the first CTA, of both
  uint64_t* w_empty = w_full + S::kW;
  uint64_t* code_full = w_empty + S::kW;
  uint64_t* code_empty = code_full + kCodeStages;
  uint64_t* acc_full = code_empty + kCodeStages;   // [2]
  uint64_t* acc_free = acc_full + 2;               // [2]; with shared columns [0] alone, a phase a tile; a pair's: in the first CTA
  uint64_t* drain_bar = acc_free + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* gave_up = reinterpret_cast<int*>(tmem_ptr + 1);
  volatile int* asked = gave_up + 1;               // [2]: stages of tokens that this CTA asked for; in a pair's first one also: the second did

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;
  const int worker = kPair ? blockIdx.x >> 1 : blockIdx.x, workers = kPair ? gridDim.x >> 1 : gridDim.x;
  const int n_tiles = (p.N + kCtas * kRowsW - 1) / (kCtas * kRowsW), total = n_tiles * pieces.n;
  const int nkb = (p.K + kDepth * S::kSub - 1) / (kDepth * S::kSub), nkc = (p.K + kCodeDepth - 1) / kCodeDepth;
  auto tile_at = [&](int it, int& n0, int& m0, int& count) {
    const int q = it / pieces.n;
    m0 = (it - q * pieces.n) * pieces.per;
    count = min(pieces.per, p.M - m0);
    n0 = (q * kCtas + rank) * kRowsW;
  };
  auto in_first = [&](uint64_t* bar) { return kPair ? mapa_u32(smem_u32(bar), 0) : smem_u32(bar); };
  auto arrive_first = [&](uint64_t* bar) {
    if (kPair) mbar_arrive_cluster_relaxed(in_first(bar));
    else mbar_arrive(bar);
  };
  auto commit = [&](uint64_t* bar) {
    if (kPair) umma_commit_pair(bar);
    else umma_commit(bar);
  };
  // a warp that gives up tells the other CTA, too
  auto tell = [&] {
    *gave_up = 1;
    if (kPair) st_dsmem_u32(mapa_u32(smem_u32(const_cast<int*>(gave_up)), rank ^ 1), 1u);
  };

  if (tid == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    for (int i = 0; i < S::kTok; ++i) {
      mbar_init(&tok_full[i], 1);
      mbar_init(&tok_empty[i], 1);
    }
    for (int i = 0; i < S::kW; ++i) {
      mbar_init(&w_full[i], 4 * kCtas);
      mbar_init(&w_empty[i], 1);
    }
    for (int i = 0; i < kCodeStages; ++i) {
      mbar_init(&code_full[i], 1);
      mbar_init(&code_empty[i], kUnpack);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], kEpi * kCtas);
    }
    mbar_init(drain_bar, 1);
    *gave_up = 0;
    fence_barrier_init();
  }
  for (int v = warp; v < 256; v += S::kThreads / 32) {      // the table
    const uint32_t lo = v & 15, hi = v >> 4;
    const float a = mx4_number(lo), b = mx4_number(hi);
    *reinterpret_cast<uint32_t*>(smem_raw + (kTable - kSmemFrom) + v * 256 + lane * 4) = pack_bf16(a, b);
  }
  if (warp == kMma) {
    if (kPair) tmem_alloc_pair<S::kCols>(tmem_ptr);
    else tmem_alloc<S::kCols>(tmem_ptr);
  }
  tc_fence_before();
  __syncthreads();
  if (kPair) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const int role = warp == kTma || warp == kCode ? 0 : warp == kMma ? 1 : warp >= kFirstUnpack ? 2 : 3;
  bool ok = kPair ? !mx4_pair_quits(limit, role, rank) : limit.quits != role;

  if (warp == kTma) {
    const bool one = elect_one();
    const int tok_rows = kPair ? pieces.per / 2 : pieces.per;
    const uint32_t tok_bytes = S::kSub * pieces.per * 128;      // of both CTAs
    int s = 0, rounds = 0;                // stage, and rounds through all of them
    uint32_t ph = 1, here = 1;            // the first round passes
    for (int it = worker; it < total && ok; it += workers) {
      int n0, m0, count;
      tile_at(it, n0, m0, count);
      for (int kb = 0; kb < nkb; ++kb) {
        if (!__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&tok_empty[s], ph, gave_up, limit.tries);
        if (!ok) break;
        uint8_t* st = smem + s * S::kTokBytes;
        uint64_t* full = &tok_full[s];
        if (++s == S::kTok) {
          s = 0;
          ph ^= 1;
          ++rounds;
        }
        here = mx4_test(&tok_empty[s], ph);
        if (one) {
          if (rank == 0) mbar_arrive_expect_tx(full, tok_bytes);
          // a box is a tile's rows: of boxes of 32 rows, 8 a stage, 8192 x 8192 x 8192 took 1.23 ms, and 0.72 without the tokens
#pragma unroll
          for (int i = 0; i < S::kSub; ++i) {
            if (kPair) tma_load_2d_pair(st, &tmap_x, in_first(full), kb * kDepth, m0 + rank * tok_rows);
            else tma_load_2d(st + i * S::kTokRows * 128, &tmap_x, full, (kb * S::kSub + i) * kDepth, m0);
          }
        }
        __syncwarp();
      }
    }
    if (lane == 0) {
      if (!ok) tell();
      // what was asked for lands before the CTA's memory is given back, whichever warp gave up (a pair's: at its end)
      if (kPair) asked[0] = rounds * S::kTok + s;
      else
        for (int i = 0; i < S::kTok; ++i) {
          const int round = i < s ? rounds : rounds - 1;
          if (round >= 0) mbar_drain(&tok_full[i], round & 1);
        }
    }
    __syncwarp();
  } else if (warp == kCode) {
    const bool one = elect_one();
    const int kts = 2 * nkc;
    int s = 0, rounds = 0;
    uint32_t ph = 1, here = 1;
    for (int it = worker; it < total && ok; it += workers) {
      int n0, m0, count;
      tile_at(it, n0, m0, count);
      // the second CTA's rows may begin past the last weight row: TMA fills in zeros, scales are not loaded
      const bool scales = n0 < p.N;
      const uint8_t* scale = p.w_scales + static_cast<size_t>(n0 >> 7) * kts * 512;
      for (int kc = 0; kc < nkc; ++kc) {
        if (!__all_sync(0xffffffffu, here)) ok = mx4_warp_wait(&code_empty[s], ph, gave_up, limit.tries);
        if (!ok) break;
        uint8_t* st = codes_s + s * kCodeStage;
        uint64_t* full = &code_full[s];
        if (++s == kCodeStages) {
          s = 0;
          ph ^= 1;
          ++rounds;
        }
        here = mx4_test(&code_empty[s], ph);
        if (one) {
          mbar_arrive_expect_tx(full, kCodeBytes + (scales ? 1024 : 0));
          tma_load_2d(st, &tmap_w, full, kc * 128, n0);
          if (scales) mx4_bulk_load(st + kCodeBytes, scale + kc * 1024, 1024, full);
        }
        __syncwarp();
      }
    }
    if (lane == 0) {
      if (!ok) tell();
      for (int i = 0; i < kCodeStages; ++i) {
        const int round = i < s ? rounds : rounds - 1;
        if (round >= 0) mbar_drain(&code_full[i], round & 1);
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    if (rank == 0) {
      // The whole warp walks the loop and one lane issues: what the instructions are given stays in uniform registers.
      const bool one = elect_one();
      const uint64_t bd0 = make_smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128);
      int k = 0, s = 0, w = 0;
      uint32_t ph = 0, wph = 0;
      for (int it = worker; it < total && ok; it += workers, ++k) {
        int n0, m0, count;
        tile_at(it, n0, m0, count);
        const uint32_t idesc = make_idesc_bf16(kCtas * kRowsW, kPair ? pieces.per : (count + 15) & ~15, 0, 0), acc = tmem + (k & 1) * S::kAcc1;
        if (S::kShared > 0) ok = k == 0 || mx4_warp_wait(&acc_free[0], (k - 1) & 1, gave_up, limit.tries);
        else ok = mx4_warp_wait(&acc_free[k & 1], ((k >> 1) & 1) ^ 1, gave_up, limit.tries);
        uint32_t tok_here = 0, w_here = 0;
        for (int kb = 0; kb < nkb && ok; ++kb) {
          if (!__all_sync(0xffffffffu, tok_here & w_here))
            ok = mx4_warp_wait(&tok_full[s], ph, gave_up, limit.tries) && mx4_warp_wait(&w_full[w], wph, gave_up, limit.tries);
          if (!ok) break;
          tc_fence_after();
          const uint64_t bd = bd0 + s * (S::kTokBytes >> 4);
          const uint32_t wa = tmem + S::kWeights + 32 * S::kSub * w;
          uint64_t *tok_done = &tok_empty[s], *w_done = &w_empty[w];
          if (++s == S::kTok) {
            s = 0;
            ph ^= 1;
          }
          if (++w == S::kW) {
            w = 0;
            wph ^= 1;
          }
          tok_here = mx4_test(&tok_full[s], ph);
          w_here = mx4_test(&w_full[w], wph);
          if (one) {      // columns past K are zeros on both sides
#pragma unroll
            for (int i = 0; i < 4 * S::kSub; ++i)
              umma_ts<kPair>(acc, wa + 8 * i, bd + (i / 4) * (S::kTokRows * 128 >> 4) + 2 * (i % 4), idesc, (kb | i) != 0);
            commit(tok_done);
            commit(w_done);
          }
          __syncwarp();
        }
        if (ok && one) commit(&acc_full[k & 1]);
        __syncwarp();
      }
      if (!ok && lane == 0) tell();
      if (one) commit(drain_bar);      // a pair's: reports to both CTAs
    }
    // products under way, and what they report to this CTA, end before TMEM and the CTA's memory are given back
    if (lane == 0 && !mbar_wait_limited(drain_bar, 0, gave_up, limit.tries)) mbar_drain(drain_bar, 0);
    __syncwarp();
  } else if (warp >= kFirstUnpack) {
    const int group = (warp - kFirstUnpack) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t here = window + kTable + lane * 4;
    int j = 0, cs = 0;                    // stages so far (all tiles), code stage
    uint32_t cph = 0, code_here = 0;
    for (int it = worker; it < total && ok; it += workers) {
      for (int kc = 0; kc < nkc && ok; ++kc) {
        if (!__all_sync(0xffffffffu, code_here)) ok = mx4_warp_wait(&code_full[cs], cph, gave_up, limit.tries);
        if (!ok) break;
        const uint8_t* st = codes_s + cs * kCodeStage;
        uint64_t* code_done = &code_empty[cs];
        if (++cs == kCodeStages) {
          cs = 0;
          cph ^= 1;
        }
        code_here = mx4_test(&code_full[cs], cph);
        const int steps = min(kSteps, nkb - kSteps * kc);
        for (int step = 0; step < steps && ok; ++step, ++j) {
          if (j % S::kGroups != group) continue;
          const int w = j % S::kW;
          const uint32_t w_free = mx4_test(&w_empty[w], ((j / S::kW) & 1) ^ 1);
#pragma unroll
          for (int i = 0; i < S::kSub; ++i) {
            const int q = step * S::kSub + i;
            const uint4 c0 = *reinterpret_cast<const uint4*>(st + row * 128 + (((2 * q) ^ (row & 7)) << 4));
            const uint4 c1 = *reinterpret_cast<const uint4*>(st + row * 128 + (((2 * q + 1) ^ (row & 7)) << 4));
            const uint32_t sw = *reinterpret_cast<const uint32_t*>(st + kCodeBytes + (q >> 1) * 512 + lane * 16 + quad * 4) >> (16 * (q & 1));
            const uint32_t b0 = sw & 255u, b1 = (sw >> 8) & 255u;
            const uint32_t c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
            uint32_t y[32];
#pragma unroll
            for (int e = 0; e < 8; ++e) look_up8(c[e], here, *reinterpret_cast<uint32_t(*)[4]>(y + 4 * e));
            // 2^(byte - 127) as a pair of bf16, 0: their subnormal 2^-127, 255: NaN
            const uint32_t f0 = b0 == 255u ? 0x7fff7fffu : (b0 == 0u ? 0x00400040u : b0 * 0x00800080u);
            const uint32_t f1 = b1 == 255u ? 0x7fff7fffu : (b1 == 0u ? 0x00400040u : b1 * 0x00800080u);
#pragma unroll
            for (int e = 0; e < 32; ++e) y[e] = mul_bf16x2(y[e], e < 16 ? f0 : f1);
            if (i == 0) {
              if (!__all_sync(0xffffffffu, w_free)) ok = mx4_warp_wait(&w_empty[w], ((j / S::kW) & 1) ^ 1, gave_up, limit.tries);
              if (!ok) break;
              tc_fence_after();
            }
            tmem_st_32x32b_x32(tmem + (static_cast<uint32_t>(quad * 32) << 16) + S::kWeights + 32 * (S::kSub * w + i), y);
          }
          if (!ok) break;
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_first(&w_full[w]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(code_done);
      }
    }
    if (!ok && lane == 0) tell();
    tc_fence_before();
  } else {
    const int quad = warp & 3, half = warp >> 2;
    int k = 0;
    for (int it = worker; it < total && ok; it += workers, ++k) {
      int n0, m0, count;
      tile_at(it, n0, m0, count);
      // all lanes or none: the TMEM loads need the whole warp
      ok = mx4_warp_wait(&acc_full[k & 1], (k >> 1) & 1, gave_up, limit.tries);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16) + (k & 1) * S::kAcc1;
      const int n = n0 + quad * 32 + lane;
      const float bias = p.bias && n < p.N ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]) : 0.f;
      const int first = S::kShared > 0 && (k & 1) == 0 ? BT - S::kShared : 0;      // the shared columns first
      bool told = false;
      auto free_acc = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && it + workers < total) arrive_first(&acc_free[S::kShared > 0 ? 0 : k & 1]);      // someone waits for it
        told = true;
      };
      mx4_with_epilogue(p, [&](auto epi) {
        constexpr int EPI = decltype(epi)::value;
#pragma unroll 1
        for (int i = half; i < BT / 16; i += 2) {
          const int c = S::kShared > 0 ? (first + 16 * i) & (BT - 1) : 16 * i;
          if (S::kShared > 0 && !told && i >= S::kShared / 16) free_acc();
          if (c >= count) continue;
          float r[16];
          tmem_ld_32x32b_x16(acc + c, reinterpret_cast<uint32_t*>(r));
          tmem_ld_wait();
          mx4_store_col<EPI>(p, x, r, m0 + c, m0 + count, n, bias);
        }
      });
      if (!told) free_acc();
    }
    if (!ok && lane == 0) tell();
    tc_fence_before();
  }
  __syncthreads();
  if (kPair) {
    if (tid == 0) {
      if (rank == 1) st_dsmem_u32(mapa_u32(smem_u32(const_cast<int*>(asked + 1)), 0), asked[0]);
      if (*gave_up) tell();      // both CTAs take the branch below, or neither does
    }
    __syncwarp();
    cluster_sync_all();
    if (*gave_up) {      // otherwise the products have consumed what was asked for, and the epilogues the products
      if (tid == 0) {
        if (rank == 0) mx4_settle_pair(tok_full, S::kTok, asked[0], asked[1], S::kSub * (pieces.per / 2) * 128);
        mbar_drain(drain_bar, 0);
      }
      __syncthreads();
      cluster_sync_all();
    }
  }
  if (warp == kMma) {
    tc_fence_after();
    if (kPair) tmem_dealloc_pair<S::kCols>(tmem);
    else tmem_dealloc<S::kCols>(tmem);
  }
  if (tid == 0 && *gave_up) {
    *failed = 1u;
    __threadfence_system();
  }
}

template <int BT, bool kPair>
int launch(const vila_mx4_linear_params& p, const vila_glinear_ext& x, const Pieces& pieces, int tries, cudaStream_t stream) {
  using S = Shape<BT, kPair>;
  constexpr int kCtas = kPair ? 2 : 1;
  static PerDeviceOnce once;
  VB_ALLOW_SMEM(once, mx4_mixed_kernel<BT, kPair>, static_cast<int>(kSmem));
  CUtensorMap tw, tx;
  if (int rc = make_tmap_2d_u8(&tw, p.w_codes, p.N, mx4_pitch(p.K), mx4_pitch(p.K), kRowsW, 128, 128)) return rc;
  if (int rc = make_tmap_2d_bf16(&tx, p.x, p.M, p.K, p.ldx, pieces.per / kCtas, kDepth, 128)) return rc;
  const long long tiles = static_cast<long long>((p.N + kCtas * kRowsW - 1) / (kCtas * kRowsW)) * pieces.n, most = num_sms() / kCtas;
  VB_CHECK(tiles < (1LL << 30), "mx4_linear: too many tiles (M=%d N=%d)", p.M, p.N);
  VB_CUDA(launch_serial_cluster(mx4_mixed_kernel<BT, kPair>, dim3(static_cast<unsigned>(kCtas * (tiles < most ? tiles : most))), dim3(S::kThreads), kSmem, stream,
                                dim3(kCtas), tw, tx, p, x, pieces, wait_limit(tries), failed_word()));
  return 0;
}

}  // namespace

bool mx4_mixed_tc_takes(const vila_mx4_linear_params& p) {      // what a tensor map of x needs
  return p.x != nullptr && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx % 8 == 0 && p.ldx >= p.K;
}

int mx4_mixed_tc(const vila_mx4_linear_params& p, const vila_glinear_ext& x, int tries, cudaStream_t stream) {
  VB_CHECK(failed_word() != nullptr, "mx4_linear: no pinned host memory for the status word");
  const int n_tiles = (p.N + kRowsW - 1) / kRowsW;
  Pieces pc;
  pc.n = (p.M + 255) / 256;
  while ((pc.n + 1) * n_tiles <= num_sms() && (p.M + pc.n) / (pc.n + 1) >= 48) ++pc.n;      // shorter tiles where SMs would stand idle
  pc.per = ((p.M + pc.n - 1) / pc.n + 15) & ~15;
  pc.n = (p.M + pc.per - 1) / pc.per;
  if (pc.per <= 64) return launch<64, false>(p, x, pc, tries, stream);
  if (pc.per <= 96) return launch<96, false>(p, x, pc, tries, stream);
  if (pc.per <= 128) return launch<128, false>(p, x, pc, tries, stream);
  pc.per = (pc.per + 31) & ~31;
  pc.n = (p.M + pc.per - 1) / pc.per;
  return launch<256, true>(p, x, pc, tries, stream);
}

}  // namespace vb
