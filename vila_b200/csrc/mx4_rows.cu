// Linear layers of up to 8 bf16 rows on up to 16 M microscaled 4-bit weights (and, by tiles of 16 rows, of up to 16 on any, and of
// any off 16-byte boundaries, where the caller gives no workspace): out[m, n] = epi(sum_k x[m, k] w[n, k] + bias[n]).
//
// Bound by the stream of weights (17 bytes per 32 of them), or for the smallest layers by latency.  mma.sync m16n8k16 in f16: 16
// weight rows are the M side, 8 tokens the N side; tensor-core tiles of 128 tokens would stand empty here, and the sums of
// a block stay in registers, where its scale is applied.
//
//   weights   a 4-bit number is an f16 number as it is (cvt e2m1x2 -> f16x2); a block's 32 products per output are summed by two
//             mma from zero, then enter the row's fp32 sum times the block's scales: acc += (part * 2^t) * 2^e, 2^t the tokens', 2^e the
//             weights'.  No weight is rounded.  In this order, and with 2^-9 in the tokens' scale that the finished sum takes out again, no
//             scale leaves fp32's range before its result does: |part * 2^t| is below 32 * 6 * 2^128 * 2^-9 < 2^127, and it is a multiple of
//             2^-143 (bf16's least step, half a unit of a weight, the 2^-9), which fp32 holds.
//   tokens    f16 too, scaled per block by a power of two that brings its largest magnitude to 2^14 .. 2^15: bf16's 8 bits
//             fit f16's 11, and what is 2^29 times smaller than that largest is rounded to multiples of 2^-39 of it, under
//             the rounding of the fp32 sum (a block's weights differ by 12 at most).
//   columns   lane t of a quad takes columns 8 t .. 8 t + 7 of a block, of weights and tokens alike (the order within a sum is
//             free): one word of codes per row and block, one 16-byte load of tokens
//   warps     a warp owns 16 rows of a tile of 128 (rows r % 32 = 4 w .. 4 w + 3: their scale words are 64 consecutive bytes) and
//             streams them through a ring of its own with cp.async: no barrier among warps but around the tokens
//   K         split over a cluster of up to 8 CTAs where the row tiles do not fill the GPU; the parts are added in rank order
//             through distributed shared memory, so that a result does not depend on timing
#include <cuda_fp16.h>

#include "../../include/vila_b200.h"
#include "common.cuh"
#include "glinear_epi.cuh"
#include "kernels.h"
#include "mma_bf16.cuh"
#include "mx4.cuh"

namespace vb {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kRows = 128;                       // weight rows of a CTA
constexpr int kStages = 6;                       // of a warp's ring, 128 columns each
constexpr int kStage = 16 * 64 + 64;             // 16 rows of codes, their scale words
constexpr int kTokBytes = 36 * 1024;             // of tokens that are in shared memory at a time

// Columns whose tokens fit: all of a CTA's, if they do (one token: up to 16384)
__host__ __device__ __forceinline__ int chunk_of(int tokens, int columns) {
  const int most = (kTokBytes / tokens - 64) * 8 / 17 / 256 * 256;      // 2 bytes a column, 4 a block (and 64 bytes a row)
  return columns < most ? (columns + 255) / 256 * 256 : most;
}
template <int TM> struct Smem {
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kRed = kRows * (TM + 1) * 4;
  static constexpr int kTotal = kTokBytes + kRing + kRed;
};

constexpr int kUnits = 9;      // the sums are held in units of 2^kUnits

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// the scales of two neighbouring blocks (bytes 2 h, 2 h + 1 of a scale word)
__device__ __forceinline__ void scales2(uint32_t word, int h, float& s0, float& s1) {
  uint32_t d;
  const uint16_t two = static_cast<uint16_t>(word >> (16 * h));
  asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(d) : "h"(two));
  s0 = bf_lo(d);
  s1 = bf_hi(d);
}

// The tokens of columns [k0, k0 + chunk) as f16, with their scales; a warp takes 256 columns of a token, a lane 8.
template <int TM>
__device__ __forceinline__ void stage_tokens(const vila_mx4_linear_params& p, int m0, int k0, int k1, int chunk, __half* tok, float* tok_scale) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tokens = min(TM, p.M - m0);
  const int pieces = (min(k1 - k0, chunk) + 255) / 256, pitch16 = chunk + 32;      // 64 bytes off the bank of the row before
  for (int it = warp; it < tokens * pieces; it += kWarps) {
    const int m = it / pieces, c = (it - m * pieces) * 256 + lane * 8, k = k0 + c;
    uint32_t h[4];
    const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(p.x) + static_cast<size_t>(m0 + m) * p.ldx;
    float v[8];
    if (k + 8 <= p.K && ((reinterpret_cast<uintptr_t>(p.x) | (p.ldx * 2)) & 15) == 0) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + k));
      v[0] = bf_lo(a.x); v[1] = bf_hi(a.x); v[2] = bf_lo(a.y); v[3] = bf_hi(a.y);
      v[4] = bf_lo(a.z); v[5] = bf_hi(a.z); v[6] = bf_lo(a.w); v[7] = bf_hi(a.w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = k + i < p.K ? __bfloat162float(row[k + i]) : 0.f;
    }
    uint32_t top = 0;      // of the finite ones: infinities and NaN stay what they are
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
      top = max(top, a < 0x7f800000u ? a : 0u);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int up = min(127, 14 + 127 - static_cast<int>(top >> 23));    // >= -113
    const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 q = __floats2half2_rn(v[2 * i] * f, v[2 * i + 1] * f);
      h[i] = *reinterpret_cast<const uint32_t*>(&q);
    }
    const float back = __uint_as_float(static_cast<uint32_t>(141 - up) << 23) * 0x1p-23f;      // 2^(-up - kUnits): 141 - up is 14 .. 254
    *reinterpret_cast<uint4*>(tok + m * pitch16 + c) = make_uint4(h[0], h[1], h[2], h[3]);
    if ((lane & 3) == 0) tok_scale[(c >> 5) * tokens + m] = back;
  }
}

template <int TM>
__global__ void __launch_bounds__(kThreads)
mx4_rows_kernel(const vila_mx4_linear_params p, const vila_glinear_ext ext, int split) {
  constexpr int NT = TM / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring_all = smem + kTokBytes;
  float* red = reinterpret_cast<float*>(ring_all + Smem<TM>::kRing);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(blockIdx.x) % split, n0 = static_cast<int>(blockIdx.x) / split * kRows, m0 = blockIdx.y * TM;
  const int pitch = mx4_pitch(p.K), kts = mx4_ktiles(p.K), nk = (p.K + 127) / 128;
  const int kt0 = static_cast<int>(static_cast<long long>(nk) * rank / split), kt1 = static_cast<int>(static_cast<long long>(nk) * (rank + 1) / split);
  uint8_t* ring = ring_all + warp * (kStages * kStage);
  const int tokens = min(TM, p.M - m0), chunk = chunk_of(tokens, (kt1 - kt0) * 128), tok_pitch = chunk + 32;
  __half* tok = reinterpret_cast<__half*>(smem);
  float* tok_scale = reinterpret_cast<float*>(smem + tokens * tok_pitch * 2);

  // this lane's part of a stage: two pieces of codes (rows i0, i0 + 8 of the warp's 16), lanes 0 .. 3 one of scales
  const int i0 = lane >> 2, b0 = lane & 3;
  auto row_of = [&](int i) { return n0 + 4 * warp + (i & 3) + 32 * (i >> 2); };
  const uint8_t *src0 = p.w_codes + static_cast<size_t>(row_of(i0)) * pitch + b0 * 16, *src1 = p.w_codes + static_cast<size_t>(row_of(i0 + 8)) * pitch + b0 * 16;
  const bool ok0 = row_of(i0) < p.N, ok1 = row_of(i0 + 8) < p.N;
  const uint8_t* src_s = p.w_scales + mx4_scale_at(n0 + 4 * warp + (lane & 3), 0, kts);
  const uint32_t ring_a = smem_u32(ring);
  const uint32_t dst0 = ring_a + i0 * 64 + ((b0 ^ ((i0 >> 1) & 3)) << 4), dst1 = dst0 + 8 * 64, dst_s = ring_a + 1024 + lane * 16;
  auto fetch = [&](int kt, int stage) {
    if (kt < kt1) {
      const bool in = kt * 64 + b0 * 16 < pitch;
      const uint32_t o = stage * kStage;
      cp16(dst0 + o, ok0 && in ? src0 + kt * 64 : p.w_codes, ok0 && in);
      cp16(dst1 + o, ok1 && in ? src1 + kt * 64 : p.w_codes, ok1 && in);
      if (lane < 4) cp16(dst_s + o, src_s + static_cast<size_t>(kt) * 512, true);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fetch(kt0 + s, s);

  // this lane's token of an operand and its two of a sum; columns past the last token repeat it and are not read
  int row[NT], col0[NT], col1[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    row[j] = min(j * 8 + g, tokens - 1) * tok_pitch;
    col0[j] = min(j * 8 + 2 * t, tokens - 1);
    col1[j] = min(j * 8 + 2 * t + 1, tokens - 1);
  }
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;

  int stage = 0;
  for (int kc = kt0; kc < kt1; kc += chunk / 128) {
    if (kc != kt0) __syncthreads();
    stage_tokens<TM>(p, m0, kc * 128, kt1 * 128, chunk, tok, tok_scale);
    __syncthreads();
    const int kend = min(kt1, kc + chunk / 128);
    for (int kt = kc; kt < kend; ++kt) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();
      {
        const int next = stage == 0 ? kStages - 1 : stage - 1;      // the stage that was read last
        fetch(kt + kStages - 1, next);
      }
      const uint8_t* st = ring + stage * kStage;
      const uint32_t sw0 = *reinterpret_cast<const uint32_t*>(st + 1024 + (g & 3) * 16 + (g >> 2) * 4);
      const uint32_t sw1 = *reinterpret_cast<const uint32_t*>(st + 1024 + (g & 3) * 16 + (g >> 2) * 4 + 8);
      float ws0[4], ws1[4];
      scales2(sw0, 0, ws0[0], ws0[1]);
      scales2(sw0, 1, ws0[2], ws0[3]);
      scales2(sw1, 0, ws1[0], ws1[1]);
      scales2(sw1, 1, ws1[2], ws1[3]);
      const __half* tk = tok + (kt - kc) * 128 + t * 8;
      const float* ts = tok_scale + (kt - kc) * 4 * tokens;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(st + g * 64 + ((b ^ ((g >> 1) & 3)) << 4) + t * 4);
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(st + g * 64 + 512 + ((b ^ ((g >> 1) & 3)) << 4) + t * 4);
        const uint32_t a00 = mx4_pair_f16<0>(w0), a01 = mx4_pair_f16<1>(w0), a02 = mx4_pair_f16<2>(w0), a03 = mx4_pair_f16<3>(w0);
        const uint32_t a10 = mx4_pair_f16<0>(w1), a11 = mx4_pair_f16<1>(w1), a12 = mx4_pair_f16<2>(w1), a13 = mx4_pair_f16<3>(w1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 x = *reinterpret_cast<const uint4*>(tk + row[j] + b * 32);
          float part[4];
          mma_f16_first(part, a00, a10, a01, a11, x.x, x.y);
          mma_f16(part, a02, a12, a03, a13, x.z, x.w);
          const float2 xs = make_float2(ts[b * tokens + col0[j]], ts[b * tokens + col1[j]]);
          acc[j][0] = fmaf(part[0] * xs.x, ws0[b], acc[j][0]);
          acc[j][1] = fmaf(part[1] * xs.y, ws0[b], acc[j][1]);
          acc[j][2] = fmaf(part[2] * xs.x, ws1[b], acc[j][2]);
          acc[j][3] = fmaf(part[3] * xs.y, ws1[b], acc[j][3]);
        }
      }
      __syncwarp();       // the stage is free
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // sums by row of the tile, then every rank of the cluster finishes its share of the rows
  auto local = [&](int i) { return 4 * warp + (i & 3) + 32 * (i >> 2); };
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* r0 = red + local(g) * (TM + 1) + j * 8 + t * 2;
    float* r1 = red + local(g + 8) * (TM + 1) + j * 8 + t * 2;
    r0[0] = acc[j][0];
    r0[1] = acc[j][1];
    r1[0] = acc[j][2];
    r1[1] = acc[j][3];
  }
  if (split > 1) cluster_sync_all();
  else __syncthreads();
  const int share = kRows / split, first = rank * share;
  const uint32_t red_a = smem_u32(red);
  const bool gated = (p.flags & kGluFlags) != 0;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
  auto total = [&](int row, int m) {
    if (split == 1) return red[row * (TM + 1) + m] * static_cast<float>(1 << kUnits);
    float v = 0.f;
    for (int q = 0; q < split; ++q) v += ld_dsmem_f32(mapa_u32(red_a + (row * (TM + 1) + m) * 4, q));
    return v * static_cast<float>(1 << kUnits);
  };
  const int per = gated ? share / 2 : share;
  for (int i = tid; i < per * tokens; i += kThreads) {
    const int m = i / per, j = i - m * per;
    if (gated) {
      const int row = first + 2 * j, n = n0 + row;
      if (n >= p.N) continue;      // N is even
      const float zg = total(row, m) + (bias ? __bfloat162float(bias[n]) : 0.f);
      const float zu = total(row + 1, m) + (bias ? __bfloat162float(bias[n + 1]) : 0.f);
      out[static_cast<size_t>(m0 + m) * p.ldo + n / 2] = __float2bfloat16_rn(glu(zg, zu, p.flags, ext));
    } else {
      const int row = first + j, n = n0 + row;
      if (n >= p.N) continue;
      const float z = total(row, m) + (bias ? __bfloat162float(bias[n]) : 0.f);
      out[static_cast<size_t>(m0 + m) * p.ldo + n] = __float2bfloat16_rn(activate(z, p.act, ext));
    }
  }
  if (split > 1) cluster_sync_all();      // the others still read this CTA's sums
}

template <int TM>
int launch(const vila_mx4_linear_params& p, const vila_glinear_ext& ext, cudaStream_t stream) {
  static PerDeviceOnce once;
  VB_ALLOW_SMEM(once, mx4_rows_kernel<TM>, Smem<TM>::kTotal);
  const int tiles = (p.N + kRows - 1) / kRows, groups = (p.M + TM - 1) / TM, nk = (p.K + 127) / 128;
  static Mx4Clusters clusters;
  const int split = clusters.split(mx4_rows_kernel<TM>, kThreads, Smem<TM>::kTotal, static_cast<long long>(tiles) * groups, nk / 2);
  VB_CHECK(groups <= 65535 && static_cast<long long>(tiles) * split < (1LL << 31), "mx4_linear: M=%d N=%d", p.M, p.N);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * split, groups, 1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<TM>::kTotal;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  VB_CUDA(cudaLaunchKernelEx(&cfg, mx4_rows_kernel<TM>, p, ext, split));
  return 0;
}

}  // namespace

int mx4_rows(const vila_mx4_linear_params& p, const vila_glinear_ext& ext, cudaStream_t stream) {
  return p.M <= 8 ? launch<8>(p, ext, stream) : launch<16>(p, ext, stream);
}

}  // namespace vb
