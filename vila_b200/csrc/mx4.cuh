// Microscaled 4-bit rows ("Mx4"), shared by the kernels that make and read them.
//
// A row is cut into blocks of 32 columns.  A block is one power of two 2^(byte - 127) and 32 numbers of 4 bits (sign, two
// exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6).
//   codes   [rows, 16 * blocks] bytes, the even column in a byte's low half; columns past the last one are 0
//   scales  in the order in which the tensor core wants them in TMEM, so that a stage of a product is one straight copy:
//           [row tiles of 128][column tiles of 128, an even number][32 rows r % 32][4 row groups r / 32][4 blocks]
//           (512 bytes a tile, a row's 4 blocks are one word).  Rows and blocks past the last ones are 0 (finite: a NaN there
//           would meet the zeros that TMA fills in).
#pragma once
#include "common.cuh"

namespace vb {

constexpr int kMx4Block = 32;
__host__ __device__ __forceinline__ int mx4_pitch(int cols) { return (cols + 31) / 32 * 16; }           // bytes of a row of codes
__host__ __device__ __forceinline__ int mx4_ktiles(int cols) { return (cols + 255) / 256 * 2; }
// where the word of row r's blocks 4 * kt .. 4 * kt + 3 starts
__host__ __device__ __forceinline__ size_t mx4_scale_at(int r, int kt, int ktiles) {
  return (static_cast<size_t>(r >> 7) * ktiles + kt) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}
__host__ __device__ __forceinline__ size_t mx4_scale_bytes(int rows, int cols) {
  return static_cast<size_t>((rows + 127) / 128) * mx4_ktiles(cols) * 512;
}

// a scale byte as a number: 2^(b - 127), 255: NaN
__device__ __forceinline__ float mx4_scale(uint32_t b) {
  return __uint_as_float(b == 255u ? 0x7fffffffu : (b == 0u ? 0x00400000u : b << 23));
}
// the number of a code
__device__ __forceinline__ float mx4_number(uint32_t c) {
  const uint32_t e = (c >> 1) & 3u, m = c & 1u;
  const float v = e == 0u ? 0.5f * m : __uint_as_float((126u + e) << 23 | m << 22);
  return c & 8u ? -v : v;
}
// the two numbers of byte `i` of w as f16 (exact), the low half's first
template <int kByte>
__device__ __forceinline__ uint32_t mx4_pair_f16(uint32_t w) {
  uint32_t d;
  if (kByte == 0)
    asm("{.reg .b8 a, b, c, e; mov.b32 {a, b, c, e}, %1; cvt.rn.f16x2.e2m1x2 %0, a;}" : "=r"(d) : "r"(w));
  else if (kByte == 1)
    asm("{.reg .b8 a, b, c, e; mov.b32 {a, b, c, e}, %1; cvt.rn.f16x2.e2m1x2 %0, b;}" : "=r"(d) : "r"(w));
  else if (kByte == 2)
    asm("{.reg .b8 a, b, c, e; mov.b32 {a, b, c, e}, %1; cvt.rn.f16x2.e2m1x2 %0, c;}" : "=r"(d) : "r"(w));
  else
    asm("{.reg .b8 a, b, c, e; mov.b32 {a, b, c, e}, %1; cvt.rn.f16x2.e2m1x2 %0, e;}" : "=r"(d) : "r"(w));
  return d;
}
// eight numbers, already divided by their block's scale, to 4 bits each: nearest, ties to the even code, at most 6
__device__ __forceinline__ uint32_t mx4_encode8(const float (&v)[8]) {
  uint32_t d;
  asm("{.reg .b8 a, b, c, e;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 e, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, e};}"
      : "=r"(d)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return d;
}

// A warp's wait on an mbarrier: every lane asks, and none leaves before the others.  Both are needed.  What a phase's end makes visible (bytes that
// TMA wrote, sums in TMEM) it makes visible to the lane that saw it, so that a lane which reads such bytes has to have asked itself.  And tcgen05's
// .sync.aligned instructions behind the wait are undefined for a warp that has parted, as it has where one lane polls in a loop of its own.
// Warps that issue tcgen05 instructions stay converged but for the one branch in which a lane issues them, which also takes less time than
// issuing from a lane on its own (8192 x 8192 x 8192 in 4 bits: 186 us and 254).
__device__ __forceinline__ bool mx4_warp_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up, int tries) {
  for (int i = 0; i < tries; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *gave_up != 0)) return false;
  }
  *gave_up = 1;
  return false;
}
// Whether an mbarrier's phase is over, without waiting for it.  The answer takes about 200 clocks: it is asked for a stage ahead, and the
// lanes vote on it (__all_sync) when they need it.
__device__ __forceinline__ uint32_t mx4_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{.reg .pred P; mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2; selp.u32 %0, 1, 0, P;}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok;
}
// Whether a warp of role `role` in CTA `rank` of a pair is to give up before its first wait (WaitLimit).
__device__ __forceinline__ bool mx4_pair_quits(const WaitLimit& limit, int role, int rank) {
  return limit.quits >= 0 && (limit.quits & 3) == role && ((limit.quits >> 2) == 0 || (limit.quits >> 2) == rank + 1);
}
// The end of a pair of which a warp gave up.  Both CTAs' loads of a stage report to the first CTA's barrier, which it arms for both.  Stages are
// asked for in order, stage j by barrier j % stages, and neither CTA gets more than a round ahead of what both have asked for (a stage is free
// once both CTAs' loads of it have been consumed).  `own` stages were asked for by the first CTA, `other` by the second; no more will be, as
// both CTAs' warps are behind a cluster barrier.  Stages that the second alone asked for are armed for its bytes; those that the first alone
// asked for no longer wait for the second's.  Then every barrier's last phase ends with the last byte that is on its way.
__device__ __forceinline__ void mx4_settle_pair(uint64_t* full, int stages, int own, int other, uint32_t second_bytes) {
  for (int j = own; j < other; ++j) mbar_arrive_expect_tx(&full[j % stages], second_bytes);
  for (int j = other; j < own; ++j) mbar_complete_tx(&full[j % stages], second_bytes);
  const int most = own > other ? own : other;
  for (int j = most - stages > 0 ? most - stages : 0; j < most; ++j) mbar_drain(&full[j % stages], (j / stages) & 1);
}
// consecutive bytes (a multiple of 16, on 16-byte boundaries)
__device__ __forceinline__ void mx4_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// How many clusters of a kernel the GPU holds at once, by cluster size (1, 2, 4, 8), asked for once a device: a cluster lies within a
// group of SMs, so that 28 clusters of 5 are more than the 148 SMs take at a time, and one too many takes as long again.  Host threads may ask
// at the same time; a question that fails is asked again by the next call.
struct Mx4Clusters {
  std::atomic<int> most[64][4] = {};      // 0: not asked yet, -1: none
  template <typename K>
  int of(K* kernel, int log2, int threads, size_t smem) {
    int d = 0;
    cudaGetDevice(&d);
    if (d < 0 || d >= 64) d = 0;
    int n = most[d][log2].load(std::memory_order_relaxed);
    if (n == 0) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u << log2);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 1u << log2;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        return -1;
      }
      if (n <= 0) n = -1;
      most[d][log2].store(n, std::memory_order_relaxed);
    }
    return n;
  }
  // the largest size (a power of two, at most 8 and `limit`) of which the GPU holds `tiles`; 1: none
  template <typename K>
  int split(K* kernel, int threads, size_t smem, long long tiles, long long limit) {
    int s = 1;
    for (int l = 1; l <= 3 && (2 << (l - 1)) <= limit && tiles <= of(kernel, l, threads, smem); ++l) s = 1 << l;
    return s;
  }
};

}  // namespace vb
