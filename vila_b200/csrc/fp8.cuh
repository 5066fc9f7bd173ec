// 8-bit floating point rows with an fp32 scale per block of 128 ("Fp8"), shared by the kernels that make and read them.
//
// A block is 128 columns of one row (activations) or of 128 rows (weights): scale s = max(largest magnitude / 448, 2^-126), element = e4m3
// number nearest to x * (1 / s).  2^-126 keeps both quotients among the normal numbers.  include/vila_b200.h has the layouts.
#pragma once
#include <cuda_fp16.h>
#include "common.cuh"

namespace vb {

constexpr int kFp8Block = 128;
constexpr int kFp8Chunk = 16;      // columns of a lane: 16 bytes of codes; 8 neighbouring lanes hold a block

__host__ __device__ __forceinline__ int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }

// A block's scale and what its elements are multiplied with, from its largest magnitude's bits (magnitudes order as integers, NaN above infinity).
struct Fp8Scale {
  float scale, inv;
  bool fine;      // otherwise the block has an infinity or a NaN: its scale is a NaN, its codes are 0
};
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t top) {
  Fp8Scale s;
  s.fine = top < 0x7f800000u;
  const float v = fmaxf(__fdiv_rn(__uint_as_float(top), 448.f), 1.17549435e-38f);
  s.scale = s.fine ? v : __uint_as_float(0x7fffffffu);
  s.inv = s.fine ? __frcp_rn(v) : 0.f;
  return s;
}
// the largest magnitude of the 8 lanes that hold a block
__device__ __forceinline__ uint32_t fp8_top8(uint32_t top) {
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  return max(top, __shfl_xor_sync(0xffffffffu, top, 4));
}
// two numbers to e4m3, nearest, ties to even, at most 448; the first in the low byte
__device__ __forceinline__ uint32_t fp8_encode2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ uint32_t fp8_encode4(float a, float b, float c, float d) { return fp8_encode2(a, b) | fp8_encode2(c, d) << 16; }
// 16 numbers of a block to codes
__device__ __forceinline__ uint4 fp8_encode16(const float (&v)[16], const Fp8Scale& s) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = fp8_encode4(v[4 * i] * s.inv, v[4 * i + 1] * s.inv, v[4 * i + 2] * s.inv, v[4 * i + 3] * s.inv);
  return s.fine ? make_uint4(c[0], c[1], c[2], c[3]) : make_uint4(0u, 0u, 0u, 0u);
}
// the two numbers of a pair of codes
__device__ __forceinline__ float2 fp8_decode2(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// ---- products ----
// kind::f8f6f4, e4m3 x e4m3 -> fp32: [4,6) D is F32 (1)  [7,10) A, [10,13) B: E4M3 (0)  [17,23) N >> 3  [24,29) M >> 4
__host__ __device__ constexpr uint32_t fp8_idesc(uint32_t M, uint32_t N) { return (1u << 4) | ((N >> 3) << 17) | ((M >> 4) << 24); }
// d += a b, two numbers at a time
__device__ __forceinline__ void fp8_fma2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{.reg .b64 ra, rb, rd; mov.b64 ra, {%2,%3}; mov.b64 rb, {%4,%5}; mov.b64 rd, {%0,%1}; fma.rn.f32x2 rd, ra, rb, rd; "
      "mov.b64 {%0,%1}, rd;}"
      : "+f"(d0), "+f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// Both scales of a block's products, which are finite and not negative, or NaN.  A product past fp32's largest number is given as minus its 2^-128th:
// the sums that it is for go through fp8_widen first, so that sums of zero stay zero and what fp32 can hold is what it is.
__device__ __forceinline__ float fp8_both_scales(float a, float b) {
  const float s = a * b;
  return s > 3.40282347e38f ? -(a * 0x1p-64f * (b * 0x1p-64f)) : s;
}
__device__ __forceinline__ bool fp8_is_wide(float both) { return both < 0.f; }
// A block's sums of a warp's lanes in TMEM, `columns` from `at` on, times -2^128 where both(column) is wide.  In place and by a short loop: on the
// registers that the sums go to behind it, it made the kernel of CTA pairs spill.
template <typename F>
__device__ __forceinline__ void fp8_widen(uint32_t at, int columns, F&& both) {
#pragma unroll 1
  for (int c = 0; c < columns; c += 8) {
    float r[8];
    tmem_ld_32x32b_x8(at + c, reinterpret_cast<uint32_t*>(r));
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = fp8_is_wide(both(c + i)) ? r[i] * 0x1p64f * -0x1p64f : r[i];
    tmem_st_32x32b_x8(at + c, reinterpret_cast<uint32_t*>(r));
  }
  tmem_st_wait();
}

}  // namespace vb
