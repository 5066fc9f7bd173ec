// Rows to microscaled 4-bit numbers and back, and the order of the scales (mx4.cuh).
//
// Quantisation, per block of 32 columns with largest magnitude m: byte = max(floor(log2 m) - 2 + 127, 0) (2 is the exponent of
// 4-bit numbers' largest, 6 = 1.5 * 2^2), code = x * 2^(127 - byte) rounded to the nearest 4-bit number, ties to the even code,
// 6 beyond 6.  Both scalings are by powers of two and within fp32's range, so that the codes are those of the definition, bit by bit.
// A block with an infinity or a NaN has scale byte 255 and reads as NaN.
//
// A lane takes a block: its 32 columns are 64 or 128 consecutive bytes (32 at a load), its maximum needs no other lane, its codes are one
// store of 16 bytes, and the scales of four lanes are one word.  Bound by memory if the instructions allow it: a lane with 8 columns
// spent 14 instructions a column, most of them on what a block has once, and took 41 us for 18944 x 3584 where the bytes take 26.
// Rows off 16-byte boundaries are read and written 32 neighbours at a time and change hands in shared memory.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "dtype_any.cuh"
#include "kernels.h"
#include "mx4.cuh"

namespace vb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

enum { kApart = 0, kBy16 = 16, kBy32 = 32 };      // how rows lie: anywhere, on boundaries of 16 or 32 bytes

__device__ __forceinline__ void ldg32(const void* p, uint32_t* v) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p));
}
__device__ __forceinline__ void stg32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7]) : "memory");
}
template <bool kF32> struct Block {
  static constexpr int kWords = kF32 ? 32 : 16;
  uint32_t w[kWords];
};
// The blocks of a warp, lane l's in row r from column c0 on: words of `x` (r < 0: none).  stage: [32][kWords + 1] words.
template <bool kF32, int kHow>
__device__ __forceinline__ void load_block(const void* x, int64_t ldx, int r, int c0, int cols, int lane, uint32_t* stage, Block<kF32>& v) {
  constexpr int kWords = Block<kF32>::kWords, kSize = kF32 ? 4 : 2;
  const uint8_t* src = static_cast<const uint8_t*>(x) + (static_cast<int64_t>(r) * ldx + c0) * kSize;
  const int n = r < 0 ? 0 : cols - c0;
  if (kHow != kApart) {
    if (n >= 32) {
      if (kHow == kBy32) {
#pragma unroll
        for (int i = 0; i < kWords; i += 8) ldg32(src + i * 4, v.w + i);
      } else {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(v.w + i) = __ldg(reinterpret_cast<const uint4*>(src + i * 4));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if (kF32) v.w[i] = i < n ? ld_raw(src, 1, i) : 0u;
        else v.w[i] = (2 * i < n ? ld_raw(src, 0, 2 * i) : 0u) | (2 * i + 1 < n ? ld_raw(src, 0, 2 * i + 1) : 0u) << 16;
      }
    }
  } else {
    const unsigned long long at = reinterpret_cast<unsigned long long>(src);
    __syncwarp();
    uint32_t e[32];
#pragma unroll
    for (int b = 0; b < 32; ++b) {      // lane l fetches column l of block b, all blocks' on their way together
      const uint8_t* from = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, at, b));
      e[b] = lane < __shfl_sync(0xffffffffu, n, b) ? ld_raw(from, kF32 ? 1 : 0, lane) : 0u;
    }
#pragma unroll
    for (int b = 0; b < 32; ++b) {
      if (kF32) stage[b * (kWords + 1) + lane] = e[b];
      else reinterpret_cast<uint16_t*>(stage + b * (kWords + 1))[lane] = static_cast<uint16_t>(e[b]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kWords; ++i) v.w[i] = stage[lane * (kWords + 1) + i];
  }
}
template <bool kF32, int kHow>
__device__ __forceinline__ void store_block(void* out, int64_t ldo, int r, int c0, int cols, int lane, uint32_t* stage, const Block<kF32>& v) {
  constexpr int kWords = Block<kF32>::kWords, kSize = kF32 ? 4 : 2;
  uint8_t* dst = static_cast<uint8_t*>(out) + (static_cast<int64_t>(r) * ldo + c0) * kSize;
  const int n = r < 0 ? 0 : cols - c0;
  if (kHow != kApart) {
    if (n >= 32) {
      if (kHow == kBy32) {
#pragma unroll
        for (int i = 0; i < kWords; i += 8) stg32(dst + i * 4, v.w + i);
      } else {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) stg_v4(dst + i * 4, make_uint4(v.w[i], v.w[i + 1], v.w[i + 2], v.w[i + 3]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < n) {
          if (kF32) reinterpret_cast<uint32_t*>(dst)[i] = v.w[i % kWords];
          else reinterpret_cast<uint16_t*>(dst)[i] = static_cast<uint16_t>(v.w[i / 2] >> (16 * (i & 1)));
        }
    }
  } else {
    const unsigned long long at = reinterpret_cast<unsigned long long>(dst);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kWords; ++i) stage[lane * (kWords + 1) + i] = v.w[i];
    __syncwarp();
#pragma unroll 8
    for (int b = 0; b < 32; ++b) {
      uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, at, b));
      if (lane < __shfl_sync(0xffffffffu, n, b)) {
        if (kF32) reinterpret_cast<uint32_t*>(to)[lane] = stage[b * (kWords + 1) + lane];
        else reinterpret_cast<uint16_t*>(to)[lane] = reinterpret_cast<const uint16_t*>(stage + b * (kWords + 1))[lane];
      }
    }
  }
}

// Items are blocks: `per` a row (those of whole tiles of 256 columns), rows up to whole tiles of 128; those past the last row or column
// have a scale alone.  r0: the first row of this launch.
template <bool kF32, int kHow>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int r0, int rows, int cols, uint32_t items) {
  constexpr int kWords = Block<kF32>::kWords;
  __shared__ uint32_t stage_all[kHow == kApart ? kWarps * 32 * (kWords + 1) : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = mx4_pitch(cols), kts = mx4_ktiles(cols);
  const uint32_t per = kts * 4, step = gridDim.x * kThreads;
  uint32_t* stage = stage_all + (kHow == kApart ? warp * 32 * (kWords + 1) : 0);
  for (uint32_t it0 = blockIdx.x * kThreads + warp * 32; it0 < items; it0 += step) {      // items is a multiple of 32
    const uint32_t it = it0 + lane;
    const int rr = it / per, j = it - rr * per, r = r0 + rr;
    const bool there = r < rows && j * 32 < cols;
    Block<kF32> v;
    load_block<kF32, kHow>(x, ldx, there ? r : -1, j * 32, cols, lane, stage, v);
    uint32_t top = 0;                               // magnitudes order as integers, NaN above infinity
    if (kF32) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) top = max(top, v.w[i] & 0x7fffffffu);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) top = __vmaxu2(top, v.w[i] & 0x7fff7fffu);
      top = max(top << 16, top & 0xffff0000u);
    }
    const bool finite = top < 0x7f800000u;
    const uint32_t e = top >> 23, byte = finite ? (e > 2 ? e - 2 : 0u) : 255u;
    const float inv = __uint_as_float((254u - (finite ? byte : 0u)) << 23);
    uint32_t c[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t raw = v.w[kF32 ? 8 * g + i : 4 * g + i / 2];
        f[i] = (kF32 ? __uint_as_float(raw) : (i & 1 ? bf_hi(raw) : bf_lo(raw))) * inv;
      }
      c[g] = finite ? mx4_encode8(f) : 0u;
    }
    if (there) stg_v4(codes + static_cast<size_t>(r) * pitch + j * 16, make_uint4(c[0], c[1], c[2], c[3]));
    uint32_t word = there ? byte << (8 * (lane & 3)) : 0u;      // `it` and the lane agree on the block's place in its word: per is a multiple of 4
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    if ((lane & 3) == 0) *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(r, j >> 2, kts)) = word;
  }
}

// blocks of the rows alone: `per` a row, whole tiles of 256 columns again
template <bool kF32, int kHow>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t* codes, const uint8_t* scales, void* out, int64_t ldo, int r0, int rows, int cols, uint32_t items) {
  constexpr int kWords = Block<kF32>::kWords;
  __shared__ uint32_t stage_all[kHow == kApart ? kWarps * 32 * (kWords + 1) : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = mx4_pitch(cols), kts = mx4_ktiles(cols);
  const uint32_t per = kts * 4, step = gridDim.x * kThreads;
  uint32_t* stage = stage_all + (kHow == kApart ? warp * 32 * (kWords + 1) : 0);
  for (uint32_t it0 = blockIdx.x * kThreads + warp * 32; it0 < items; it0 += step) {
    const uint32_t it = it0 + lane;
    const int rr = it / per, j = it - rr * per, r = r0 + rr;
    const bool there = r < rows && j * 32 < cols;
    uint4 c4 = make_uint4(0u, 0u, 0u, 0u);
    uint32_t byte = 0;
    if (there) {
      c4 = __ldg(reinterpret_cast<const uint4*>(codes + static_cast<size_t>(r) * pitch + j * 16));
      byte = __ldg(scales + mx4_scale_at(r, j >> 2, kts) + (j & 3));
    }
    const float s = mx4_scale(byte);
    const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
    Block<kF32> v;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t h[4] = {mx4_pair_f16<0>(c[g]), mx4_pair_f16<1>(c[g]), mx4_pair_f16<2>(c[g]), mx4_pair_f16<3>(c[g])};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        if (kF32) {
          v.w[(8 * g + 2 * i) % kWords] = __float_as_uint(f.x * s);
          v.w[(8 * g + 2 * i + 1) % kWords] = __float_as_uint(f.y * s);
        } else {
          v.w[(4 * g + i) % kWords] = pack_bf16(f.x * s, f.y * s);
        }
      }
    }
    store_block<kF32, kHow>(out, ldo, there ? r : -1, j * 32, cols, lane, stage, v);
  }
}

// scales [rows, blocks] <-> the tiled order; a thread moves one word of the tiled order
__global__ void __launch_bounds__(kThreads)
scales_kernel(uint8_t* plain, uint8_t* tiled, int rows, int rows_padded, int cols, int to_tiled) {
  const int blocks = (cols + 31) / 32, kts = mx4_ktiles(cols);
  const long long items = static_cast<long long>(rows_padded) * kts, step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long it = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; it < items; it += step) {
    const int r = static_cast<int>(it / kts), kt = static_cast<int>(it - static_cast<long long>(r) * kts);
    uint32_t* w = reinterpret_cast<uint32_t*>(tiled + mx4_scale_at(r, kt, kts));
    uint8_t* p = plain + static_cast<size_t>(r) * blocks + kt * 4;
    const int n = r < rows ? min(4, blocks - kt * 4) : 0;
    uint32_t v = to_tiled ? 0u : *w;
    for (int i = 0; i < n; ++i) {
      if (to_tiled) v |= static_cast<uint32_t>(p[i]) << (8 * i);
      else p[i] = static_cast<uint8_t>(v >> (8 * i));
    }
    if (to_tiled) *w = v;
  }
}

int grid_for(long long warps_of_work) {
  const long long blocks = (warps_of_work + kWarps - 1) / kWarps, most = static_cast<long long>(num_sms()) * 8;
  return static_cast<int>(blocks < most ? blocks : most);
}
int how(const void* p, int64_t ld, int esize) {
  const uint64_t a = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(ld) * esize;
  return a % 32 == 0 ? kBy32 : (a % 16 == 0 ? kBy16 : kApart);
}
// f(first row, rows, items) for as many rows (whole tiles of 128) as items are counted in 32 bits
template <typename F>
int by_rows(int rows, int cols, F&& f) {
  const int64_t per = mx4_ktiles(cols) * 4ll;
  const int64_t most = (0xffff0000ll - 148 * 8 * kThreads * 8) / per / 128 * 128;      // below 2^32 with a grid's step to spare
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    if (int rc = f(static_cast<int>(r), static_cast<uint32_t>((n + 127) / 128 * 128 * per))) return rc;
  }
  return 0;
}
// x: the rows as numbers (or plain scale bytes), of `size` bytes each
int check_rows(const char* what, int rows, int cols, const uint8_t* codes, const uint8_t* scales, const void* x, int size) {
  VB_CHECK(rows >= 0 && cols > 0 && rows <= (1 << 30) && cols <= (1 << 25), "%s: rows=%d cols=%d", what, rows, cols);
  VB_CHECK(rows == 0 || (codes != nullptr && scales != nullptr && reinterpret_cast<uintptr_t>(codes) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(scales) % 16 == 0),
           "%s: codes and scales start on 16-byte boundaries", what);
  VB_CHECK(rows == 0 || (x != nullptr && reinterpret_cast<uintptr_t>(x) % size == 0), "%s: a null pointer, or one off its elements' boundaries", what);
  return 0;
}

}  // namespace

int mx4_quantize(const void* x, int dt, int64_t ldx, uint8_t* codes, uint8_t* scales, int rows, int cols, cudaStream_t stream) {
  VB_CHECK(dt == VILA_DT_BF16 || dt == VILA_DT_F32, "mx4_quantize: dtype code %d", dt);
  const bool f32 = dt == VILA_DT_F32;
  if (int rc = check_rows("mx4_quantize", rows, cols, codes, scales, x, f32 ? 4 : 2)) return rc;
  if (rows == 0) return 0;
  const int h = how(x, ldx, f32 ? 4 : 2);
  auto k = f32 ? (h == kBy32 ? quantize_kernel<true, kBy32> : (h == kBy16 ? quantize_kernel<true, kBy16> : quantize_kernel<true, kApart>))
               : (h == kBy32 ? quantize_kernel<false, kBy32> : (h == kBy16 ? quantize_kernel<false, kBy16> : quantize_kernel<false, kApart>));
  return by_rows(rows, cols, [&](int r0, uint32_t items) {
    VB_CUDA(launch_serial(k, dim3(grid_for(items / 32)), dim3(kThreads), 0, stream, x, ldx, codes, scales, r0, rows, cols, items));
    return 0;
  });
}

int mx4_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int dt, int64_t ldo, int rows, int cols, cudaStream_t stream) {
  VB_CHECK(dt == VILA_DT_BF16 || dt == VILA_DT_F32, "mx4_dequantize: dtype code %d", dt);
  const bool f32 = dt == VILA_DT_F32;
  if (int rc = check_rows("mx4_dequantize", rows, cols, codes, scales, out, f32 ? 4 : 2)) return rc;
  VB_CHECK(rows <= 1 || ldo >= cols, "mx4_dequantize: ldo=%lld cols=%d", static_cast<long long>(ldo), cols);
  if (rows == 0) return 0;
  const int h = how(out, ldo, f32 ? 4 : 2);
  auto k = f32 ? (h == kBy32 ? dequantize_kernel<true, kBy32> : (h == kBy16 ? dequantize_kernel<true, kBy16> : dequantize_kernel<true, kApart>))
               : (h == kBy32 ? dequantize_kernel<false, kBy32> : (h == kBy16 ? dequantize_kernel<false, kBy16> : dequantize_kernel<false, kApart>));
  return by_rows(rows, cols, [&](int r0, uint32_t items) {
    VB_CUDA(launch_serial(k, dim3(grid_for(items / 32)), dim3(kThreads), 0, stream, codes, scales, out, ldo, r0, rows, cols, items));
    return 0;
  });
}

int mx4_scales(uint8_t* plain, uint8_t* tiled, int rows, int cols, int to_tiled, cudaStream_t stream) {
  if (int rc = check_rows("mx4_scales", rows, cols, tiled, tiled, plain, 1)) return rc;
  if (rows == 0) return 0;
  const int padded = (rows + 127) / 128 * 128;
  const int grid = grid_for((static_cast<long long>(padded) * mx4_ktiles(cols) + 31) / 32);
  VB_CUDA(launch_serial(scales_kernel, dim3(grid), dim3(kThreads), 0, stream, plain, tiled, rows, padded, cols, to_tiled));
  return 0;
}

}  // namespace vb
