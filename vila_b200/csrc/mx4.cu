// Rows to microscaled 4-bit numbers and back, and the order of the scales (mx4.cuh).
//
// Quantisation, per block of 32 columns with largest magnitude m: byte = max(floor(log2 m) - 2 + 127, 0) (2 is the exponent of
// 4-bit numbers' largest, 6 = 1.5 * 2^2), code = x * 2^(127 - byte) rounded to the nearest 4-bit number, ties to the even code,
// 6 beyond 6.  Both scalings are by powers of two and within fp32's range, so that the codes are those of the definition, bit by bit.
// A block with an infinity or a NaN has scale byte 255 and reads as NaN.
//
// A warp takes 1024 columns of a row, 256 at a time, a lane 8 consecutive ones: four lanes are a block, whose maximum is two
// shuffles away, and the codes of 256 columns are 128 consecutive bytes.  Bound by memory: each byte is read and written once, the
// four loads of a warp are under way together.  Rows off 16-byte boundaries are read and written a lane an element, next to its neighbours',
// and change hands in shared memory.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "dtype_any.cuh"
#include "kernels.h"
#include "mx4.cuh"

namespace vb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kUnroll = 4;

// 8 consecutive elements of a lane, raw; 0 past the row's end
template <bool kF32> struct Raw {
  uint32_t w[kF32 ? 8 : 4];
  __device__ __forceinline__ float at(int i) const {
    return kF32 ? __uint_as_float(w[i]) : (i & 1 ? bf_hi(w[i / 2]) : bf_lo(w[i / 2]));
  }
};
template <bool kF32, bool kVec>
__device__ __forceinline__ void load8(const void* x, size_t row_off, int c256, int cols, int lane, uint32_t* stage, Raw<kF32>& v) {
  const int c0 = c256 + lane * 8;
  if (kVec) {
    if (c0 + 8 <= cols) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + (row_off + c0) * (kF32 ? 4 : 2));
      *reinterpret_cast<uint4*>(v.w) = __ldg(p);
      if (kF32) *reinterpret_cast<uint4*>(v.w + 4) = __ldg(p + 1);
    } else if (kF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v.w[i] = c0 + i < cols ? ld_raw(x, 1, row_off + c0 + i) : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v.w[i] = (c0 + 2 * i < cols ? ld_raw(x, 0, row_off + c0 + 2 * i) : 0u) | (c0 + 2 * i + 1 < cols ? ld_raw(x, 0, row_off + c0 + 2 * i + 1) : 0u) << 16;
    }
  } else {
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c256 + i * 32 + lane < cols ? ld_raw(x, kF32 ? 1 : 0, row_off + c256 + i * 32 + lane) : 0u;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (kF32) stage[i * 32 + lane] = e[i];
      else reinterpret_cast<uint16_t*>(stage)[i * 32 + lane] = static_cast<uint16_t>(e[i]);
    }
    __syncwarp();
    *reinterpret_cast<uint4*>(v.w) = *reinterpret_cast<const uint4*>(stage + lane * (kF32 ? 8 : 4));
    if (kF32) *reinterpret_cast<uint4*>(v.w + 4) = *reinterpret_cast<const uint4*>(stage + lane * 8 + 4);
  }
}

// grid: rows by warps (strided), columns by 1024 in y
template <bool kF32, bool kVec>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int rows, int rows_padded, int cols) {
  __shared__ __align__(16) uint32_t stage_all[kVec ? 1 : kWarps * 256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = mx4_pitch(cols), chunks = (cols + 255) / 256;
  uint32_t* stage = stage_all + (kVec ? 0 : warp * 256);
  const int ch0 = blockIdx.y * kUnroll, n = min(kUnroll, chunks - ch0);
  for (int r = blockIdx.x * kWarps + warp; r < rows_padded; r += gridDim.x * kWarps) {
    Raw<kF32> v[kUnroll];
    if (r < rows)
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
        if (j < n) load8<kF32, kVec>(x, static_cast<size_t>(r) * ldx, (ch0 + j) * 256, cols, lane, stage, v[j]);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      if (j >= n) break;
      const int ch = ch0 + j;
      uint32_t word = 0;
      if (r < rows) {
        uint32_t top = 0;                               // magnitudes order as integers, NaN above infinity
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f[i] = v[j].at(i);
          top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool finite = top < 0x7f800000u;
        const uint32_t e = top >> 23, byte = finite ? (e > 2 ? e - 2 : 0u) : 255u;
        const float inv = __uint_as_float((254u - (finite ? byte : 0u)) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = finite ? f[i] * inv : 0.f;
        const uint32_t c = mx4_encode8(f);
        const int at = ch * 128 + lane * 4;
        if (at < pitch) *reinterpret_cast<uint32_t*>(codes + static_cast<size_t>(r) * pitch + at) = c;
        word = byte << (8 * ((lane >> 2) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
      }
      if ((lane & 15) == 0)
        *reinterpret_cast<uint32_t*>(scales + mx4_scale_at(r, 2 * ch + (lane >> 4), 2 * chunks)) = word;
    }
  }
}

template <bool kF32, bool kVec>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t* codes, const uint8_t* scales, void* out, int64_t ldo, int rows, int cols) {
  __shared__ __align__(16) uint32_t stage_all[kVec ? 1 : kWarps * 256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = mx4_pitch(cols), chunks = (cols + 255) / 256;
  uint32_t* stage = stage_all + (kVec ? 0 : warp * 256);
  const int ch0 = blockIdx.y * kUnroll, n = min(kUnroll, chunks - ch0);
  for (int r = blockIdx.x * kWarps + warp; r < rows; r += gridDim.x * kWarps) {
    uint32_t c[kUnroll], b[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int ch = ch0 + j, at = ch * 128 + lane * 4;
      c[j] = j < n && at < pitch ? __ldg(reinterpret_cast<const uint32_t*>(codes + static_cast<size_t>(r) * pitch + at)) : 0u;
      b[j] = j < n ? __ldg(scales + mx4_scale_at(r, 2 * ch + (lane >> 4), 2 * chunks) + ((lane >> 2) & 3)) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      if (j >= n) break;
      const float s = mx4_scale(b[j]);
      const uint32_t h[4] = {mx4_pair_f16<0>(c[j]), mx4_pair_f16<1>(c[j]), mx4_pair_f16<2>(c[j]), mx4_pair_f16<3>(c[j])};
      uint32_t v[kF32 ? 8 : 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        if (kF32) {
          v[2 * i] = __float_as_uint(f.x * s);
          v[(2 * i + 1) % (kF32 ? 8 : 4)] = __float_as_uint(f.y * s);
        } else {
          v[i] = pack_bf16(f.x * s, f.y * s);
        }
      }
      const int c256 = (ch0 + j) * 256, c0 = c256 + lane * 8;
      const size_t o = static_cast<size_t>(r) * ldo;
      if (kVec) {
        if (c0 + 8 <= cols) {
          uint4* p = reinterpret_cast<uint4*>(static_cast<uint8_t*>(out) + (o + c0) * (kF32 ? 4 : 2));
          p[0] = make_uint4(v[0], v[1], v[2], v[3]);
          if (kF32) p[1] = make_uint4(v[4 % (kF32 ? 8 : 4)], v[5 % (kF32 ? 8 : 4)], v[6 % (kF32 ? 8 : 4)], v[7 % (kF32 ? 8 : 4)]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c0 + i < cols) {
              if (kF32) static_cast<uint32_t*>(out)[o + c0 + i] = v[i % (kF32 ? 8 : 4)];
              else static_cast<uint16_t*>(out)[o + c0 + i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
            }
        }
      } else {
        __syncwarp();
        *reinterpret_cast<uint4*>(stage + lane * (kF32 ? 8 : 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        if (kF32)
          *reinterpret_cast<uint4*>(stage + lane * 8 + 4) =
              make_uint4(v[4 % (kF32 ? 8 : 4)], v[5 % (kF32 ? 8 : 4)], v[6 % (kF32 ? 8 : 4)], v[7 % (kF32 ? 8 : 4)]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = c256 + i * 32 + lane;
          if (col < cols) {
            if (kF32) static_cast<uint32_t*>(out)[o + col] = stage[i * 32 + lane];
            else static_cast<uint16_t*>(out)[o + col] = reinterpret_cast<const uint16_t*>(stage)[i * 32 + lane];
          }
        }
      }
    }
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
// rows by warps in x, 1024 columns in y; x strides over the rows where there are many
dim3 grid_of(int rows, int cols) {
  const int y = (cols + 256 * kUnroll - 1) / (256 * kUnroll);
  const int blocks = (rows + kWarps - 1) / kWarps, most = (num_sms() * 8 + y - 1) / y;
  return dim3(blocks < most ? blocks : most, y);
}
bool aligned(const void* p, int64_t ld, int esize) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0; }
int check_rows(const char* what, int rows, int cols, const uint8_t* codes, const uint8_t* scales) {
  VB_CHECK(rows >= 0 && cols > 0 && rows <= (1 << 30) && cols <= (1 << 25), "%s: rows=%d cols=%d", what, rows, cols);
  VB_CHECK(rows == 0 || (codes != nullptr && scales != nullptr && reinterpret_cast<uintptr_t>(codes) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(scales) % 16 == 0),
           "%s: codes and scales start on 16-byte boundaries", what);
  return 0;
}

}  // namespace

int mx4_quantize(const void* x, int dt, int64_t ldx, uint8_t* codes, uint8_t* scales, int rows, int cols, cudaStream_t stream) {
  if (int rc = check_rows("mx4_quantize", rows, cols, codes, scales)) return rc;
  VB_CHECK(dt == VILA_DT_BF16 || dt == VILA_DT_F32, "mx4_quantize: dtype code %d", dt);
  if (rows == 0) return 0;
  const int padded = (rows + 127) / 128 * 128;
  const bool f32 = dt == VILA_DT_F32, vec = aligned(x, ldx, f32 ? 4 : 2);
  auto k = f32 ? (vec ? quantize_kernel<true, true> : quantize_kernel<true, false>)
               : (vec ? quantize_kernel<false, true> : quantize_kernel<false, false>);
  VB_CUDA(launch_serial(k, grid_of(padded, cols), dim3(kThreads), 0, stream, x, ldx, codes, scales, rows, padded, cols));
  return 0;
}

int mx4_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int dt, int64_t ldo, int rows, int cols, cudaStream_t stream) {
  if (int rc = check_rows("mx4_dequantize", rows, cols, codes, scales)) return rc;
  VB_CHECK(dt == VILA_DT_BF16 || dt == VILA_DT_F32, "mx4_dequantize: dtype code %d", dt);
  if (rows == 0) return 0;
  const bool f32 = dt == VILA_DT_F32, vec = aligned(out, ldo, f32 ? 4 : 2);
  auto k = f32 ? (vec ? dequantize_kernel<true, true> : dequantize_kernel<true, false>)
               : (vec ? dequantize_kernel<false, true> : dequantize_kernel<false, false>);
  VB_CUDA(launch_serial(k, grid_of(rows, cols), dim3(kThreads), 0, stream, codes, scales, out, ldo, rows, cols));
  return 0;
}

int mx4_scales(uint8_t* plain, uint8_t* tiled, int rows, int cols, int to_tiled, cudaStream_t stream) {
  if (int rc = check_rows("mx4_scales", rows, cols, tiled, tiled)) return rc;
  if (rows == 0) return 0;
  const int padded = (rows + 127) / 128 * 128;
  const int grid = grid_for((static_cast<long long>(padded) * mx4_ktiles(cols) + 31) / 32);
  VB_CUDA(launch_serial(scales_kernel, dim3(grid), dim3(kThreads), 0, stream, plain, tiled, rows, padded, cols, to_tiled));
  return 0;
}

}  // namespace vb
