// Rows to microscaled 4-bit numbers and back, and the order of the scales (mx4.cuh).
//
// Quantisation, per block of 32 columns with largest magnitude m: byte = max(floor(log2 m) - 2 + 127, 0) (2 is the exponent of
// 4-bit numbers' largest, 6 = 1.5 * 2^2), code = x * 2^(127 - byte) rounded to the nearest 4-bit number, ties to the even code,
// 6 beyond 6.  Both scalings are by powers of two and within fp32's range, so that the codes are those of the definition, bit by bit.
// A block with an infinity or a NaN has scale byte 255 and reads as NaN.
//
// One warp takes 256 columns of a row, a lane 8 consecutive ones: four lanes are a block, whose maximum is two shuffles away,
// and the codes of a warp are 128 consecutive bytes.  Bound by memory: it reads and writes each byte once.
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "dtype_any.cuh"
#include "kernels.h"
#include "mx4.cuh"

namespace vb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// 8 consecutive elements from column c0 on, 0 past the row's end
template <bool kF32, bool kVec>
__device__ __forceinline__ void load8(const void* x, size_t row_off, int c0, int cols, float (&v)[8]) {
  if (kVec && c0 + 8 <= cols) {
    if (kF32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + row_off + c0);
      const float4 a = __ldg(p), b = __ldg(p + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(x) + row_off + c0));
      v[0] = bf_lo(a.x); v[1] = bf_hi(a.x); v[2] = bf_lo(a.y); v[3] = bf_hi(a.y);
      v[4] = bf_lo(a.z); v[5] = bf_hi(a.z); v[6] = bf_lo(a.w); v[7] = bf_hi(a.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? ld_any(x, kF32 ? 1 : 0, row_off + c0 + i) : 0.f;
  }
}

template <bool kF32, bool kVec>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int rows, int rows_padded, int cols) {
  const int lane = threadIdx.x & 31, pitch = mx4_pitch(cols), chunks = (cols + 255) / 256;
  const long long items = static_cast<long long>(rows_padded) * chunks, step = static_cast<long long>(gridDim.x) * kWarps;
  for (long long it = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5); it < items; it += step) {
    const int r = static_cast<int>(it / chunks), ch = static_cast<int>(it - static_cast<long long>(r) * chunks);
    uint32_t word = 0;
    if (r < rows) {
      float v[8];
      load8<kF32, kVec>(x, static_cast<size_t>(r) * ldx, ch * 256 + lane * 8, cols, v);
      uint32_t top = 0;                               // magnitudes order as integers, NaN above infinity
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool finite = top < 0x7f800000u;
      const uint32_t e = top >> 23, byte = finite ? (e > 2 ? e - 2 : 0u) : 255u;
      const float inv = __uint_as_float((254u - (finite ? byte : 0u)) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = finite ? v[i] * inv : 0.f;
      const uint32_t c = mx4_encode8(v);
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

template <bool kF32, bool kVec>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t* codes, const uint8_t* scales, void* out, int64_t ldo, int rows, int cols) {
  const int lane = threadIdx.x & 31, pitch = mx4_pitch(cols), chunks = (cols + 255) / 256;
  const long long items = static_cast<long long>(rows) * chunks, step = static_cast<long long>(gridDim.x) * kWarps;
  for (long long it = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5); it < items; it += step) {
    const int r = static_cast<int>(it / chunks), ch = static_cast<int>(it - static_cast<long long>(r) * chunks);
    const int at = ch * 128 + lane * 4, c0 = ch * 256 + lane * 8;
    if (at >= pitch) continue;
    const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(codes + static_cast<size_t>(r) * pitch + at));
    const float s = mx4_scale(__ldg(scales + mx4_scale_at(r, 2 * ch + (lane >> 4), 2 * chunks) + ((lane >> 2) & 3)));
    const uint32_t h[4] = {mx4_pair_f16<0>(c), mx4_pair_f16<1>(c), mx4_pair_f16<2>(c), mx4_pair_f16<3>(c)};
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
    const size_t o = static_cast<size_t>(r) * ldo + c0;
    if (kVec && c0 + 8 <= cols) {
      if (kF32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + o);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        stg_v4(static_cast<__nv_bfloat16*>(out) + o,
               make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < cols) st_any(out, kF32 ? 1 : 0, o + i, v[i]);
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
bool aligned(const void* p, int64_t ld, int esize) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0; }
int check_rows(const char* what, int rows, int cols, const uint8_t* codes, const uint8_t* scales) {
  VB_CHECK(rows >= 0 && cols > 0 && rows <= (1 << 30) && cols <= (1 << 30), "%s: rows=%d cols=%d", what, rows, cols);
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
  const int grid = grid_for(static_cast<long long>(padded) * ((cols + 255) / 256));
  const bool f32 = dt == VILA_DT_F32, vec = aligned(x, ldx, f32 ? 4 : 2);
  auto k = f32 ? (vec ? quantize_kernel<true, true> : quantize_kernel<true, false>)
               : (vec ? quantize_kernel<false, true> : quantize_kernel<false, false>);
  VB_CUDA(launch_serial(k, dim3(grid), dim3(kThreads), 0, stream, x, ldx, codes, scales, rows, padded, cols));
  return 0;
}

int mx4_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int dt, int64_t ldo, int rows, int cols, cudaStream_t stream) {
  if (int rc = check_rows("mx4_dequantize", rows, cols, codes, scales)) return rc;
  VB_CHECK(dt == VILA_DT_BF16 || dt == VILA_DT_F32, "mx4_dequantize: dtype code %d", dt);
  if (rows == 0) return 0;
  const int grid = grid_for(static_cast<long long>(rows) * ((cols + 255) / 256));
  const bool f32 = dt == VILA_DT_F32, vec = aligned(out, ldo, f32 ? 4 : 2);
  auto k = f32 ? (vec ? dequantize_kernel<true, true> : dequantize_kernel<true, false>)
               : (vec ? dequantize_kernel<false, true> : dequantize_kernel<false, false>);
  VB_CUDA(launch_serial(k, dim3(grid), dim3(kThreads), 0, stream, codes, scales, out, ldo, rows, cols));
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
