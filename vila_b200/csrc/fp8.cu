// Rows and weights to 8-bit numbers with a scale per block of 128 and back, and the norm before a layer with its result in that form (fp8.cuh).
//
// All three are bound by memory.  A lane takes 16 neighbouring columns, 32 or 64 bytes in and 16 bytes of codes out, so that 8 lanes hold a
// block of a row: its largest magnitude takes three shuffles, and the numbers wait in registers for it.  Data are read once.
//
// Rows of 16470 x 3584 bf16: 31.4 us in a captured graph, 27.3 at the rate of a copy; a weight of 37888 x 3584: 62.3 us, 62.3 at that rate.
// The norm of 16470 x 3584 with a residual 67 us, 6.1 TB/s; of 2048 rows 12.1 us, 7.9 at a copy's rate: 2.3 rounds of CTAs, which each load x and the
// residual, meet, and then load the norm's weights.  A single row is 1.3 us, and the call 13: the host's.
#include "../../include/vila_b200.h"
#include "fp8.cuh"
#include "dtype_any.cuh"
#include "kernels.h"

namespace vb {
namespace {

constexpr int kThreads = 256;

enum { kApart = 0, kBy16 = 16, kBy32 = 32 };      // how rows lie: anywhere, on boundaries of 16 or 32 bytes

__device__ __forceinline__ void ldg32(const void* p, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void stg32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7]) : "memory");
}
// 16 columns as they lie: `n` of them are there (others read as 0)
template <bool kF32> struct Chunk {
  static constexpr int kWords = kF32 ? 16 : 8;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* row, int c0, int n, int how) {
    const uint8_t* src = static_cast<const uint8_t*>(row) + static_cast<int64_t>(c0) * (kF32 ? 4 : 2);
    if (n >= kFp8Chunk && how == kBy32) {
#pragma unroll
      for (int i = 0; i < kWords; i += 8) ldg32(src + 4 * i, w + i);
    } else if (n >= kFp8Chunk && how == kBy16) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 q = ldg_v4(src + 4 * i);
        w[i] = q.x; w[i + 1] = q.y; w[i + 2] = q.z; w[i + 3] = q.w;
      }
    } else {
      uint32_t e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = i < n ? ld_raw(src, kF32 ? 1 : 0, i) : 0u;
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = kF32 ? e[i] : e[2 * i % 16] | e[(2 * i + 1) % 16] << 16;
    }
  }
  __device__ __forceinline__ void store(void* row, int c0, int n, int how) const {
    uint8_t* dst = static_cast<uint8_t*>(row) + static_cast<int64_t>(c0) * (kF32 ? 4 : 2);
    if (n >= kFp8Chunk && how == kBy32) {
#pragma unroll
      for (int i = 0; i < kWords; i += 8) stg32(dst + 4 * i, w + i);
    } else if (n >= kFp8Chunk && how == kBy16) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) stg_v4(dst + 4 * i, make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]));
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < n) {
          if (kF32) reinterpret_cast<uint32_t*>(dst)[i] = w[i % kWords];
          else reinterpret_cast<uint16_t*>(dst)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
        }
    }
  }
  __device__ __forceinline__ void numbers(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = kF32 ? __uint_as_float(w[i % kWords]) : (i & 1 ? bf_hi(w[i / 2]) : bf_lo(w[i / 2]));
  }
  __device__ __forceinline__ void set(const float (&v)[16]) {      // rounded to the type
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = kF32 ? __float_as_uint(v[i]) : pack_bf16(v[2 * i % 16], v[(2 * i + 1) % 16]);
  }
  __device__ __forceinline__ uint32_t top() const {      // the largest magnitude's bits, as fp32
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) t = kF32 ? max(t, w[i] & 0x7fffffffu) : __vmaxu2(t, w[i] & 0x7fff7fffu);
    return kF32 ? t : max(t << 16, t & 0xffff0000u);
  }
};
__device__ __forceinline__ uint32_t top_of(const float (&v)[16]) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) t = max(t, __float_as_uint(v[i]) & 0x7fffffffu);
  return t;
}

// ---- rows ----
// Items are chunks, whole blocks of them; r0: the first row of this launch.  items is a multiple of 8, and so is where a warp starts:
// the lanes of a block are there together, and all lanes of a warp take part in the shuffles.
template <bool kF32>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const void* x, int64_t ldx, int how, uint8_t* codes, int64_t ldc, float* scales, int64_t lds, int r0, int cols, uint32_t per,
                     uint32_t items) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t step = gridDim.x * kThreads;
  for (uint32_t it0 = blockIdx.x * kThreads + threadIdx.x - lane; it0 < items; it0 += step) {
    const uint32_t it = it0 + lane;
    const bool there = it < items;
    const uint32_t rr = there ? it / per : 0u;
    const int r = r0 + static_cast<int>(rr), c0 = there ? static_cast<int>(it - rr * per) * kFp8Chunk : 0, n = there ? cols - c0 : 0;
    Chunk<kF32> q;
    q.load(static_cast<const uint8_t*>(x) + static_cast<int64_t>(r) * ldx * (kF32 ? 4 : 2), c0, n, how);
    const Fp8Scale s = fp8_scale(fp8_top8(q.top()));
    if (n > 0) {
      float v[16];
      q.numbers(v);
      stg_v4(codes + static_cast<int64_t>(r) * ldc + c0, fp8_encode16(v, s));      // a row's codes have room for whole chunks
      if ((lane & 7) == 0) scales[static_cast<int64_t>(c0 / kFp8Block) * lds + r] = s.scale;
    }
    __syncwarp();
  }
}

// ---- weights: a CTA takes a block of 128 x 128, a thread a chunk of every 32nd row of it ----
template <bool kF32>
__global__ void __launch_bounds__(kThreads)
quantize_weight_kernel(const void* x, int64_t ldx, int how, uint8_t* codes, int64_t ldc, float* scales, int64_t lds, int rows, int cols) {
  __shared__ uint32_t tops[kThreads / 32];
  const int lane = threadIdx.x & 31, kb = blockIdx.x, rb = blockIdx.y;
  const int c0 = kb * kFp8Block + (threadIdx.x & 7) * kFp8Chunk, n = cols - c0;
  Chunk<kF32> q[4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = rb * kFp8Block + i * 32 + (threadIdx.x >> 3);
    q[i].load(static_cast<const uint8_t*>(x) + static_cast<int64_t>(r) * ldx * (kF32 ? 4 : 2), c0, r < rows ? n : 0, how);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, q[i].top());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) top = max(top, tops[i]);
  const Fp8Scale s = fp8_scale(top);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = rb * kFp8Block + i * 32 + (threadIdx.x >> 3);
    float v[16];
    q[i].numbers(v);
    if (r < rows && n > 0) stg_v4(codes + static_cast<int64_t>(r) * ldc + c0, fp8_encode16(v, s));
  }
  if (threadIdx.x == 0) scales[rb * lds + kb] = s.scale;
}

// ---- back ----
template <bool kF32>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t* codes, int64_t ldc, const float* scales, int64_t lds, void* out, int64_t ldo, int how, int r0, int cols,
                  uint32_t per, uint32_t items, int block_rows) {
  const uint32_t step = gridDim.x * kThreads;
  for (uint32_t it = blockIdx.x * kThreads + threadIdx.x; it < items; it += step) {
    const uint32_t rr = it / per;
    const int r = r0 + static_cast<int>(rr), c0 = static_cast<int>(it - rr * per) * kFp8Chunk, kb = c0 / kFp8Block;
    const uint4 c4 = ldg_v4(codes + static_cast<int64_t>(r) * ldc + c0);
    const float s = block_rows == 1 ? scales[kb * lds + r] : scales[r / kFp8Block * lds + kb];
    const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = fp8_decode2(c[i / 2] >> (16 * (i & 1)) & 0xffffu);
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
    Chunk<kF32> q;
    q.set(v);
    q.store(static_cast<uint8_t*>(out) + static_cast<int64_t>(r) * ldo * (kF32 ? 4 : 2), c0, cols - c0, how);
  }
}

// ---- the norm: a CTA takes a row, a thread kIter chunks of it, T threads apart ----
struct Norm {
  const void *x, *residual, *w;
  void* sum;
  int64_t ldx, ldr, ld_sum, ldc, lds;
  uint8_t* codes;
  float* scales;
  float eps;
  int cols, x_how, r_how, sum_how, w_how, r_f32, w_f32;
};
template <bool kF32, int kIter>
__global__ void __launch_bounds__(512) norm_kernel(const Norm p) {
  __shared__ float red[32];
  griddep_launch_dependents();
  griddep_wait();
  const int row = blockIdx.x, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const uint8_t* x = static_cast<const uint8_t*>(p.x) + static_cast<int64_t>(row) * p.ldx * (kF32 ? 4 : 2);
  Chunk<kF32> q[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int c0 = (threadIdx.x + i * blockDim.x) * kFp8Chunk;
    q[i].load(x, c0, p.cols - c0, p.x_how);
  }
  if (p.residual != nullptr) {
    const uint8_t* res = static_cast<const uint8_t*>(p.residual) + static_cast<int64_t>(row) * p.ldr * (p.r_f32 ? 4 : 2);
    uint8_t* sum = static_cast<uint8_t*>(p.sum) + static_cast<int64_t>(row) * p.ld_sum * (kF32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int c0 = (threadIdx.x + i * blockDim.x) * kFp8Chunk, n = p.cols - c0;
      float v[16], a[16];
      if (p.r_f32) {
        Chunk<true> c;
        c.load(res, c0, n, p.r_how);
        c.numbers(a);
      } else {
        Chunk<false> c;
        c.load(res, c0, n, p.r_how);
        c.numbers(a);
      }
      q[i].numbers(v);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] += a[j];
      q[i].set(v);
      q[i].store(sum, c0, n, p.sum_how);
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    float v[16];
    q[i].numbers(v);
#pragma unroll
    for (int j = 0; j < 16; ++j) s = fmaf(v[j], v[j], s);
  }
  s = warp_sum(s);
  if (lane == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = warp_sum(lane < warps ? red[lane] : 0.f);
  const float rstd = 1.f / sqrtf(s / p.cols + p.eps);
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int c0 = (threadIdx.x + i * blockDim.x) * kFp8Chunk, n = p.cols - c0;
    float v[16];
    q[i].numbers(v);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] *= rstd;
    if (p.w != nullptr) {
      float a[16];
      if (p.w_f32) {
        Chunk<true> c;
        c.load(p.w, c0, n, p.w_how);
        c.numbers(a);
      } else {
        Chunk<false> c;
        c.load(p.w, c0, n, p.w_how);
        c.numbers(a);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] *= a[j];
    }
    // columns past the last one are zeros, but where rstd is infinite or a NaN
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = j < n ? v[j] : 0.f;
    const Fp8Scale e = fp8_scale(fp8_top8(top_of(v)));
    if (n > 0) {
      stg_v4(p.codes + static_cast<int64_t>(row) * p.ldc + c0, fp8_encode16(v, e));
      if ((lane & 7) == 0) p.scales[static_cast<int64_t>(c0 / kFp8Block) * p.lds + row] = e.scale;
    }
  }
}

int grid_for(long long threads) {
  const long long blocks = (threads + kThreads - 1) / kThreads, most = 16ll * num_sms();
  return static_cast<int>(blocks < most ? blocks : most);
}
int how(const void* p, int64_t ld, int esize) {
  const uint64_t a = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(ld) * esize;
  return a % 32 == 0 ? kBy32 : (a % 16 == 0 ? kBy16 : kApart);
}
bool known(int dt) { return dt == VILA_DT_BF16 || dt == VILA_DT_F32; }
int size_of(int dt) { return dt == VILA_DT_F32 ? 4 : 2; }
// f(first row, items) for as many rows as items (`per` a row) are counted in 32 bits, a grid's step to spare
template <typename F>
int by_rows(int rows, int64_t per, F&& f) {
  const int64_t most = (0xffffffffll - 2ll * 16 * num_sms() * kThreads) / per;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    if (int rc = f(static_cast<int>(r), static_cast<uint32_t>(n * per))) return rc;
  }
  return 0;
}
int check_form(const char* what, const void* codes, int64_t ldc, const float* scales, int64_t lds, int rows, int cols, int block_rows) {
  VB_CHECK(rows >= 0 && cols > 0 && rows <= (1 << 30) && cols <= (1 << 25), "%s: rows=%d cols=%d", what, rows, cols);
  VB_CHECK(block_rows == 1 || block_rows == kFp8Block, "%s: block_rows=%d (1 or 128)", what, block_rows);
  if (rows == 0) return 0;
  VB_CHECK(codes != nullptr && scales != nullptr, "%s: a null pointer", what);
  VB_CHECK(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && ldc % 16 == 0 && ldc >= cols, "%s: rows of codes start on 16-byte boundaries, ldc=%lld cols=%d",
           what, static_cast<long long>(ldc), cols);
  if (block_rows == 1)
    VB_CHECK(reinterpret_cast<uintptr_t>(scales) % 16 == 0 && lds % 4 == 0 && lds >= rows, "%s: scales start on 16-byte boundaries, lds=%lld rows=%d", what,
             static_cast<long long>(lds), rows);
  else
    VB_CHECK(reinterpret_cast<uintptr_t>(scales) % 4 == 0 && lds >= fp8_blocks(cols), "%s: scales: lds=%lld cols=%d", what, static_cast<long long>(lds), cols);
  return 0;
}
int check_numbers(const char* what, const void* x, int dt) {
  VB_CHECK(known(dt), "%s: dtype code %d", what, dt);
  VB_CHECK(x != nullptr && reinterpret_cast<uintptr_t>(x) % size_of(dt) == 0, "%s: a null pointer, or one off its elements' boundaries", what);
  return 0;
}

}  // namespace

int fp8_quantize(const void* x, int dt, int64_t ldx, void* codes, int64_t ldc, float* scales, int64_t lds, int rows, int cols, int block_rows,
                 cudaStream_t stream) {
  if (int rc = check_form("fp8_quantize", codes, ldc, scales, lds, rows, cols, block_rows)) return rc;
  if (rows == 0) return 0;
  if (int rc = check_numbers("fp8_quantize", x, dt)) return rc;
  const bool f32 = dt == VILA_DT_F32;
  const int h = how(x, ldx, size_of(dt));
  uint8_t* c = static_cast<uint8_t*>(codes);
  if (block_rows == 1) {
    const uint32_t per = fp8_blocks(cols) * (kFp8Block / kFp8Chunk);
    return by_rows(rows, per, [&](int r0, uint32_t items) {
      VB_CUDA(launch_pdl(f32 ? quantize_rows_kernel<true> : quantize_rows_kernel<false>, dim3(grid_for(items)), dim3(kThreads), 0, stream, x, ldx, h, c,
                            ldc, scales, lds, r0, cols, per, items));
      return 0;
    });
  }
  constexpr int kMost = 65535;      // of a grid's second dimension
  for (int b = 0; b < fp8_blocks(rows); b += kMost) {
    const int n = fp8_blocks(rows) - b < kMost ? fp8_blocks(rows) - b : kMost;
    const int64_t r = static_cast<int64_t>(b) * kFp8Block;
    VB_CUDA(launch_serial(f32 ? quantize_weight_kernel<true> : quantize_weight_kernel<false>, dim3(fp8_blocks(cols), n), dim3(kThreads), 0, stream,
                          static_cast<const void*>(static_cast<const uint8_t*>(x) + r * ldx * size_of(dt)), ldx, h, c + r * ldc, ldc, scales + b * lds, lds,
                          static_cast<int>(rows - r), cols));
  }
  return 0;
}

int fp8_dequantize(const void* codes, int64_t ldc, const float* scales, int64_t lds, void* out, int dt, int64_t ldo, int rows, int cols,
                   int block_rows, cudaStream_t stream) {
  if (int rc = check_form("fp8_dequantize", codes, ldc, scales, lds, rows, cols, block_rows)) return rc;
  if (rows == 0) return 0;
  if (int rc = check_numbers("fp8_dequantize", out, dt)) return rc;
  VB_CHECK(rows == 1 || ldo >= cols, "fp8_dequantize: ldo=%lld cols=%d", static_cast<long long>(ldo), cols);
  const uint32_t per = (cols + kFp8Chunk - 1) / kFp8Chunk;
  const int h = how(out, ldo, size_of(dt));
  return by_rows(rows, per, [&](int r0, uint32_t items) {
    VB_CUDA(launch_serial(dt == VILA_DT_F32 ? dequantize_kernel<true> : dequantize_kernel<false>, dim3(grid_for(items)), dim3(kThreads), 0, stream,
                          static_cast<const uint8_t*>(codes), ldc, scales, lds, out, ldo, h, r0, cols, per, items, block_rows));
    return 0;
  });
}

int fp8_rmsnorm(const vila_fp8_rmsnorm_params& a, cudaStream_t stream) {
  if (int rc = check_form("fp8_rmsnorm", a.codes, a.ldc, a.scales, a.lds, a.rows, a.cols, 1)) return rc;
  VB_CHECK(a.cols <= 32768, "fp8_rmsnorm: cols=%d (at most 32768)", a.cols);
  VB_CHECK(a.eps >= 0.f, "fp8_rmsnorm: eps=%g", a.eps);
  if (a.rows == 0) return 0;
  if (int rc = check_numbers("fp8_rmsnorm", a.x, a.x_dtype)) return rc;
  if (a.w != nullptr)
    if (int rc = check_numbers("fp8_rmsnorm", a.w, a.w_dtype)) return rc;
  if (a.residual != nullptr) {
    if (int rc = check_numbers("fp8_rmsnorm", a.residual, a.residual_dtype)) return rc;
    if (int rc = check_numbers("fp8_rmsnorm", a.sum, a.x_dtype)) return rc;
    VB_CHECK(a.rows == 1 || a.ld_sum >= a.cols, "fp8_rmsnorm: ld_sum=%lld cols=%d", static_cast<long long>(a.ld_sum), a.cols);
    VB_CHECK(a.sum != a.x || a.rows == 1 || a.ld_sum == a.ldx, "fp8_rmsnorm: the sum in x's place has x's stride");
  }
  Norm p = {};
  p.x = a.x;
  p.ldx = a.ldx;
  p.x_how = how(a.x, a.ldx, size_of(a.x_dtype));
  p.residual = a.residual;
  if (a.residual != nullptr) {
    p.sum = a.sum;
    p.ldr = a.ldr;
    p.ld_sum = a.ld_sum;
    p.r_f32 = a.residual_dtype == VILA_DT_F32;
    p.r_how = how(a.residual, a.ldr, size_of(a.residual_dtype));
    p.sum_how = how(a.sum, a.ld_sum, size_of(a.x_dtype));
  }
  p.w = a.w;
  p.w_f32 = a.w != nullptr && a.w_dtype == VILA_DT_F32;
  p.w_how = how(a.w, 0, 1);
  p.codes = static_cast<uint8_t*>(a.codes);
  p.ldc = a.ldc;
  p.scales = a.scales;
  p.lds = a.lds;
  p.eps = a.eps;
  p.cols = a.cols;
  // as many threads as the row has chunks, one each up to 512 threads, then two, then four
  const int chunks = fp8_blocks(a.cols) * (kFp8Block / kFp8Chunk), iter = chunks <= 512 ? 1 : (chunks <= 1024 ? 2 : 4);
  const int threads = ((chunks + iter - 1) / iter + 31) / 32 * 32;
  const bool f32 = a.x_dtype == VILA_DT_F32;
  auto k = iter == 1 ? (f32 ? norm_kernel<true, 1> : norm_kernel<false, 1>)
                     : (iter == 2 ? (f32 ? norm_kernel<true, 2> : norm_kernel<false, 2>) : (f32 ? norm_kernel<true, 4> : norm_kernel<false, 4>));
  VB_CUDA(launch_pdl(k, dim3(a.rows), dim3(threads), 0, stream, p));
  return 0;
}

}  // namespace vb
