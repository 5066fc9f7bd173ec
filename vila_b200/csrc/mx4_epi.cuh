// What the tcgen05 kernels on microscaled rows do with their sums: bias, activation or gated unit, bf16.
#pragma once
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "glinear_epi.cuh"

namespace vb {

// An activation (VILA_ACT_*), or kMx4Gated + the flag of a gated unit, as a template parameter: the choice is made once a tile.
constexpr int kMx4Gated = 64;
template <int EPI> struct Mx4Epi { static constexpr int value = EPI; };
template <typename F>
__device__ __forceinline__ void mx4_with_epilogue(const vila_mx4_linear_params& p, F&& f) {
  if (p.flags & VILA_FLAG_GLU_CLAMP) return f(Mx4Epi<kMx4Gated + VILA_FLAG_GLU_CLAMP>());
  if (p.flags & VILA_FLAG_GEGLU) return f(Mx4Epi<kMx4Gated + VILA_FLAG_GEGLU>());
  if (p.flags & VILA_FLAG_SWIGLU) return f(Mx4Epi<kMx4Gated + VILA_FLAG_SWIGLU>());
  switch (p.act) {
    case VILA_ACT_SILU: return f(Mx4Epi<VILA_ACT_SILU>());
    case VILA_ACT_RELU2: return f(Mx4Epi<VILA_ACT_RELU2>());
    case VILA_ACT_GELU_TANH: return f(Mx4Epi<VILA_ACT_GELU_TANH>());
    case VILA_ACT_GELU_ERF: return f(Mx4Epi<VILA_ACT_GELU_ERF>());
    case VILA_ACT_XIELU: return f(Mx4Epi<VILA_ACT_XIELU>());
    default: return f(Mx4Epi<VILA_ACT_NONE>());
  }
}

// Lane = output row (token), 16 columns n .. n + 15 of the sums.  `vec`: rows of out start on 16-byte boundaries.
template <int EPI>
__device__ __forceinline__ void mx4_store_row(const vila_mx4_linear_params& p, const vila_glinear_ext& x, const float (&r)[16], int m, int n, bool vec) {
  const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
  float z[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = r[i] + (bias != nullptr && n + i < p.N ? __bfloat162float(__ldg(bias + n + i)) : 0.f);
  if (m >= p.M) return;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(m) * p.ldo;
  if constexpr (EPI >= kMx4Gated) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = pack_bf16(glu(z[4 * i], z[4 * i + 1], EPI - kMx4Gated, x), glu(z[4 * i + 2], z[4 * i + 3], EPI - kMx4Gated, x));
    if (vec && n + 16 <= p.N) {
      stg_v4(out + n / 2, make_uint4(h[0], h[1], h[2], h[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + 2 * i < p.N) reinterpret_cast<unsigned short*>(out)[n / 2 + i] = static_cast<unsigned short>(h[i / 2] >> (16 * (i & 1)));
    }
  } else {
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = pack_bf16(activate(z[2 * i], EPI, x), activate(z[2 * i + 1], EPI, x));
    if (vec && n + 16 <= p.N) {
      stg_v4(out + n, make_uint4(h[0], h[1], h[2], h[3]));
      stg_v4(out + n + 8, make_uint4(h[4], h[5], h[6], h[7]));
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (n + i < p.N) reinterpret_cast<unsigned short*>(out)[n + i] = static_cast<unsigned short>(h[i / 2] >> (16 * (i & 1)));
    }
  }
}

// Lane = weight row n, 16 tokens m .. m + 15 of the sums.  All lanes call it.
template <int EPI>
__device__ __forceinline__ void mx4_store_col(const vila_mx4_linear_params& p, const vila_glinear_ext& x, const float (&r)[16], int m, int n, float bias) {
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  if constexpr (EPI >= kMx4Gated) {
    // the lanes of a pair hold gate and up: of two tokens each lane finishes one
    const bool odd = (n & 1) != 0;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float za = r[i] + bias, zb = r[i + 1] + bias, other = __shfl_xor_sync(0xffffffffu, odd ? za : zb, 1);
      const int row = m + i + (odd ? 1 : 0);
      if (n < p.N && row < p.M)
        out[static_cast<size_t>(row) * p.ldo + n / 2] = __float2bfloat16_rn(glu(odd ? other : za, odd ? zb : other, EPI - kMx4Gated, x));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n < p.N && m + i < p.M) out[static_cast<size_t>(m + i) * p.ldo + n] = __float2bfloat16_rn(activate(r[i] + bias, EPI, x));
  }
}

}  // namespace vb
