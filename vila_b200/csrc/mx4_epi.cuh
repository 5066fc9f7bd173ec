// What the tcgen05 kernels on microscaled rows do with their sums: bias, activation or gated unit, bf16.
#pragma once
#include <type_traits>
#include "../../include/vila_b200.h"
#include "common.cuh"
#include "glinear_epi.cuh"

namespace vb {

// An activation (VILA_ACT_*), or kMx4Gated + the flag of a gated unit, as a template parameter: the choice is made once a tile.
constexpr int kMx4Gated = 64;
template <int EPI> struct Mx4Epi { static constexpr int value = EPI; };
template <typename P, typename F>
__device__ __forceinline__ void mx4_with_epilogue(const P& p, F&& f) {      // P: parameters with flags and act
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

// The activations with __expf and __fdividef: their results are rounded to bf16 right after, and under the unpacking of weights
// or a few clocks of products per output the exact ones showed (2048 x 37888 x 3584 with a gated unit: 545 us).  kNear: small negative z count
// by themselves (layers on 8-bit rows, whose result may have a scale of its own).
template <int EPI, bool kNear = false>
__device__ __forceinline__ float mx4_act(float z, const vila_glinear_ext& x) {
  if (EPI == VILA_ACT_SILU) return silu_f(z);
  if (EPI == VILA_ACT_GELU_TANH) return gelu_tanh_f(z);
  if (EPI == VILA_ACT_XIELU) return kNear ? xielu_near_f(z, x.act_pos, x.act_neg) : xielu_fast_f(z, x.act_pos, x.act_neg);
  return activate(z, EPI, x);
}
template <int EPI>
__device__ __forceinline__ float mx4_glu(float g, float u, const vila_glinear_ext& x) {
  if (EPI == kMx4Gated + VILA_FLAG_GLU_CLAMP) return glu_clamp_fast_f(g, u, x.act_alpha, x.act_limit);
  return (EPI == kMx4Gated + VILA_FLAG_GEGLU ? gelu_tanh_f(g) : silu_f(g)) * u;
}

// 32 bytes (a whole sector of a row) at once
__device__ __forceinline__ void mx4_stg32(void* p, const uint32_t* h) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]), "r"(h[4]), "r"(h[5]),
               "r"(h[6]), "r"(h[7])
               : "memory");
}

// Lane = output row (token), 32 columns n .. n + 31 of the sums.  `wide`: rows of out start on 32-byte boundaries.
template <int EPI, typename P>
__device__ __forceinline__ void mx4_store_row(const P& p, const vila_glinear_ext& x, float (&z)[32], int m, int n, bool wide) {
  constexpr bool kGated = EPI >= kMx4Gated, kNear = !std::is_same<P, vila_mx4_linear_params>::value;
  constexpr int kWords = kGated ? 8 : 16;
  if (p.bias != nullptr) {
    const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(p.bias);
    // Not by __ldg: of bf16 it is assembly without a side effect, which the compiler may run where the condition does not hold.
#pragma unroll
    for (int i = 0; i < 32; ++i) z[i] += n + i < p.N ? __bfloat162float(bias[n + i]) : 0.f;
  }
  if (m >= p.M) return;
  uint32_t h[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if constexpr (kGated) h[i] = pack_bf16(mx4_glu<EPI>(z[4 * i], z[4 * i + 1], x), mx4_glu<EPI>(z[4 * i + 2], z[4 * i + 3], x));
    else h[i] = pack_bf16(mx4_act<EPI, kNear>(z[2 * i], x), mx4_act<EPI, kNear>(z[2 * i + 1], x));
  }
  const int o = kGated ? n / 2 : n, end = kGated ? p.N / 2 : p.N;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(m) * p.ldo + o;
#pragma unroll
  for (int g = 0; g < kWords / 8; ++g) {
    if (wide && o + 16 * g + 16 <= end) {
      mx4_stg32(out + 16 * g, h + 8 * g);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (o + 16 * g + i < end) reinterpret_cast<unsigned short*>(out)[16 * g + i] = static_cast<unsigned short>(h[8 * g + i / 2] >> (16 * (i & 1)));
    }
  }
}

// Lane = weight row n, one token m.  All lanes call it.
template <int EPI>
__device__ __forceinline__ void mx4_store_one(const vila_mx4_linear_params& p, const vila_glinear_ext& x, float v, int m, int n, float bias) {
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(m) * p.ldo;
  const float z = v + bias;
  if constexpr (EPI >= kMx4Gated) {
    const float other = __shfl_xor_sync(0xffffffffu, z, 1);
    if (n < p.N && (n & 1) == 0) out[n / 2] = __float2bfloat16_rn(mx4_glu<EPI>(z, other, x));
  } else {
    if (n < p.N) out[n] = __float2bfloat16_rn(mx4_act<EPI>(z, x));
  }
}

// Lane = weight row n, 16 tokens m .. m + 15 of the sums, those below `end`.  All lanes call it.
template <int EPI>
__device__ __forceinline__ void mx4_store_col(const vila_mx4_linear_params& p, const vila_glinear_ext& x, const float (&r)[16], int m, int end, int n, float bias) {
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  if constexpr (EPI >= kMx4Gated) {
    // the lanes of a pair hold gate and up: of two tokens each lane finishes one
    const bool odd = (n & 1) != 0;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float za = r[i] + bias, zb = r[i + 1] + bias, other = __shfl_xor_sync(0xffffffffu, odd ? za : zb, 1);
      const int row = m + i + (odd ? 1 : 0);
      if (n < p.N && row < end)
        out[static_cast<size_t>(row) * p.ldo + n / 2] = __float2bfloat16_rn(mx4_glu<EPI>(odd ? other : za, odd ? zb : other, x));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n < p.N && m + i < end) out[static_cast<size_t>(m + i) * p.ldo + n] = __float2bfloat16_rn(mx4_act<EPI>(r[i] + bias, x));
  }
}

}  // namespace vb
