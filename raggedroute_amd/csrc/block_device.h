// Element types, activations and segment lookups shared by the expert block's kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "raggedroute_capi.h"

namespace rr::dev {

typedef __bf16 bf16;
typedef _Float16 f16;

// 1 / (1 + e^-v): v_exp_f32 takes powers of two. e^-v past FP32 gives 0, NaN stays.
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.0F + __builtin_amdgcn_exp2f(-1.44269504088896341F * v));
}

// act(g) = g sigmoid(t(g)): t(g) = g for SiLU, and for the tanh form of GELU
// (1 + tanh z) / 2 = sigmoid(2 z) with z = sqrt(2 / pi) (g + 0.044715 g^3).
constexpr float kGelu = 1.59576912160573071F;  // 2 sqrt(2 / pi)
constexpr float kGeluCube = 0.044715F;

__device__ __forceinline__ float activation(int kind, float g) {
  const float t = kind == RR_ACT_SILU ? g : kGelu * (g + kGeluCube * g * g * g);
  return g * sigmoid(t);
}

// act(g) and act'(g) = s + g t'(g) s (1 - s), s = sigmoid(t(g)). Past the cuts of g in the
// second term one of its other factors is 0, and no square may overflow against it: 1 - s
// from 18 on, s below -88 (for SiLU, whose slope there is the second term).
__device__ __forceinline__ void activation_grad(int kind, float g, float* act, float* grad) {
  const float t = kind == RR_ACT_SILU ? g : kGelu * (g + kGeluCube * g * g * g);
  const float s = sigmoid(t);
  const float b = g > 40.0F ? 40.0F : g < -104.0F ? -104.0F : g;
  const float slope = kind == RR_ACT_SILU ? 1.0F : kGelu * (1.0F + 3.0F * kGeluCube * b * b);
  *act = g * s;
  *grad = s + b * slope * (s * (1.0F - s));
}

// Int32 sums of K int8 products, as FP32. Of at most 2^17 products the least is 2^24 above
// -2^31, and one sum passes 31 bits: 2^17 times (-128)(-128), whose bits are those of -2^31.
template <int V>
__device__ __forceinline__ void mend_int8_sums(float (&v)[V], int K) {
  if (K != 1 << 17) return;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = v[i] == -0x1p31F ? 0x1p31F : v[i];
}

// offsets[e] cut to [0, rows]. Segments are bounded by the largest of these up to theirs: an
// offset that falls leaves its expert empty, and no row belongs to two experts.
__device__ __forceinline__ int offset_at(const int32_t* offsets, int e, int rows) {
  const int o = offsets[e];
  return o < 0 ? 0 : o > rows ? rows : o;
}

}  // namespace rr::dev
