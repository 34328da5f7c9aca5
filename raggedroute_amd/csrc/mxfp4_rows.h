// 4-bit products for few rows an expert (mxfp4_rows.hip).
#pragma once

#include <hip/hip_runtime_api.h>

#include "expert_gemm.h"

namespace rr::kern {

// out_act = act(g) u. A tile's 64 results a lane cost as much as a few slices of products, so
// that the kind is chosen once for all columns and the exponent is one polynomial: act(g) = g
// / (1 + 2^-z), z = log2(e) g for SiLU and log2(e) g (kGelu + kGelu kGeluCube g^2) for the tanh form
// of GELU (16384 rows of 64 experts, K = 1024, N = 512: 29.0 us with EpiGate, 26.7).
template <typename T>
struct EpiMxGate {
  static constexpr bool kDual = true;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int, std::size_t row, int n, int left, const float (&g)[V],
                                              const float (&u)[V]) {
    constexpr float kLog2e = 1.44269504088896341F;
    float a[V];
    auto apply = [&](auto exponent) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a[i] = g[i] * __builtin_amdgcn_rcpf(1.0F + __builtin_amdgcn_exp2f(exponent(g[i]))) * u[i];
      }
    };
    if (p.activation == RR_ACT_SILU) {
      apply([](float v) { return -kLog2e * v; });
    } else {
      apply([](float v) { return v * __builtin_fmaf(-kLog2e * rr::dev::kGelu * rr::dev::kGeluCube, v * v, -kLog2e * rr::dev::kGelu); });
    }
    Cols<T, V>::store(static_cast<T*>(p.out_act) + row * p.N + n, a, left);
  }
};

// Whether the kernel for few rows takes a product of this many rows.
bool mxfp4_rows_ok(int rows, int experts);
// prm as rr_mxfp4_gemm_kernel's.
template <class Epi>
hipError_t mxfp4_rows(const Product& prm, hipStream_t stream);

}  // namespace rr::kern
