// 4-bit products for few rows an expert (mxfp4_rows.hip).
#pragma once

#include <hip/hip_runtime_api.h>

#include "expert_gemm.h"

namespace rr::kern {

// V columns of a row of 16-bit results. Rows of an odd width start on a word boundary and off it
// by turns; off it the first and the last column are stored by themselves, so that the others are
// whole words.
template <typename T, int V>
__device__ __forceinline__ void store_columns(T* p, const float (&v)[V], int left) {
  if constexpr (sizeof(T) == 2) {
    if (left >= V && (reinterpret_cast<uintptr_t>(p) & 2) != 0) {
      typedef T inner __attribute__((ext_vector_type(V - 2), aligned(4)));
      inner o;
#pragma unroll
      for (int i = 0; i < V - 2; ++i) o[i] = static_cast<T>(v[i + 1]);
      p[0] = static_cast<T>(v[0]);
      *reinterpret_cast<inner*>(p + 1) = o;
      p[V - 1] = static_cast<T>(v[V - 1]);
      return;
    }
  }
  Cols<T, V>::store(p, v, left);
}

// out = sums
template <typename T>
struct EpiMxStore {
  static constexpr bool kDual = false;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int, std::size_t row, int n, int left, const float (&v)[V]) {
    store_columns<T, V>(static_cast<T*>(p.out) + row * p.N + n, v, left);
  }
};

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
    store_columns<T, V>(static_cast<T*>(p.out_act) + row * p.N + n, a, left);
  }
};

// Whether the kernel for few rows takes a product (dual: with two right operands). prm as
// rr_mxfp4_gemm_kernel's.
bool mxfp4_rows_ok(const Product& prm, bool dual);
template <class Epi>
hipError_t mxfp4_rows(const Product& prm, hipStream_t stream);

}  // namespace rr::kern
