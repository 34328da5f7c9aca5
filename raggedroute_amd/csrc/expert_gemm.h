// Products of the expert block on the matrix cores: what a kernel is given, and what
// becomes of the sums (epilogues). Shared by the tile kernels and the kernel for few rows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "block.h"
#include "block_device.h"

namespace rr::kern {

// One grouped product. Row products: C[r, n] = sum_k A[r, k] B_e[k, n] for the rows r of
// every expert e. Weight gradients: C_e[m, n] = sum over the expert's rows r of A[r, m]
// B[r, n]. Dual products have two right operands (b, b_up) of one shape; products of two
// parts add a second pair (a2, b_up) to the sum.
struct Product {
  const void* a;
  const void* a2;
  const void* b;
  const void* b_up;
  void* out;     // by epilogue
  void* out_up;
  void* out_act;
  const void* in;  // by epilogue
  const void* in_up;
  const int32_t* offsets;
  int experts, rows;
  int M;    // weight gradients: rows of the result
  int N;    // columns (of one right operand)
  int K;    // row products: length of one part's sum
  int lda;  // elements between rows of A
  int ldb;  // elements between rows of B as stored
  int activation;
  bool out_f32;
};

// Four elements or more of a row, FP32 in use.
template <typename T, int V>
struct Cols {
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  static __device__ __forceinline__ void store(T* p, const float (&v)[V], int left) {
    if (left >= V) {
      vec o;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = static_cast<T>(v[i]);
      *reinterpret_cast<vec*>(p) = o;
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i < left) p[i] = static_cast<T>(v[i]);
    }
  }
  static __device__ __forceinline__ void load(const T* p, float (&v)[V], int left) {
    if (left >= V) {
      const vec o = *reinterpret_cast<const vec*>(p);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = static_cast<float>(o[i]);
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < left ? static_cast<float>(p[i]) : 0.0F;
  }
};

// Epilogues: emit(product, expert, row, column, columns left in the row, sums of V
// columns of the one or two right operands). `row` counts the rows of the result.

// out = sums, in T or FP32
template <typename T>
struct EpiStore {
  static constexpr bool kDual = false;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int, std::size_t row, int n, int left, const float (&v)[V]) {
    const std::size_t at = row * p.N + n;
    if (p.out_f32) {
      Cols<float, V>::store(static_cast<float*>(p.out) + at, v, left);
    } else {
      Cols<T, V>::store(static_cast<T*>(p.out) + at, v, left);
    }
  }
};

// out = sums of the first right operand, out_up = of the second
template <typename T>
struct EpiPair {
  static constexpr bool kDual = true;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int, std::size_t row, int n, int left, const float (&g)[V],
                                              const float (&u)[V]) {
    const std::size_t at = row * p.N + n;
    Cols<T, V>::store(static_cast<T*>(p.out) + at, g, left);
    Cols<T, V>::store(static_cast<T*>(p.out_up) + at, u, left);
  }
};

// out_act = act(g) u; out, out_up = g, u where they are kept
template <typename T>
struct EpiGate {
  static constexpr bool kDual = true;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int, std::size_t row, int n, int left, const float (&g)[V],
                                              const float (&u)[V]) {
    const std::size_t at = row * p.N + n;
    if (p.out != nullptr) {
      Cols<T, V>::store(static_cast<T*>(p.out) + at, g, left);
      Cols<T, V>::store(static_cast<T*>(p.out_up) + at, u, left);
    }
    float a[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = rr::dev::activation(p.activation, g[i]) * u[i];
    Cols<T, V>::store(static_cast<T*>(p.out_act) + at, a, left);
  }
};

// sums = da: out = d gate, out_up = d up, from gate (in) and up (in_up). Both are rounded to T
// once, as operands of the matrix instructions; with g and u kept in T the gradients are
// off by 1.8 times the rounding of their own result (FP32 copies of g and u, 1.4 times,
// would double what a step keeps of every row).
template <typename T>
struct EpiDGate {
  static constexpr bool kDual = false;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int, std::size_t row, int n, int left, const float (&da)[V]) {
    const std::size_t at = row * p.N + n;
    float g[V], u[V];
    Cols<T, V>::load(static_cast<const T*>(p.in) + at, g, left);
    Cols<T, V>::load(static_cast<const T*>(p.in_up) + at, u, left);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float act, grad;
      rr::dev::activation_grad(p.activation, g[i], &act, &grad);
      g[i] = da[i] * u[i] * grad;
      u[i] = da[i] * act;
    }
    Cols<T, V>::store(static_cast<T*>(p.out) + at, g, left);
    Cols<T, V>::store(static_cast<T*>(p.out_up) + at, u, left);
  }
};

// int32 sums (converted) times the row's and the channels' scales. in: channel scales,
// in_up: those of the second operand, a2: row scales. LONGEST: the one sum past int32 is mended
// (not in the direct tile kernels, whose registers are full: the gated one would spill).
template <typename T, bool LONGEST>
struct EpiInt8 {
  static constexpr bool kDual = false;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int e, std::size_t row, int n, int left, float (&v)[V]) {
    if constexpr (LONGEST) rr::dev::mend_int8_sums(v, p.K);
    const float rs = static_cast<const float*>(p.a2)[row];
    float s[V], y[V];
    Cols<float, V>::load(static_cast<const float*>(p.in) + static_cast<std::size_t>(e) * p.N + n, s, left);
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = v[i] * rs * s[i];
    Cols<T, V>::store(static_cast<T*>(p.out) + row * p.N + n, y, left);
  }
};

template <typename T, bool LONGEST>
struct EpiInt8Gate {
  static constexpr bool kDual = true;
  template <int V>
  static __device__ __forceinline__ void emit(const Product& p, int e, std::size_t row, int n, int left, float (&g)[V],
                                              float (&u)[V]) {
    if constexpr (LONGEST) {
      rr::dev::mend_int8_sums(g, p.K);
      rr::dev::mend_int8_sums(u, p.K);
    }
    const float rs = static_cast<const float*>(p.a2)[row];
    const std::size_t channel = static_cast<std::size_t>(e) * p.N + n;
    float sg[V], su[V], y[V];
    Cols<float, V>::load(static_cast<const float*>(p.in) + channel, sg, left);
    Cols<float, V>::load(static_cast<const float*>(p.in_up) + channel, su, left);
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = rr::dev::activation(p.activation, g[i] * rs * sg[i]) * (u[i] * rs * su[i]);
    Cols<T, V>::store(static_cast<T*>(p.out) + row * p.N + n, y, left);
  }
};

// ---- few rows an expert (expert_rows.hip) ----
// Whether the kernel for few rows takes a row product of this many rows.
bool expert_rows_ok(int rows, int experts, bool int8);
// Workgroups that share an expert's sum of `length` (1: no parts are needed).
int expert_rows_splits(int rows, int experts, int columns, int length);
// parts: FP32 [1, dual products 2][splits][rows][N] where splits > 1 (16-bit products only).
template <typename T, class Epi>
hipError_t expert_rows(const Product& prm, float* parts, int splits, hipStream_t stream);

}  // namespace rr::kern
