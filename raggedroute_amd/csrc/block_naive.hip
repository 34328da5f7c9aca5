// Naive forms of the expert block's products: one thread per output, FP32 sums in
// ascending order. The semantic floor behind RR_FAMILY_NAIVE.
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "block.h"
#include "block_device.h"
#include "mxfp4.h"

namespace rr::kern {
namespace {

using rr::dev::activation;
using rr::dev::activation_grad;
using rr::dev::offset_at;

constexpr unsigned kThreads = 256;
constexpr std::size_t kMaxBlocks = 65535;

dim3 grid_for(std::size_t outputs) {
  const std::size_t blocks = (outputs + kThreads - 1) / kThreads;
  return dim3(static_cast<unsigned>(blocks < 1 ? 1 : blocks < kMaxBlocks ? blocks : kMaxBlocks));
}

// Calls f(i) for every output i < count of this thread.
template <typename F>
__device__ __forceinline__ void for_outputs(std::size_t count, F f) {
  const std::size_t stride = static_cast<std::size_t>(kThreads) * gridDim.x;
  for (std::size_t i = static_cast<std::size_t>(blockIdx.x) * kThreads + threadIdx.x; i < count; i += stride) f(i);
}

// First row of expert e: the largest offset up to its own.
__device__ int first_row(const int32_t* offsets, int e, int rows) {
  int most = 0;
  for (int i = 0; i <= e; ++i) most = max(most, offset_at(offsets, i, rows));
  return most;
}

// The expert whose segment holds `row`, or -1.
__device__ int expert_of(const int32_t* offsets, int experts, int rows, int row) {
  if (row < offset_at(offsets, 0, rows)) return -1;
  for (int e = 0; e < experts; ++e) {
    if (row < offset_at(offsets, e + 1, rows)) return e;
  }
  return -1;
}

template <typename T>
__global__ void rr_ffn_gate_up_naive_kernel(FfnParams p) {
  const auto* x = static_cast<const T*>(p.x);
  const auto* wg = static_cast<const T*>(p.w_gate);
  const auto* wu = static_cast<const T*>(p.w_up);
  const std::size_t K = p.hidden, F = p.inner;
  for_outputs(p.rows * F, [&](std::size_t i) {
    const std::size_t row = i / F, f = i % F;
    const int e = expert_of(p.offsets, p.experts, p.rows, static_cast<int>(row));
    if (e < 0) return;
    float g = 0.0F, u = 0.0F;
    for (std::size_t k = 0; k < K; ++k) {
      const float v = static_cast<float>(x[row * K + k]);
      g = __builtin_fmaf(v, static_cast<float>(wg[(e * K + k) * F + f]), g);
      u = __builtin_fmaf(v, static_cast<float>(wu[(e * K + k) * F + f]), u);
    }
    if (p.gate != nullptr) {
      static_cast<T*>(p.gate)[i] = static_cast<T>(g);
      static_cast<T*>(p.up)[i] = static_cast<T>(u);
    }
    static_cast<T*>(p.act)[i] = static_cast<T>(activation(p.activation, g) * u);
  });
}

template <typename T>
__global__ void rr_ffn_down_naive_kernel(FfnParams p) {
  const auto* a = static_cast<const T*>(p.act);
  const auto* wd = static_cast<const T*>(p.w_down);
  const std::size_t F = p.inner, N = p.output;
  for_outputs(p.rows * N, [&](std::size_t i) {
    const std::size_t row = i / N, n = i % N;
    const int e = expert_of(p.offsets, p.experts, p.rows, static_cast<int>(row));
    if (e < 0) return;
    float s = 0.0F;
    for (std::size_t f = 0; f < F; ++f) {
      s = __builtin_fmaf(static_cast<float>(a[row * F + f]), static_cast<float>(wd[(e * F + f) * N + n]), s);
    }
    if (p.y_f32) {
      static_cast<float*>(p.y)[i] = s;
    } else {
      static_cast<T*>(p.y)[i] = static_cast<T>(s);
    }
  });
}

template <typename T>
__global__ void rr_ffn_d_gate_up_naive_kernel(FfnParams p) {
  const auto* dy = static_cast<const T*>(p.dy);
  const auto* wd = static_cast<const T*>(p.w_down);
  const std::size_t F = p.inner, N = p.output;
  for_outputs(p.rows * F, [&](std::size_t i) {
    const std::size_t row = i / F, f = i % F;
    const int e = expert_of(p.offsets, p.experts, p.rows, static_cast<int>(row));
    if (e < 0) return;
    float da = 0.0F;
    for (std::size_t n = 0; n < N; ++n) {
      da = __builtin_fmaf(static_cast<float>(dy[row * N + n]), static_cast<float>(wd[(e * F + f) * N + n]), da);
    }
    float act, grad;
    activation_grad(p.activation, static_cast<float>(static_cast<const T*>(p.gate)[i]), &act, &grad);
    static_cast<T*>(p.d_gate)[i] = static_cast<T>(da * static_cast<float>(static_cast<const T*>(p.up)[i]) * grad);
    static_cast<T*>(p.d_up)[i] = static_cast<T>(da * act);
  });
}

template <typename T>
__global__ void rr_ffn_dx_naive_kernel(FfnParams p) {
  const auto* dg = static_cast<const T*>(p.d_gate);
  const auto* du = static_cast<const T*>(p.d_up);
  const auto* wg = static_cast<const T*>(p.w_gate);
  const auto* wu = static_cast<const T*>(p.w_up);
  const std::size_t K = p.hidden, F = p.inner;
  for_outputs(p.rows * K, [&](std::size_t i) {
    const std::size_t row = i / K, k = i % K;
    const int e = expert_of(p.offsets, p.experts, p.rows, static_cast<int>(row));
    if (e < 0) return;
    float s = 0.0F;
    for (std::size_t f = 0; f < F; ++f) {
      s = __builtin_fmaf(static_cast<float>(dg[row * F + f]), static_cast<float>(wg[(e * K + k) * F + f]), s);
    }
    for (std::size_t f = 0; f < F; ++f) {
      s = __builtin_fmaf(static_cast<float>(du[row * F + f]), static_cast<float>(wu[(e * K + k) * F + f]), s);
    }
    static_cast<T*>(p.dx)[i] = static_cast<T>(s);
  });
}

// dw[e][i][j] = sum over the rows r of expert e of a[r][i] b[r][j]
template <typename T>
__global__ void rr_ffn_dw_naive_kernel(const T* a, const T* b, T* dw, const int32_t* offsets, int rows, int experts,
                                       std::size_t I, std::size_t J) {
  for_outputs(experts * I * J, [&](std::size_t o) {
    const int e = static_cast<int>(o / (I * J));
    const std::size_t i = o / J % I, j = o % J;
    const int first = first_row(offsets, e, rows), end = max(first, offset_at(offsets, e + 1, rows));
    float s = 0.0F;
    for (int r = first; r < end; ++r) s = __builtin_fmaf(static_cast<float>(a[r * I + i]), static_cast<float>(b[r * J + j]), s);
    dw[o] = static_cast<T>(s);
  });
}

__global__ void rr_int8_gemm_naive_kernel(Int8Params p) {
  const std::size_t K = p.hidden, N = p.output;
  for_outputs(p.rows * N, [&](std::size_t i) {
    const std::size_t row = i / N, n = i % N;
    const int e = expert_of(p.offsets, p.experts, p.rows, static_cast<int>(row));
    if (e < 0) return;
    auto product = [&](const int8_t* w, const float* scale) {
      uint32_t s = 0;
      for (std::size_t k = 0; k < K; ++k) s += static_cast<uint32_t>(static_cast<int>(p.q[row * K + k]) * static_cast<int>(w[(e * N + n) * K + k]));
      float sum[1] = {static_cast<float>(static_cast<int32_t>(s))};
      rr::dev::mend_int8_sums(sum, p.hidden);
      return sum[0] * p.q_scale[row] * scale[e * N + n];
    };
    float v = product(p.w, p.w_scale);
    if (p.w_up != nullptr) v = activation(p.activation, v) * product(p.w_up, p.w_up_scale);
    if (p.dtype == RR_DTYPE_FP32) {
      static_cast<float*>(p.y)[i] = v;
    } else if (p.dtype == RR_DTYPE_BF16) {
      static_cast<rr::dev::bf16*>(p.y)[i] = static_cast<rr::dev::bf16>(v);
    } else {
      static_cast<rr::dev::f16*>(p.y)[i] = static_cast<rr::dev::f16>(v);
    }
  });
}

// An E2M1 number.
__device__ float e2m1(int code) {
  const int e = (code >> 1) & 3, m = code & 1;
  const float v = e == 0 ? 0.5F * m : 0.5F * static_cast<float>((2 + m) << (e - 1));
  return (code & 8) != 0 ? -v : v;
}

__global__ void rr_mxfp4_gemm_naive_kernel(MxGemmParams p) {
  const std::size_t N = p.output, blocks = mx_blocks(p.hidden);
  const std::size_t channels = static_cast<std::size_t>(p.experts) * N;
  for_outputs(p.rows * N, [&](std::size_t i) {
    const std::size_t row = i / N, n = i % N;
    const int e = expert_of(p.offsets, p.experts, p.rows, static_cast<int>(row));
    if (e < 0) return;
    const std::size_t channel = e * N + n;
    auto product = [&](const uint8_t* w, const uint8_t* w_scale) {
      float sum = 0.0F;
      for (std::size_t b = 0; b < blocks; ++b) {
        float part = 0.0F;  // (exact: quarters up to 32 * 36)
        for (std::size_t k = 0; k < 16; ++k) {
          const int x = p.q[(row * blocks + b) * 16 + k], y = w[(channel * blocks + b) * 16 + k];
          part += e2m1(x & 15) * e2m1(y & 15) + e2m1(x >> 4) * e2m1(y >> 4);
        }
        const int xs = p.q_scale[(b / 8 * p.rows + row) * 8 + b % 8], ys = w_scale[(b / 8 * channels + channel) * 8 + b % 8];
        sum += xs == 255 || ys == 255 ? __builtin_nanf("") : ldexpf(part, xs + ys - 254);
      }
      return sum;
    };
    float v = product(p.w, p.w_scale);
    if (p.w_up != nullptr) v = activation(p.activation, v) * product(p.w_up, p.w_up_scale);
    if (p.dtype == RR_DTYPE_FP32) {
      static_cast<float*>(p.y)[i] = v;
    } else if (p.dtype == RR_DTYPE_BF16) {
      static_cast<rr::dev::bf16*>(p.y)[i] = static_cast<rr::dev::bf16>(v);
    } else {
      static_cast<rr::dev::f16*>(p.y)[i] = static_cast<rr::dev::f16>(v);
    }
  });
}

template <typename T>
hipError_t ffn_forward(const FfnParams& p, hipStream_t stream) {
  const std::size_t rows = p.rows;
  if (rows == 0) return hipSuccess;
  rr_ffn_gate_up_naive_kernel<T><<<grid_for(rows * p.inner), kThreads, 0, stream>>>(p);
  rr_ffn_down_naive_kernel<T><<<grid_for(rows * p.output), kThreads, 0, stream>>>(p);
  return hipGetLastError();
}

template <typename T>
hipError_t ffn_backward(const FfnParams& p, hipStream_t stream) {
  const std::size_t rows = p.rows, K = p.hidden, F = p.inner, N = p.output;
  if (rows != 0) rr_ffn_d_gate_up_naive_kernel<T><<<grid_for(rows * F), kThreads, 0, stream>>>(p);
  if (rows != 0 && p.dx != nullptr) rr_ffn_dx_naive_kernel<T><<<grid_for(rows * K), kThreads, 0, stream>>>(p);
  auto weights = [&](const void* a, const void* b, void* dw, std::size_t I, std::size_t J) {
    if (dw == nullptr) return;
    rr_ffn_dw_naive_kernel<T><<<grid_for(p.experts * I * J), kThreads, 0, stream>>>(
        static_cast<const T*>(a), static_cast<const T*>(b), static_cast<T*>(dw), p.offsets, p.rows, p.experts, I, J);
  };
  weights(p.x, p.d_gate, p.dw_gate, K, F);
  weights(p.x, p.d_up, p.dw_up, K, F);
  weights(p.act, p.dy, p.dw_down, F, N);
  return hipGetLastError();
}

}  // namespace

hipError_t gated_ffn_naive(const FfnParams& p, hipStream_t stream) {
  return p.bf16 ? ffn_forward<rr::dev::bf16>(p, stream) : ffn_forward<rr::dev::f16>(p, stream);
}

hipError_t gated_ffn_backward_naive(const FfnParams& p, hipStream_t stream) {
  return p.bf16 ? ffn_backward<rr::dev::bf16>(p, stream) : ffn_backward<rr::dev::f16>(p, stream);
}

hipError_t int8_grouped_gemm_naive(const Int8Params& p, hipStream_t stream) {
  if (p.rows == 0) return hipSuccess;
  rr_int8_gemm_naive_kernel<<<grid_for(static_cast<std::size_t>(p.rows) * p.output), kThreads, 0, stream>>>(p);
  return hipGetLastError();
}

hipError_t mxfp4_grouped_gemm_naive(const MxGemmParams& p, hipStream_t stream) {
  rr_mxfp4_gemm_naive_kernel<<<grid_for(static_cast<std::size_t>(p.rows) * p.output), kThreads, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace rr::kern
