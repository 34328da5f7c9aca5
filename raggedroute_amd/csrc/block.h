// Parameters and launchers of the expert block's operators (gated feed-forward,
// int8 products, norms). Arguments are validated by block.cpp; every launcher
// returns the launch error.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace rr::kern {

// Gated feed-forward block, forward and backward (see raggedroute_capi.h for the
// formulas and shapes). Rows of expert e: [offsets[e], offsets[e + 1]), cut to
// [0, rows].
struct FfnParams {
  const void* x;
  const void* w_gate;
  const void* w_up;
  const void* w_down;
  const int32_t* offsets;
  void* gate;  // forward: optional
  void* up;
  void* act;
  void* y;         // forward
  const void* dy;  // backward, as all below
  void* dx;        // optional, as the other gradients
  void* dw_gate;
  void* dw_up;
  void* dw_down;
  float* parts;  // workspace, forward: gated_ffn_parts() floats
  void* d_gate;  // workspace, backward: [rows, inner]
  void* d_up;
  int rows, experts, hidden, inner, output;
  int activation;
  bool bf16;   // else FP16
  bool y_f32;  // forward: y is FP32
};

constexpr int kMostInt8Hidden = 131072;  // length of an int8 sum

struct Int8Params {
  const int8_t* q;
  const float* q_scale;
  const int8_t* w;
  const float* w_scale;
  const int8_t* w_up;  // gated
  const float* w_up_scale;
  const int32_t* offsets;
  void* y;
  int rows, experts, hidden, output;
  int activation;
  int dtype;  // of y
};

struct NormParams {
  const void* x;  // backward: h
  const void* block;
  const void* post_weight;
  const void* gate;
  const void* pre_weight;
  void* h;  // forward
  void* n;
  const void* dh;  // backward, as all below
  const void* dn;
  void* dx;
  void* dblock;
  void* dgate;
  void* dpre_weight;
  void* dpost_weight;
  float* sums;  // workspace
  float scale, eps;
  int gate_tokens, tokens, hidden;
  int dtype;
  bool block_f32;  // block (and dblock) FP32 beside a 16-bit dtype
};

// ---- products on the matrix cores ----
// FP32 values of workspace that the forward call needs.
std::size_t gated_ffn_parts(int rows, int experts, int hidden, int inner, int output);
hipError_t gated_ffn(const FfnParams& prm, hipStream_t stream);
hipError_t gated_ffn_backward(const FfnParams& prm, hipStream_t stream);
hipError_t int8_grouped_gemm(const Int8Params& prm, hipStream_t stream);

// ---- naive forms (block_naive.hip) ----
hipError_t gated_ffn_naive(const FfnParams& prm, hipStream_t stream);
hipError_t gated_ffn_backward_naive(const FfnParams& prm, hipStream_t stream);
hipError_t int8_grouped_gemm_naive(const Int8Params& prm, hipStream_t stream);

// ---- norms and quantisation (block_norm.hip) ----
hipError_t block_norm(const NormParams& prm, hipStream_t stream);
std::size_t block_norm_backward_workspace(const NormParams& prm);
hipError_t block_norm_backward(const NormParams& prm, hipStream_t stream);
hipError_t quantize_rows(const void* x, int8_t* q, float* scale, int rows, int hidden, int dtype, hipStream_t stream);

}  // namespace rr::kern
