// Parameters and launchers of the operators that take tokens to their experts and back,
// with their gradients (formulas and shapes in raggedroute_capi.h). Arguments are
// validated by tokens.cpp; every launcher returns the launch error.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace rr::kern {

struct SortParams {
  const void* x;
  const int32_t* ids;
  int32_t* offsets;
  int32_t* route_pos;
  int32_t* sorted_route;  // optional
  void* x_sorted;         // optional
  int32_t* counts;        // workspace: sort_tokens_counts() numbers
  int tokens, experts, top_k, hidden;
  int dtype;
  bool x_f32;  // x FP32 beside a 16-bit dtype
};

// Rows of tokens and their sorted rows. Forward: out[t] = sum_j w[t, j] sorted[pos[t, j]].
struct CombineParams {
  const void* sorted;
  const int32_t* route_pos;
  const float* weights;  // optional: 1
  void* out;
  const void* dy;      // backward, as all below
  void* dy_sorted;     // optional
  float* dweights;     // optional
  int tokens, top_k, hidden;
  int dtype;
  bool tokens_f32;  // the tokens' rows FP32 beside a 16-bit dtype
};

struct GateBackwardParams {
  const int32_t* ids;
  const float* weights;
  const float* dweights;
  float* dlogits;
  int tokens, experts, top_k;
};

// 32-bit numbers of workspace that sort_tokens needs.
std::size_t sort_tokens_counts(int64_t routes, int experts);
hipError_t sort_tokens(const SortParams& prm, hipStream_t stream);
hipError_t combine_tokens(const CombineParams& prm, hipStream_t stream);
hipError_t combine_tokens_backward(const CombineParams& prm, hipStream_t stream);
hipError_t topk_gate_backward(const GateBackwardParams& prm, hipStream_t stream);

}  // namespace rr::kern
