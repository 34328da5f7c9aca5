// Parameters and launchers of the 4-bit operators (layouts and formulas in
// raggedroute_capi.h). Arguments are validated by mxfp4.cpp; every launcher returns the
// launch error.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace rr::kern {

constexpr int kMxBlock = 32;   // elements that share a scale
constexpr int kMxSlice = 256;  // elements whose scales lie side by side

constexpr int mx_blocks(int hidden) { return (hidden + kMxBlock - 1) / kMxBlock; }
constexpr int mx_slices(int hidden) { return (hidden + kMxSlice - 1) / kMxSlice; }

struct MxQuantizeParams {
  const void* x;
  const int32_t* sorted_route;  // optional
  uint8_t* q;
  uint8_t* scale;
  int rows, hidden;
  int tokens, top_k;  // with sorted_route
  int dtype;
};

struct MxGemmParams {
  const uint8_t* q;
  const uint8_t* q_scale;
  const uint8_t* w;
  const uint8_t* w_scale;
  const uint8_t* w_up;  // gated
  const uint8_t* w_up_scale;
  const int32_t* offsets;
  void* y;
  int rows, experts, hidden, output;
  int activation;
  int dtype;  // of y
};

hipError_t quantize_rows_mxfp4(const MxQuantizeParams& prm, hipStream_t stream);
hipError_t mxfp4_grouped_gemm(const MxGemmParams& prm, hipStream_t stream);
hipError_t mxfp4_grouped_gemm_naive(const MxGemmParams& prm, hipStream_t stream);  // block_naive.hip

}  // namespace rr::kern
