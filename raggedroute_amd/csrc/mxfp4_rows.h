// 4-bit products for few rows an expert (mxfp4_rows.hip).
#pragma once

#include <hip/hip_runtime_api.h>

#include "expert_gemm.h"

namespace rr::kern {

// Whether the kernel for few rows takes a product of this many rows.
bool mxfp4_rows_ok(int rows, int experts);
// prm as rr_mxfp4_gemm_kernel's.
template <class Epi>
hipError_t mxfp4_rows(const Product& prm, hipStream_t stream);

}  // namespace rr::kern
