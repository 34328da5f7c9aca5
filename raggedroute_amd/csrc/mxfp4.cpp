// C ABI of the 4-bit operators: argument checks -> kernel family -> launch, in the order
// of block.cpp's wrappers.
#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>
#include <limits>

#include "block_checks.h"
#include "common.h"
#include "mxfp4.h"

extern "C" {

size_t rr_quantize_rows_mxfp4_workspace_size(const rr_quantize_rows_mxfp4_args*) { return 0; }
size_t rr_mxfp4_grouped_gemm_workspace_size(const rr_mxfp4_grouped_gemm_args*) { return 0; }

rr_status rr_quantize_rows_mxfp4(const rr_quantize_rows_mxfp4_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("quantize_rows_mxfp4: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("quantize_rows_mxfp4: no runtime context was given");
  const rr_quantize_rows_mxfp4_args& a = *args;
  if (a.rows < 0 || !rr::width_ok(a.hidden)) {
    return rr::invalid_argument("quantize_rows_mxfp4: needs rows >= 0 and 1 <= hidden <= 1048576");
  }
  if (a.sorted_route != nullptr && (a.tokens < 0 || a.top_k < 1 || a.top_k > RR_MAX_SORT_TOP_K ||
                                    static_cast<int64_t>(a.tokens) * a.top_k > std::numeric_limits<int32_t>::max())) {
    return rr::invalid_argument(
        "quantize_rows_mxfp4: with sorted_route needs tokens >= 0, top_k in 1..64 and tokens * top_k within 31 bits");
  }
  if (!rr::is_block_type(a.dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE, "quantize_rows_mxfp4: dtype must be FP32, FP16 or BF16");
  }
  const rr_status status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.rows == 0 || (a.sorted_route != nullptr && a.tokens == 0)) return rr::ok_status();
  if (rr::any_null({a.x, a.q, a.scale})) {
    return rr::invalid_argument("quantize_rows_mxfp4: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::is_aligned(a.x, rr::type_size(a.dtype)) || !rr::is_aligned(a.sorted_route, alignof(int32_t)) ||
      !rr::is_aligned(a.q, 16) || !rr::is_aligned(a.scale, 8)) {
    return rr::invalid_argument(
        "quantize_rows_mxfp4: x and sorted_route must be aligned to their element types, q to 16 bytes, scale to 8");
  }
  rr::kern::MxQuantizeParams p{};
  p.x = a.x;
  p.sorted_route = a.sorted_route;
  p.q = a.q;
  p.scale = a.scale;
  p.rows = a.rows;
  p.hidden = a.hidden;
  p.tokens = a.tokens;
  p.top_k = a.top_k;
  p.dtype = a.dtype;
  return rr::device_status(rr::kern::quantize_rows_mxfp4(p, context->stream),
                           "quantize_rows_mxfp4: the kernel did not launch");
}

rr_status rr_mxfp4_grouped_gemm(const rr_mxfp4_grouped_gemm_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("mxfp4_grouped_gemm: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("mxfp4_grouped_gemm: no runtime context was given");
  const rr_mxfp4_grouped_gemm_args& a = *args;
  if (a.rows < 0 || !rr::experts_ok(a.experts) || !rr::width_ok(a.hidden) || !rr::width_ok(a.output)) {
    return rr::invalid_argument(
        "mxfp4_grouped_gemm: needs rows >= 0, 1 <= experts <= 1024 and hidden, output in 1..1048576");
  }
  if (!rr::is_block_type(a.dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE, "mxfp4_grouped_gemm: dtype must be FP32, FP16 or BF16");
  }
  if (a.w_up != nullptr && !rr::activation_ok(a.activation)) {
    return rr::invalid_argument("mxfp4_grouped_gemm: the activation is none of SiLU and tanh-GELU");
  }
  bool naive = false;
  const rr_status status = rr::choose_family(a.kernel, context->architecture, &naive);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.rows == 0) return rr::ok_status();
  if (rr::any_null({a.q, a.q_scale, a.w, a.w_scale, a.offsets, a.y}) || (a.w_up != nullptr && a.w_up_scale == nullptr)) {
    return rr::invalid_argument("mxfp4_grouped_gemm: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.q, a.w, a.w_up}, 16) || !rr::all_aligned({a.q_scale, a.w_scale, a.w_up_scale}, 8) ||
      !rr::is_aligned(a.offsets, alignof(int32_t)) || !rr::is_aligned(a.y, rr::type_size(a.dtype))) {
    return rr::invalid_argument(
        "mxfp4_grouped_gemm: q, w and w_up must be aligned to 16 bytes, scales to 8, the others to their element type");
  }
  rr::kern::MxGemmParams p{};
  p.q = a.q;
  p.q_scale = a.q_scale;
  p.w = a.w;
  p.w_scale = a.w_scale;
  p.w_up = a.w_up;
  p.w_up_scale = a.w_up_scale;
  p.offsets = a.offsets;
  p.y = a.y;
  p.rows = a.rows;
  p.experts = a.experts;
  p.hidden = a.hidden;
  p.output = a.output;
  p.activation = a.activation;
  p.dtype = a.dtype;
  return rr::device_status(
      naive ? rr::kern::mxfp4_grouped_gemm_naive(p, context->stream) : rr::kern::mxfp4_grouped_gemm(p, context->stream),
      "mxfp4_grouped_gemm: a kernel did not launch");
}

}  // extern "C"
