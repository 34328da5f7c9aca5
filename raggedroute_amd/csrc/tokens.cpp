// C ABI of the operators that take tokens to their experts and back: argument checks ->
// launch, in the order of block.cpp's wrappers.
#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>
#include <limits>

#include "block_checks.h"
#include "common.h"
#include "tokens.h"

namespace rr {
namespace {

bool routes_ok(int32_t tokens, int32_t top_k) noexcept {
  return tokens >= 0 && top_k >= 1 && top_k <= RR_MAX_SORT_TOP_K &&
         static_cast<int64_t>(tokens) * top_k <= std::numeric_limits<int32_t>::max();
}

// dtype of the sorted rows, `other` of the tokens' rows
bool types_ok(int32_t dtype, int32_t other) noexcept {
  return is_block_type(dtype) && (other == dtype || other == RR_DTYPE_FP32);
}

}  // namespace
}  // namespace rr

extern "C" {

size_t rr_sort_tokens_workspace_size(const rr_sort_tokens_args* args) {
  if (args == nullptr || !rr::routes_ok(args->tokens, args->top_k) || !rr::experts_ok(args->experts)) return 0;
  return rr::kern::sort_tokens_counts(static_cast<int64_t>(args->tokens) * args->top_k, args->experts) * sizeof(int32_t);
}
size_t rr_sort_tokens_backward_workspace_size(const rr_sort_tokens_backward_args*) { return 0; }
size_t rr_combine_tokens_workspace_size(const rr_combine_tokens_args*) { return 0; }
size_t rr_combine_tokens_backward_workspace_size(const rr_combine_tokens_backward_args*) { return 0; }
size_t rr_topk_gate_backward_workspace_size(const rr_topk_gate_backward_args*) { return 0; }

rr_status rr_sort_tokens(const rr_sort_tokens_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("sort_tokens: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("sort_tokens: no runtime context was given");
  const rr_sort_tokens_args& a = *args;
  // (the maps alone have no rows)
  if (!rr::routes_ok(a.tokens, a.top_k) || !rr::experts_ok(a.experts) || (a.x_sorted != nullptr && !rr::width_ok(a.hidden))) {
    return rr::invalid_argument(
        "sort_tokens: needs tokens >= 0, top_k in 1..64, tokens * top_k within 31 bits, 1 <= experts <= 1024 and, with "
        "x_sorted, hidden in 1..1048576");
  }
  if (!rr::types_ok(a.dtype, a.x_dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE,
                           "sort_tokens: dtype must be FP32, FP16 or BF16 and x_dtype the same or FP32");
  }
  rr_status status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  // without tokens the offsets are still written (zeros)
  if (a.offsets == nullptr || (a.tokens != 0 && rr::any_null({a.expert_ids, a.route_pos})) ||
      (a.tokens != 0 && a.x_sorted != nullptr && a.x == nullptr)) {
    return rr::invalid_argument("sort_tokens: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.expert_ids, a.offsets, a.route_pos, a.sorted_route}, alignof(int32_t)) ||
      !rr::is_aligned(a.x, rr::type_size(a.x_dtype)) || !rr::is_aligned(a.x_sorted, rr::type_size(a.dtype))) {
    return rr::invalid_argument("sort_tokens: every buffer must be aligned to its element type");
  }
  status = rr::check_workspace(context, rr_sort_tokens_workspace_size(args),
                               "sort_tokens: the workspace must hold the counts of parts of the routes");
  if (status.code != RR_STATUS_SUCCESS) return status;
  rr::kern::SortParams p{};
  p.counts = static_cast<int32_t*>(context->workspace);
  p.x = a.x;
  p.ids = a.expert_ids;
  p.offsets = a.offsets;
  p.route_pos = a.route_pos;
  p.sorted_route = a.sorted_route;
  p.x_sorted = a.x_sorted;
  p.tokens = a.tokens;
  p.experts = a.experts;
  p.top_k = a.top_k;
  p.hidden = a.hidden;
  p.dtype = a.dtype;
  p.x_f32 = a.x_dtype == RR_DTYPE_FP32 && a.dtype != RR_DTYPE_FP32;
  return rr::device_status(rr::kern::sort_tokens(p, context->stream), "sort_tokens: a kernel did not launch");
}

rr_status rr_sort_tokens_backward(const rr_sort_tokens_backward_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("sort_tokens_backward: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("sort_tokens_backward: no runtime context was given");
  const rr_sort_tokens_backward_args& a = *args;
  if (!rr::routes_ok(a.tokens, a.top_k) || !rr::width_ok(a.hidden)) {
    return rr::invalid_argument(
        "sort_tokens_backward: needs tokens >= 0, top_k in 1..64, tokens * top_k within 31 bits and hidden in 1..1048576");
  }
  if (!rr::types_ok(a.dtype, a.x_dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE,
                           "sort_tokens_backward: dtype must be FP32, FP16 or BF16 and x_dtype the same or FP32");
  }
  const rr_status status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.tokens == 0) return rr::ok_status();
  if (rr::any_null({a.dx_sorted, a.route_pos, a.dx})) {
    return rr::invalid_argument("sort_tokens_backward: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::is_aligned(a.dx_sorted, rr::type_size(a.dtype)) || !rr::is_aligned(a.dx, rr::type_size(a.x_dtype)) ||
      !rr::is_aligned(a.route_pos, alignof(int32_t))) {
    return rr::invalid_argument("sort_tokens_backward: every buffer must be aligned to its element type");
  }
  rr::kern::CombineParams p{};
  p.sorted = a.dx_sorted;
  p.route_pos = a.route_pos;
  p.out = a.dx;
  p.tokens = a.tokens;
  p.top_k = a.top_k;
  p.hidden = a.hidden;
  p.dtype = a.dtype;
  p.tokens_f32 = a.x_dtype == RR_DTYPE_FP32 && a.dtype != RR_DTYPE_FP32;
  return rr::device_status(rr::kern::combine_tokens(p, context->stream), "sort_tokens_backward: the kernel did not launch");
}

rr_status rr_combine_tokens(const rr_combine_tokens_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("combine_tokens: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("combine_tokens: no runtime context was given");
  const rr_combine_tokens_args& a = *args;
  if (!rr::routes_ok(a.tokens, a.top_k) || !rr::width_ok(a.hidden)) {
    return rr::invalid_argument(
        "combine_tokens: needs tokens >= 0, top_k in 1..64, tokens * top_k within 31 bits and hidden in 1..1048576");
  }
  if (!rr::types_ok(a.dtype, a.y_dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE,
                           "combine_tokens: dtype must be FP32, FP16 or BF16 and y_dtype the same or FP32");
  }
  const rr_status status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.tokens == 0) return rr::ok_status();
  if (rr::any_null({a.y_sorted, a.route_pos, a.y})) {
    return rr::invalid_argument("combine_tokens: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::is_aligned(a.y_sorted, rr::type_size(a.dtype)) || !rr::is_aligned(a.y, rr::type_size(a.y_dtype)) ||
      !rr::is_aligned(a.route_pos, alignof(int32_t)) || !rr::is_aligned(a.route_weights, alignof(float))) {
    return rr::invalid_argument("combine_tokens: every buffer must be aligned to its element type");
  }
  rr::kern::CombineParams p{};
  p.sorted = a.y_sorted;
  p.route_pos = a.route_pos;
  p.weights = a.route_weights;
  p.out = a.y;
  p.tokens = a.tokens;
  p.top_k = a.top_k;
  p.hidden = a.hidden;
  p.dtype = a.dtype;
  p.tokens_f32 = a.y_dtype == RR_DTYPE_FP32 && a.dtype != RR_DTYPE_FP32;
  return rr::device_status(rr::kern::combine_tokens(p, context->stream), "combine_tokens: the kernel did not launch");
}

rr_status rr_combine_tokens_backward(const rr_combine_tokens_backward_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("combine_tokens_backward: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("combine_tokens_backward: no runtime context was given");
  const rr_combine_tokens_backward_args& a = *args;
  if (!rr::routes_ok(a.tokens, a.top_k) || !rr::width_ok(a.hidden)) {
    return rr::invalid_argument(
        "combine_tokens_backward: needs tokens >= 0, top_k in 1..64, tokens * top_k within 31 bits and hidden in "
        "1..1048576");
  }
  if (!rr::types_ok(a.dtype, a.y_dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE,
                           "combine_tokens_backward: dtype must be FP32, FP16 or BF16 and y_dtype the same or FP32");
  }
  const rr_status status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.tokens == 0 || (a.dy_sorted == nullptr && a.droute_weights == nullptr)) return rr::ok_status();
  if (rr::any_null({a.dy, a.route_pos}) || (a.droute_weights != nullptr && a.y_sorted == nullptr)) {
    return rr::invalid_argument("combine_tokens_backward: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.y_sorted, a.dy_sorted}, rr::type_size(a.dtype)) ||
      !rr::is_aligned(a.dy, rr::type_size(a.y_dtype)) ||
      !rr::all_aligned({a.route_pos, a.route_weights, a.droute_weights}, alignof(float))) {
    return rr::invalid_argument("combine_tokens_backward: every buffer must be aligned to its element type");
  }
  rr::kern::CombineParams p{};
  p.sorted = a.y_sorted;
  p.route_pos = a.route_pos;
  p.weights = a.route_weights;
  p.dy = a.dy;
  p.dy_sorted = a.dy_sorted;
  p.dweights = a.droute_weights;
  p.tokens = a.tokens;
  p.top_k = a.top_k;
  p.hidden = a.hidden;
  p.dtype = a.dtype;
  p.tokens_f32 = a.y_dtype == RR_DTYPE_FP32 && a.dtype != RR_DTYPE_FP32;
  return rr::device_status(rr::kern::combine_tokens_backward(p, context->stream),
                           "combine_tokens_backward: the kernel did not launch");
}

rr_status rr_topk_gate_backward(const rr_topk_gate_backward_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("topk_gate_backward: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("topk_gate_backward: no runtime context was given");
  const rr_topk_gate_backward_args& a = *args;
  if (!rr::routes_ok(a.tokens, a.top_k) || !rr::experts_ok(a.experts)) {
    return rr::invalid_argument(
        "topk_gate_backward: needs tokens >= 0, top_k in 1..64, tokens * top_k within 31 bits and 1 <= experts <= 1024");
  }
  const rr_status status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.tokens == 0) return rr::ok_status();
  if (rr::any_null({a.expert_ids, a.weights, a.dweights, a.dlogits})) {
    return rr::invalid_argument("topk_gate_backward: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.expert_ids, a.weights, a.dweights, a.dlogits}, alignof(float))) {
    return rr::invalid_argument("topk_gate_backward: every buffer must be aligned to its element type");
  }
  rr::kern::GateBackwardParams p{};
  p.ids = a.expert_ids;
  p.weights = a.weights;
  p.dweights = a.dweights;
  p.dlogits = a.dlogits;
  p.tokens = a.tokens;
  p.experts = a.experts;
  p.top_k = a.top_k;
  return rr::device_status(rr::kern::topk_gate_backward(p, context->stream),
                           "topk_gate_backward: the kernel did not launch");
}

}  // extern "C"
