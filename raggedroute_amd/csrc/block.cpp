// C ABI of the expert block's operators: argument checks -> kernel family -> launch.
//
// Checks go in the order of the other wrappers: struct and context, sizes, data
// types, architecture and family, then (unless there is nothing to do) pointers,
// alignment and workspace. Wrappers never allocate and never synchronise.
#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>
#include <initializer_list>

#include "block.h"
#include "common.h"

namespace rr {
namespace {

constexpr std::size_t kWorkspaceAlignment = 16;

bool is_16bit(int32_t dtype) noexcept { return dtype == RR_DTYPE_FP16 || dtype == RR_DTYPE_BF16; }
bool is_block_type(int32_t dtype) noexcept { return dtype == RR_DTYPE_FP32 || is_16bit(dtype); }
std::size_t type_size(int32_t dtype) noexcept { return dtype == RR_DTYPE_FP32 ? 4 : 2; }

bool width_ok(int32_t width) noexcept { return width >= 1 && width <= RR_MAX_BLOCK_WIDTH; }
bool experts_ok(int32_t experts) noexcept { return experts >= 1 && experts <= RR_MAX_EXPERTS; }
bool activation_ok(int32_t activation) noexcept {
  return activation == RR_ACT_SILU || activation == RR_ACT_GELU_TANH;
}

bool any_null(std::initializer_list<const void*> pointers) noexcept {
  for (const void* p : pointers) {
    if (p == nullptr) return true;
  }
  return false;
}

bool all_aligned(std::initializer_list<const void*> pointers, std::size_t alignment) noexcept {
  for (const void* p : pointers) {
    if (!is_aligned(p, alignment)) return false;
  }
  return true;
}

// These operators run on gfx950; id 950 is the one optimized implementation and, unless
// `naive` is null, the naive family has kernels.
rr_status choose_family(rr_kernel_selection kernel, int32_t architecture, bool* naive) noexcept {
  int32_t resolved = RR_ARCH_OTHER;
  const rr_status status = rr_resolve_device_architecture(architecture, &resolved);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (resolved != RR_ARCH_GFX950) {
    return make_status(RR_STATUS_UNSUPPORTED_ARCHITECTURE, "expert block: kernels exist for gfx950 (MI355X) only");
  }
  const bool native = (kernel.family == RR_FAMILY_AUTO && kernel.implementation_id == 0) ||
                      (kernel.family == RR_FAMILY_OPTIMIZED && kernel.implementation_id == RR_IMPL_GFX950_NATIVE);
  const bool plain = naive != nullptr && kernel.family == RR_FAMILY_NAIVE && kernel.implementation_id == 0;
  if (!native && !plain) {
    return make_status(RR_STATUS_UNSUPPORTED_KERNEL_VARIANT,
                       "expert block: no kernel has that family and implementation id");
  }
  if (naive != nullptr) *naive = plain;
  return ok_status();
}

rr_status check_workspace(const rr_runtime_context* context, std::size_t bytes, const char* message) noexcept {
  if (bytes == 0) return ok_status();
  if (context->workspace == nullptr || context->workspace_bytes < bytes) {
    return make_status(RR_STATUS_INSUFFICIENT_WORKSPACE, message);
  }
  if (!is_aligned(context->workspace, kWorkspaceAlignment)) {
    return invalid_argument("expert block: the workspace must start on a 16-byte boundary");
  }
  return ok_status();
}

std::size_t round_up(std::size_t bytes) noexcept {
  return (bytes + kWorkspaceAlignment - 1) / kWorkspaceAlignment * kWorkspaceAlignment;
}

// One of the backward pass's two [rows, inner] parts.
std::size_t ffn_part_bytes(const rr_gated_ffn_backward_args& a) noexcept {
  return round_up(static_cast<std::size_t>(a.rows) * static_cast<std::size_t>(a.inner) * type_size(a.dtype));
}

kern::NormParams norm_params(const rr_block_norm_args& a) noexcept {
  kern::NormParams p{};
  p.x = a.x;
  p.block = a.block;
  p.post_weight = a.block != nullptr ? a.post_weight : nullptr;
  p.gate = a.block != nullptr ? a.gate : nullptr;
  p.pre_weight = a.pre_weight;
  p.h = a.h;
  p.n = a.n;
  p.scale = a.residual_scale;
  p.eps = a.eps;
  p.gate_tokens = a.gate_tokens;
  p.tokens = a.tokens;
  p.hidden = a.hidden;
  p.dtype = a.dtype;
  p.block_f32 = a.block_dtype == RR_DTYPE_FP32 && a.dtype != RR_DTYPE_FP32;
  return p;
}

kern::NormParams norm_params(const rr_block_norm_backward_args& a) noexcept {
  kern::NormParams p{};
  p.x = a.h;
  p.block = a.block;
  p.post_weight = a.block != nullptr ? a.post_weight : nullptr;
  p.gate = a.block != nullptr ? a.gate : nullptr;
  p.pre_weight = a.pre_weight;
  p.dh = a.dh;
  p.dn = a.dn;
  p.dx = a.dx;
  p.dblock = p.block != nullptr ? a.dblock : nullptr;
  p.dgate = p.gate != nullptr ? a.dgate : nullptr;
  p.dpre_weight = a.dpre_weight;
  p.dpost_weight = a.dpost_weight;  // (zeros without a post norm)
  p.scale = a.residual_scale;
  p.eps = a.eps;
  p.gate_tokens = a.gate_tokens;
  p.tokens = a.tokens;
  p.hidden = a.hidden;
  p.dtype = a.dtype;
  p.block_f32 = a.block_dtype == RR_DTYPE_FP32 && a.dtype != RR_DTYPE_FP32;
  return p;
}

// Sizes and types that the two norm entries share.
template <typename Args>
rr_status check_norm(const Args& a) noexcept {
  if (a.tokens < 0 || !width_ok(a.hidden)) {
    return invalid_argument("block_norm: needs tokens >= 0 and 1 <= hidden <= 1048576");
  }
  if (!(a.eps > 0.0F)) return invalid_argument("block_norm: eps must be positive");
  if (a.block != nullptr && a.gate != nullptr && a.gate_tokens < 1) {
    return invalid_argument("block_norm: a gate needs gate_tokens >= 1");
  }
  if (!is_block_type(a.dtype) || (a.block_dtype != a.dtype && a.block_dtype != RR_DTYPE_FP32)) {
    return make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE,
                       "block_norm: dtype must be FP32, FP16 or BF16 and block_dtype the same or FP32");
  }
  return ok_status();
}

}  // namespace
}  // namespace rr

extern "C" {

size_t rr_gated_ffn_workspace_size(const rr_gated_ffn_args* args) {
  if (args == nullptr || args->rows <= 0 || args->experts <= 0 || args->hidden <= 0 || args->inner <= 0 ||
      args->output <= 0 || args->kernel.family == RR_FAMILY_NAIVE) {
    return 0;
  }
  return rr::kern::gated_ffn_parts(args->rows, args->experts, args->hidden, args->inner, args->output) * sizeof(float);
}
size_t rr_gated_ffn_backward_workspace_size(const rr_gated_ffn_backward_args* args) {
  if (args == nullptr || args->rows <= 0 || args->inner <= 0) return 0;
  return 2 * rr::ffn_part_bytes(*args);
}
size_t rr_block_norm_workspace_size(const rr_block_norm_args*) { return 0; }
size_t rr_block_norm_backward_workspace_size(const rr_block_norm_backward_args* args) {
  if (args == nullptr || args->tokens <= 0 || args->hidden <= 0 ||
      (args->block != nullptr && args->gate != nullptr && args->gate_tokens < 1)) {
    return 0;
  }
  return rr::kern::block_norm_backward_workspace(rr::norm_params(*args));
}
size_t rr_quantize_rows_workspace_size(const rr_quantize_rows_args*) { return 0; }
size_t rr_int8_grouped_gemm_workspace_size(const rr_int8_grouped_gemm_args*) { return 0; }

rr_status rr_gated_ffn(const rr_gated_ffn_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("gated_ffn: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("gated_ffn: no runtime context was given");
  const rr_gated_ffn_args& a = *args;
  if (a.rows < 0 || !rr::experts_ok(a.experts) || !rr::width_ok(a.hidden) || !rr::width_ok(a.inner) ||
      !rr::width_ok(a.output)) {
    return rr::invalid_argument(
        "gated_ffn: needs rows >= 0, 1 <= experts <= 1024 and hidden, inner, output in 1..1048576");
  }
  if (!rr::activation_ok(a.activation)) return rr::invalid_argument("gated_ffn: the activation is none of SiLU and tanh-GELU");
  if ((a.gate == nullptr) != (a.up == nullptr)) {
    return rr::invalid_argument("gated_ffn: gate and up are kept together or not at all");
  }
  if (!rr::is_16bit(a.dtype) || (a.y_dtype != a.dtype && a.y_dtype != RR_DTYPE_FP32)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE,
                           "gated_ffn: dtype must be FP16 or BF16 and y_dtype the same or FP32");
  }
  bool naive = false;
  rr_status status = rr::choose_family(a.kernel, context->architecture, &naive);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.rows == 0) return rr::ok_status();
  if (rr::any_null({a.x, a.w_gate, a.w_up, a.w_down, a.offsets, a.act, a.y})) {
    return rr::invalid_argument("gated_ffn: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.x, a.w_gate, a.w_up, a.w_down, a.gate, a.up, a.act}, 2) ||
      !rr::is_aligned(a.y, rr::type_size(a.y_dtype)) || !rr::is_aligned(a.offsets, alignof(int32_t))) {
    return rr::invalid_argument("gated_ffn: every buffer must be aligned to its element type");
  }
  status = rr::check_workspace(context, rr_gated_ffn_workspace_size(args),
                               "gated_ffn: the workspace must hold the parts of split sums");
  if (status.code != RR_STATUS_SUCCESS) return status;
  rr::kern::FfnParams p{};
  p.parts = static_cast<float*>(context->workspace);
  p.x = a.x;
  p.w_gate = a.w_gate;
  p.w_up = a.w_up;
  p.w_down = a.w_down;
  p.offsets = a.offsets;
  p.gate = a.gate;
  p.up = a.up;
  p.act = a.act;
  p.y = a.y;
  p.rows = a.rows;
  p.experts = a.experts;
  p.hidden = a.hidden;
  p.inner = a.inner;
  p.output = a.output;
  p.activation = a.activation;
  p.bf16 = a.dtype == RR_DTYPE_BF16;
  p.y_f32 = a.y_dtype == RR_DTYPE_FP32;
  return rr::device_status(naive ? rr::kern::gated_ffn_naive(p, context->stream) : rr::kern::gated_ffn(p, context->stream),
                           "gated_ffn: a kernel did not launch");
}

rr_status rr_gated_ffn_backward(const rr_gated_ffn_backward_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("gated_ffn_backward: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("gated_ffn_backward: no runtime context was given");
  const rr_gated_ffn_backward_args& a = *args;
  if (a.rows < 0 || !rr::experts_ok(a.experts) || !rr::width_ok(a.hidden) || !rr::width_ok(a.inner) ||
      !rr::width_ok(a.output)) {
    return rr::invalid_argument(
        "gated_ffn_backward: needs rows >= 0, 1 <= experts <= 1024 and hidden, inner, output in 1..1048576");
  }
  if (!rr::activation_ok(a.activation)) {
    return rr::invalid_argument("gated_ffn_backward: the activation is none of SiLU and tanh-GELU");
  }
  if ((a.dw_gate == nullptr) != (a.dw_up == nullptr)) {
    return rr::invalid_argument("gated_ffn_backward: dw_gate and dw_up are computed together or not at all");
  }
  if (!rr::is_16bit(a.dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE, "gated_ffn_backward: dtype must be FP16 or BF16");
  }
  bool naive = false;
  rr_status status = rr::choose_family(a.kernel, context->architecture, &naive);
  if (status.code != RR_STATUS_SUCCESS) return status;
  // without rows the weight gradients are still written (zeros)
  if (a.offsets == nullptr ||
      (a.rows != 0 && rr::any_null({a.x, a.w_gate, a.w_up, a.w_down, a.gate, a.up, a.act, a.dy}))) {
    return rr::invalid_argument("gated_ffn_backward: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.x, a.w_gate, a.w_up, a.w_down, a.gate, a.up, a.act, a.dy, a.dx, a.dw_gate, a.dw_up, a.dw_down}, 2) ||
      !rr::is_aligned(a.offsets, alignof(int32_t))) {
    return rr::invalid_argument("gated_ffn_backward: every buffer must be aligned to its element type");
  }
  const std::size_t bytes = rr_gated_ffn_backward_workspace_size(args);
  status = rr::check_workspace(context, bytes, "gated_ffn_backward: the workspace must hold d gate and d up");
  if (status.code != RR_STATUS_SUCCESS) return status;
  rr::kern::FfnParams p{};
  p.x = a.x;
  p.w_gate = a.w_gate;
  p.w_up = a.w_up;
  p.w_down = a.w_down;
  p.offsets = a.offsets;
  p.gate = const_cast<void*>(a.gate);  // read only
  p.up = const_cast<void*>(a.up);
  p.act = const_cast<void*>(a.act);
  p.dy = a.dy;
  p.dx = a.dx;
  p.dw_gate = a.dw_gate;
  p.dw_up = a.dw_up;
  p.dw_down = a.dw_down;
  p.d_gate = context->workspace;
  p.d_up = bytes != 0 ? static_cast<char*>(context->workspace) + bytes / 2 : nullptr;
  p.rows = a.rows;
  p.experts = a.experts;
  p.hidden = a.hidden;
  p.inner = a.inner;
  p.output = a.output;
  p.activation = a.activation;
  p.bf16 = a.dtype == RR_DTYPE_BF16;
  return rr::device_status(
      naive ? rr::kern::gated_ffn_backward_naive(p, context->stream) : rr::kern::gated_ffn_backward(p, context->stream),
      "gated_ffn_backward: a kernel did not launch");
}

rr_status rr_block_norm(const rr_block_norm_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("block_norm: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("block_norm: no runtime context was given");
  const rr_block_norm_args& a = *args;
  rr_status status = rr::check_norm(a);
  if (status.code != RR_STATUS_SUCCESS) return status;
  status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.tokens == 0) return rr::ok_status();
  if (a.x == nullptr || (a.n != nullptr && a.pre_weight == nullptr) || (a.n == nullptr && a.h == nullptr) ||
      (a.block != nullptr && a.h == nullptr)) {
    return rr::invalid_argument("block_norm: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.x, a.post_weight, a.gate, a.pre_weight, a.h, a.n}, rr::type_size(a.dtype)) ||
      !rr::is_aligned(a.block, rr::type_size(a.block_dtype))) {
    return rr::invalid_argument("block_norm: every buffer must be aligned to its element type");
  }
  return rr::device_status(rr::kern::block_norm(rr::norm_params(a), context->stream), "block_norm: a kernel did not launch");
}

rr_status rr_block_norm_backward(const rr_block_norm_backward_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("block_norm_backward: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("block_norm_backward: no runtime context was given");
  const rr_block_norm_backward_args& a = *args;
  rr_status status = rr::check_norm(a);
  if (status.code != RR_STATUS_SUCCESS) return status;
  status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  const rr::kern::NormParams p = rr::norm_params(a);
  if (a.tokens == 0) {
    // no tokens: the sums over them are zero (and tensors of none may have no address)
    if (!rr::all_aligned({a.dpre_weight, a.dpost_weight}, rr::type_size(a.dtype))) {
      return rr::invalid_argument("block_norm_backward: every buffer must be aligned to its element type");
    }
    return rr::device_status(rr::kern::block_norm_backward(p, context->stream), "block_norm_backward: a kernel did not launch");
  }
  if (a.h == nullptr || a.dx == nullptr || (a.dh == nullptr && a.dn == nullptr) ||
      (a.dn != nullptr && a.pre_weight == nullptr)) {
    return rr::invalid_argument("block_norm_backward: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.h, a.post_weight, a.gate, a.pre_weight, a.dh, a.dn, a.dx, a.dgate, a.dpre_weight, a.dpost_weight},
                       rr::type_size(a.dtype)) ||
      !rr::all_aligned({a.block, a.dblock}, rr::type_size(a.block_dtype))) {
    return rr::invalid_argument("block_norm_backward: every buffer must be aligned to its element type");
  }
  status = rr::check_workspace(context, rr_block_norm_backward_workspace_size(args),
                               "block_norm_backward: the workspace must hold the parts' column sums");
  if (status.code != RR_STATUS_SUCCESS) return status;
  rr::kern::NormParams q = p;
  q.sums = static_cast<float*>(context->workspace);
  return rr::device_status(rr::kern::block_norm_backward(q, context->stream), "block_norm_backward: a kernel did not launch");
}

rr_status rr_quantize_rows(const rr_quantize_rows_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("quantize_rows: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("quantize_rows: no runtime context was given");
  const rr_quantize_rows_args& a = *args;
  if (a.rows < 0 || !rr::width_ok(a.hidden)) {
    return rr::invalid_argument("quantize_rows: needs rows >= 0 and 1 <= hidden <= 1048576");
  }
  if (!rr::is_block_type(a.dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE, "quantize_rows: dtype must be FP32, FP16 or BF16");
  }
  const rr_status status = rr::choose_family(a.kernel, context->architecture, nullptr);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.rows == 0) return rr::ok_status();
  if (rr::any_null({a.x, a.q, a.scale})) {
    return rr::invalid_argument("quantize_rows: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::is_aligned(a.x, rr::type_size(a.dtype)) || !rr::is_aligned(a.scale, alignof(float))) {
    return rr::invalid_argument("quantize_rows: every buffer must be aligned to its element type");
  }
  return rr::device_status(rr::kern::quantize_rows(a.x, a.q, a.scale, a.rows, a.hidden, a.dtype, context->stream),
                           "quantize_rows: the kernel did not launch");
}

rr_status rr_int8_grouped_gemm(const rr_int8_grouped_gemm_args* args, const rr_runtime_context* context) {
  if (args == nullptr) return rr::invalid_argument("int8_grouped_gemm: no argument struct was given");
  if (context == nullptr) return rr::invalid_argument("int8_grouped_gemm: no runtime context was given");
  const rr_int8_grouped_gemm_args& a = *args;
  if (a.rows < 0 || !rr::experts_ok(a.experts) || !rr::width_ok(a.hidden) || a.hidden > rr::kern::kMostInt8Hidden ||
      !rr::width_ok(a.output)) {
    return rr::invalid_argument(
        "int8_grouped_gemm: needs rows >= 0, 1 <= experts <= 1024, hidden in 1..131072 and output in 1..1048576");
  }
  if (!rr::is_block_type(a.dtype)) {
    return rr::make_status(RR_STATUS_UNSUPPORTED_DATA_TYPE, "int8_grouped_gemm: dtype must be FP32, FP16 or BF16");
  }
  if (a.w_up != nullptr && !rr::activation_ok(a.activation)) {
    return rr::invalid_argument("int8_grouped_gemm: the activation is none of SiLU and tanh-GELU");
  }
  bool naive = false;
  const rr_status status = rr::choose_family(a.kernel, context->architecture, &naive);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (a.rows == 0) return rr::ok_status();
  if (rr::any_null({a.q, a.q_scale, a.w, a.w_scale, a.offsets, a.y}) || (a.w_up != nullptr && a.w_up_scale == nullptr)) {
    return rr::invalid_argument("int8_grouped_gemm: a buffer the call reads or writes is a null pointer");
  }
  if (!rr::all_aligned({a.q_scale, a.w_scale, a.w_up_scale, a.offsets}, alignof(float)) ||
      !rr::is_aligned(a.y, rr::type_size(a.dtype))) {
    return rr::invalid_argument("int8_grouped_gemm: every buffer must be aligned to its element type");
  }
  rr::kern::Int8Params p{};
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
      naive ? rr::kern::int8_grouped_gemm_naive(p, context->stream) : rr::kern::int8_grouped_gemm(p, context->stream),
      "int8_grouped_gemm: a kernel did not launch");
}

}  // extern "C"
