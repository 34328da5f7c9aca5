// Argument checks that the wrappers of the expert block's, the token and the 4-bit operators share.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

#include "common.h"

namespace rr {

constexpr std::size_t kWorkspaceAlignment = 16;

inline bool is_16bit(int32_t dtype) noexcept { return dtype == RR_DTYPE_FP16 || dtype == RR_DTYPE_BF16; }
inline bool is_block_type(int32_t dtype) noexcept { return dtype == RR_DTYPE_FP32 || is_16bit(dtype); }
inline std::size_t type_size(int32_t dtype) noexcept { return dtype == RR_DTYPE_FP32 ? 4 : 2; }

inline bool width_ok(int32_t width) noexcept { return width >= 1 && width <= RR_MAX_BLOCK_WIDTH; }
inline bool experts_ok(int32_t experts) noexcept { return experts >= 1 && experts <= RR_MAX_EXPERTS; }
inline bool activation_ok(int32_t activation) noexcept {
  return activation == RR_ACT_SILU || activation == RR_ACT_GELU_TANH;
}

inline bool any_null(std::initializer_list<const void*> pointers) noexcept {
  for (const void* p : pointers) {
    if (p == nullptr) return true;
  }
  return false;
}

inline bool all_aligned(std::initializer_list<const void*> pointers, std::size_t alignment) noexcept {
  for (const void* p : pointers) {
    if (!is_aligned(p, alignment)) return false;
  }
  return true;
}

// These operators run on gfx950; id 950 is the one optimized implementation and, unless
// `naive` is null, the naive family has kernels.
inline rr_status choose_family(rr_kernel_selection kernel, int32_t architecture, bool* naive) noexcept {
  int32_t resolved = RR_ARCH_OTHER;
  const rr_status status = rr_resolve_device_architecture(architecture, &resolved);
  if (status.code != RR_STATUS_SUCCESS) return status;
  if (resolved != RR_ARCH_GFX950) {
    return make_status(RR_STATUS_UNSUPPORTED_ARCHITECTURE, "this operator has kernels for gfx950 (MI355X) only");
  }
  const bool native = (kernel.family == RR_FAMILY_AUTO && kernel.implementation_id == 0) ||
                      (kernel.family == RR_FAMILY_OPTIMIZED && kernel.implementation_id == RR_IMPL_GFX950_NATIVE);
  const bool plain = naive != nullptr && kernel.family == RR_FAMILY_NAIVE && kernel.implementation_id == 0;
  if (!native && !plain) {
    return make_status(RR_STATUS_UNSUPPORTED_KERNEL_VARIANT,
                       "no kernel of this operator has that family and implementation id");
  }
  if (naive != nullptr) *naive = plain;
  return ok_status();
}

inline rr_status check_workspace(const rr_runtime_context* context, std::size_t bytes, const char* message) noexcept {
  if (bytes == 0) return ok_status();
  if (context->workspace == nullptr || context->workspace_bytes < bytes) {
    return make_status(RR_STATUS_INSUFFICIENT_WORKSPACE, message);
  }
  if (!is_aligned(context->workspace, kWorkspaceAlignment)) {
    return invalid_argument("the workspace of this operator must start on a 16-byte boundary");
  }
  return ok_status();
}

inline std::size_t round_up(std::size_t bytes) noexcept {
  return (bytes + kWorkspaceAlignment - 1) / kWorkspaceAlignment * kWorkspaceAlignment;
}

}  // namespace rr
