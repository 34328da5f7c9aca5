// raggedroute/block.h - the expert block around the routing chain: gated
// feed-forward with its gradients, the norms before and after it, 8-bit integer and
// 4-bit floating-point products, tokens to their experts and back with gradients. New entries (no reference counterpart); inline forwarders to
// raggedroute_capi.h, which states formulas, shapes and optional buffers.
#pragma once

#include <cstddef>
#include <cstdint>

#include "raggedroute/detail/capi_bridge.h"
#include "raggedroute/runtime.h"
#include "raggedroute/status.h"
#include "raggedroute/types.h"

namespace raggedroute {

enum class Activation {
  kSilu = 0,
  kGeluTanh,
};

struct GatedFfnArgs {
  const void* x = nullptr;
  const void* w_gate = nullptr;
  const void* w_up = nullptr;
  const void* w_down = nullptr;
  const std::int32_t* offsets = nullptr;
  void* gate = nullptr;
  void* up = nullptr;
  void* act = nullptr;
  void* y = nullptr;
  int rows = 0;
  int experts = 0;
  int hidden = 0;
  int inner = 0;
  int output = 0;
  Activation activation = Activation::kSilu;
  ScalarType dtype = ScalarType::kBf16;
  ScalarType y_dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct GatedFfnBackwardArgs {
  const void* x = nullptr;
  const void* w_gate = nullptr;
  const void* w_up = nullptr;
  const void* w_down = nullptr;
  const std::int32_t* offsets = nullptr;
  const void* gate = nullptr;
  const void* up = nullptr;
  const void* act = nullptr;
  const void* dy = nullptr;
  void* dx = nullptr;
  void* dw_gate = nullptr;
  void* dw_up = nullptr;
  void* dw_down = nullptr;
  int rows = 0;
  int experts = 0;
  int hidden = 0;
  int inner = 0;
  int output = 0;
  Activation activation = Activation::kSilu;
  ScalarType dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct BlockNormArgs {
  const void* x = nullptr;
  const void* block = nullptr;
  const void* post_weight = nullptr;
  const void* gate = nullptr;
  const void* pre_weight = nullptr;
  void* h = nullptr;
  void* n = nullptr;
  float residual_scale = 1.0F;
  float eps = 1e-6F;
  int gate_tokens = 0;
  int tokens = 0;
  int hidden = 0;
  ScalarType dtype = ScalarType::kBf16;
  ScalarType block_dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct BlockNormBackwardArgs {
  const void* h = nullptr;
  const void* block = nullptr;
  const void* post_weight = nullptr;
  const void* gate = nullptr;
  const void* pre_weight = nullptr;
  const void* dh = nullptr;
  const void* dn = nullptr;
  void* dx = nullptr;
  void* dblock = nullptr;
  void* dgate = nullptr;
  void* dpre_weight = nullptr;
  void* dpost_weight = nullptr;
  float residual_scale = 1.0F;
  float eps = 1e-6F;
  int gate_tokens = 0;
  int tokens = 0;
  int hidden = 0;
  ScalarType dtype = ScalarType::kBf16;
  ScalarType block_dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct QuantizeRowsArgs {
  const void* x = nullptr;
  std::int8_t* q = nullptr;
  float* scale = nullptr;
  int rows = 0;
  int hidden = 0;
  ScalarType dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct Int8GroupedGemmArgs {
  const std::int8_t* q = nullptr;
  const float* q_scale = nullptr;
  const std::int8_t* w = nullptr;
  const float* w_scale = nullptr;
  const std::int8_t* w_up = nullptr;
  const float* w_up_scale = nullptr;
  const std::int32_t* offsets = nullptr;
  void* y = nullptr;
  int rows = 0;
  int experts = 0;
  int hidden = 0;
  int output = 0;
  Activation activation = Activation::kSilu;
  ScalarType dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct SortTokensArgs {
  const void* x = nullptr;
  const std::int32_t* expert_ids = nullptr;
  std::int32_t* offsets = nullptr;
  std::int32_t* route_pos = nullptr;
  std::int32_t* sorted_route = nullptr;
  void* x_sorted = nullptr;
  int tokens = 0;
  int experts = 0;
  int top_k = 2;
  int hidden = 0;
  ScalarType dtype = ScalarType::kBf16;
  ScalarType x_dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct SortTokensBackwardArgs {
  const void* dx_sorted = nullptr;
  const std::int32_t* route_pos = nullptr;
  void* dx = nullptr;
  int tokens = 0;
  int top_k = 2;
  int hidden = 0;
  ScalarType dtype = ScalarType::kBf16;
  ScalarType x_dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct CombineTokensArgs {
  const void* y_sorted = nullptr;
  const std::int32_t* route_pos = nullptr;
  const float* route_weights = nullptr;
  void* y = nullptr;
  int tokens = 0;
  int top_k = 2;
  int hidden = 0;
  ScalarType dtype = ScalarType::kBf16;
  ScalarType y_dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct CombineTokensBackwardArgs {
  const void* dy = nullptr;
  const void* y_sorted = nullptr;
  const std::int32_t* route_pos = nullptr;
  const float* route_weights = nullptr;
  void* dy_sorted = nullptr;
  float* droute_weights = nullptr;
  int tokens = 0;
  int top_k = 2;
  int hidden = 0;
  ScalarType dtype = ScalarType::kBf16;
  ScalarType y_dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct TopKGateBackwardArgs {
  const std::int32_t* expert_ids = nullptr;
  const float* weights = nullptr;
  const float* dweights = nullptr;
  float* dlogits = nullptr;
  int tokens = 0;
  int experts = 0;
  int top_k = 2;
  KernelSelection kernel;
};

struct QuantizeRowsMxfp4Args {
  const void* x = nullptr;
  const std::int32_t* sorted_route = nullptr;
  std::uint8_t* q = nullptr;
  std::uint8_t* scale = nullptr;
  int rows = 0;
  int hidden = 0;
  int tokens = 0;
  int top_k = 2;
  ScalarType dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

struct Mxfp4GroupedGemmArgs {
  const std::uint8_t* q = nullptr;
  const std::uint8_t* q_scale = nullptr;
  const std::uint8_t* w = nullptr;
  const std::uint8_t* w_scale = nullptr;
  const std::uint8_t* w_up = nullptr;
  const std::uint8_t* w_up_scale = nullptr;
  const std::int32_t* offsets = nullptr;
  void* y = nullptr;
  int rows = 0;
  int experts = 0;
  int hidden = 0;
  int output = 0;
  Activation activation = Activation::kSilu;
  ScalarType dtype = ScalarType::kBf16;
  KernelSelection kernel;
};

namespace detail {

inline rr_gated_ffn_args to_c(const GatedFfnArgs& a) noexcept {
  return {a.x, a.w_gate, a.w_up, a.w_down, a.offsets, a.gate, a.up, a.act, a.y, a.rows,
          a.experts, a.hidden, a.inner, a.output, static_cast<int32_t>(a.activation),
          static_cast<int32_t>(a.dtype), static_cast<int32_t>(a.y_dtype), to_c(a.kernel)};
}
inline rr_gated_ffn_backward_args to_c(const GatedFfnBackwardArgs& a) noexcept {
  return {a.x, a.w_gate, a.w_up, a.w_down, a.offsets, a.gate, a.up, a.act, a.dy, a.dx, a.dw_gate,
          a.dw_up, a.dw_down, a.rows, a.experts, a.hidden, a.inner, a.output,
          static_cast<int32_t>(a.activation), static_cast<int32_t>(a.dtype), to_c(a.kernel)};
}
inline rr_block_norm_args to_c(const BlockNormArgs& a) noexcept {
  return {a.x, a.block, a.post_weight, a.gate, a.pre_weight, a.h, a.n, a.residual_scale, a.eps,
          a.gate_tokens, a.tokens, a.hidden, static_cast<int32_t>(a.dtype),
          static_cast<int32_t>(a.block_dtype), to_c(a.kernel)};
}
inline rr_block_norm_backward_args to_c(const BlockNormBackwardArgs& a) noexcept {
  return {a.h, a.block, a.post_weight, a.gate, a.pre_weight, a.dh, a.dn, a.dx, a.dblock, a.dgate,
          a.dpre_weight, a.dpost_weight, a.residual_scale, a.eps, a.gate_tokens, a.tokens,
          a.hidden, static_cast<int32_t>(a.dtype), static_cast<int32_t>(a.block_dtype),
          to_c(a.kernel)};
}
inline rr_quantize_rows_args to_c(const QuantizeRowsArgs& a) noexcept {
  return {a.x, a.q, a.scale, a.rows, a.hidden, static_cast<int32_t>(a.dtype), to_c(a.kernel)};
}
inline rr_int8_grouped_gemm_args to_c(const Int8GroupedGemmArgs& a) noexcept {
  return {a.q, a.q_scale, a.w, a.w_scale, a.w_up, a.w_up_scale, a.offsets, a.y, a.rows,
          a.experts, a.hidden, a.output, static_cast<int32_t>(a.activation),
          static_cast<int32_t>(a.dtype), to_c(a.kernel)};
}
inline rr_sort_tokens_args to_c(const SortTokensArgs& a) noexcept {
  return {a.x, a.expert_ids, a.offsets, a.route_pos, a.sorted_route, a.x_sorted, a.tokens,
          a.experts, a.top_k, a.hidden, static_cast<int32_t>(a.dtype),
          static_cast<int32_t>(a.x_dtype), to_c(a.kernel)};
}
inline rr_sort_tokens_backward_args to_c(const SortTokensBackwardArgs& a) noexcept {
  return {a.dx_sorted, a.route_pos, a.dx, a.tokens, a.top_k, a.hidden,
          static_cast<int32_t>(a.dtype), static_cast<int32_t>(a.x_dtype), to_c(a.kernel)};
}
inline rr_combine_tokens_args to_c(const CombineTokensArgs& a) noexcept {
  return {a.y_sorted, a.route_pos, a.route_weights, a.y, a.tokens, a.top_k, a.hidden,
          static_cast<int32_t>(a.dtype), static_cast<int32_t>(a.y_dtype), to_c(a.kernel)};
}
inline rr_combine_tokens_backward_args to_c(const CombineTokensBackwardArgs& a) noexcept {
  return {a.dy, a.y_sorted, a.route_pos, a.route_weights, a.dy_sorted, a.droute_weights, a.tokens,
          a.top_k, a.hidden, static_cast<int32_t>(a.dtype), static_cast<int32_t>(a.y_dtype),
          to_c(a.kernel)};
}
inline rr_topk_gate_backward_args to_c(const TopKGateBackwardArgs& a) noexcept {
  return {a.expert_ids, a.weights, a.dweights, a.dlogits, a.tokens, a.experts, a.top_k,
          to_c(a.kernel)};
}
inline rr_quantize_rows_mxfp4_args to_c(const QuantizeRowsMxfp4Args& a) noexcept {
  return {a.x, a.sorted_route, a.q, a.scale, a.rows, a.hidden, a.tokens, a.top_k,
          static_cast<int32_t>(a.dtype), to_c(a.kernel)};
}
inline rr_mxfp4_grouped_gemm_args to_c(const Mxfp4GroupedGemmArgs& a) noexcept {
  return {a.q, a.q_scale, a.w, a.w_scale, a.w_up, a.w_up_scale, a.offsets, a.y, a.rows, a.experts,
          a.hidden, a.output, static_cast<int32_t>(a.activation), static_cast<int32_t>(a.dtype),
          to_c(a.kernel)};
}

}  // namespace detail

inline std::size_t get_gated_ffn_workspace_size(const GatedFfnArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_gated_ffn_workspace_size(&c);
}
inline std::size_t get_gated_ffn_backward_workspace_size(const GatedFfnBackwardArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_gated_ffn_backward_workspace_size(&c);
}
inline std::size_t get_block_norm_workspace_size(const BlockNormArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_block_norm_workspace_size(&c);
}
inline std::size_t get_block_norm_backward_workspace_size(const BlockNormBackwardArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_block_norm_backward_workspace_size(&c);
}
inline std::size_t get_quantize_rows_workspace_size(const QuantizeRowsArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_quantize_rows_workspace_size(&c);
}
inline std::size_t get_int8_grouped_gemm_workspace_size(const Int8GroupedGemmArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_int8_grouped_gemm_workspace_size(&c);
}

inline std::size_t get_sort_tokens_workspace_size(const SortTokensArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_sort_tokens_workspace_size(&c);
}
inline std::size_t get_sort_tokens_backward_workspace_size(const SortTokensBackwardArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_sort_tokens_backward_workspace_size(&c);
}
inline std::size_t get_combine_tokens_workspace_size(const CombineTokensArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_combine_tokens_workspace_size(&c);
}
inline std::size_t get_combine_tokens_backward_workspace_size(const CombineTokensBackwardArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_combine_tokens_backward_workspace_size(&c);
}
inline std::size_t get_topk_gate_backward_workspace_size(const TopKGateBackwardArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_topk_gate_backward_workspace_size(&c);
}
inline std::size_t get_quantize_rows_mxfp4_workspace_size(const QuantizeRowsMxfp4Args& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_quantize_rows_mxfp4_workspace_size(&c);
}
inline std::size_t get_mxfp4_grouped_gemm_workspace_size(const Mxfp4GroupedGemmArgs& args) noexcept {
  const auto c = detail::to_c(args);
  return rr_mxfp4_grouped_gemm_workspace_size(&c);
}

inline Status gated_ffn(const GatedFfnArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_gated_ffn(&a, &c));
}
inline Status gated_ffn_backward(const GatedFfnBackwardArgs& args,
                                 const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_gated_ffn_backward(&a, &c));
}
inline Status block_norm(const BlockNormArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_block_norm(&a, &c));
}
inline Status block_norm_backward(const BlockNormBackwardArgs& args,
                                  const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_block_norm_backward(&a, &c));
}
inline Status quantize_rows(const QuantizeRowsArgs& args,
                            const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_quantize_rows(&a, &c));
}
inline Status int8_grouped_gemm(const Int8GroupedGemmArgs& args,
                                const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_int8_grouped_gemm(&a, &c));
}
inline Status sort_tokens(const SortTokensArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_sort_tokens(&a, &c));
}
inline Status sort_tokens_backward(const SortTokensBackwardArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_sort_tokens_backward(&a, &c));
}
inline Status combine_tokens(const CombineTokensArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_combine_tokens(&a, &c));
}
inline Status combine_tokens_backward(const CombineTokensBackwardArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_combine_tokens_backward(&a, &c));
}
inline Status topk_gate_backward(const TopKGateBackwardArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_topk_gate_backward(&a, &c));
}
inline Status quantize_rows_mxfp4(const QuantizeRowsMxfp4Args& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_quantize_rows_mxfp4(&a, &c));
}
inline Status mxfp4_grouped_gemm(const Mxfp4GroupedGemmArgs& args, const RuntimeContext& context) noexcept {
  const auto a = detail::to_c(args);
  const auto c = detail::to_c(context);
  return detail::from_c(rr_mxfp4_grouped_gemm(&a, &c));
}

}  // namespace raggedroute
