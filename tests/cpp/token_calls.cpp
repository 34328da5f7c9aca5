// The C++ calls of the token and 4-bit operators: every field, default and workspace query reaches the C
// entry, which stands here in the library's place.
#include <cstddef>
#include <cstdint>
#include <cstdio>

#include "raggedroute/raggedroute.h"

namespace {
int g_failures = 0;
void expect(bool condition, const char* what) {
  if (condition) return;
  std::printf("FAIL %s\n", what);
  ++g_failures;
}
const rr_runtime_context* g_context = nullptr;
rr_status answer(const rr_runtime_context* context) {
  expect(context != nullptr && context->workspace_bytes == 77 && context->architecture == RR_ARCH_GFX950, "the context");
  g_context = context;
  rr_status status{};
  status.code = RR_STATUS_INVALID_ARGUMENT;
  return status;
}
}  // namespace

// What an entry was given last, and its workspace query's answer.
#define RR_ENTRY(name, bytes)                                                             \
  namespace {                                                                             \
  rr_##name##_args g_##name;                                                              \
  }                                                                                       \
  extern "C" std::size_t rr_##name##_workspace_size(const rr_##name##_args* args) {       \
    g_##name = *args;                                                                     \
    return bytes;                                                                         \
  }                                                                                       \
  extern "C" rr_status rr_##name(const rr_##name##_args* args, const rr_runtime_context* context) { \
    g_##name = *args;                                                                     \
    return answer(context);                                                               \
  }
RR_ENTRY(sort_tokens, 11)
RR_ENTRY(sort_tokens_backward, 12)
RR_ENTRY(combine_tokens, 13)
RR_ENTRY(combine_tokens_backward, 14)
RR_ENTRY(topk_gate_backward, 15)
RR_ENTRY(quantize_rows_mxfp4, 16)
RR_ENTRY(mxfp4_grouped_gemm, 17)

namespace {

using namespace raggedroute;

std::int64_t g_memory[16];  // what pointers point to
RuntimeContext g_call;

template <class T>
void put(T*& field, int i) {
  field = reinterpret_cast<T*>(g_memory + i);
}
bool is(const void* field, int i) { return field == g_memory + i; }

template <class Args, class Call, class Size, class Check>
void forwarded(const char* name, Args args, Call call, Size size, std::size_t bytes, Check check) {
  args.kernel = {KernelFamily::kOptimized, 950};
  const Status status = call(args, g_call);
  expect(status.code == StatusCode::kInvalidArgument && g_context != nullptr, name);
  expect(check(), name);
  expect(size(args) == bytes && check(), name);
}
template <class C>
bool kernel_is(const C& c) {
  return c.kernel.family == RR_FAMILY_OPTIMIZED && c.kernel.implementation_id == 950;
}

}  // namespace

int main() {
  g_call.workspace_bytes = 77;
  g_call.architecture = DeviceArchitecture::kGfx950;
  {
    SortTokensArgs a;
    expect(a.top_k == 2 && a.dtype == ScalarType::kBf16 && a.x_dtype == ScalarType::kBf16, "sort_tokens' defaults");
    put(a.x, 0), put(a.expert_ids, 1), put(a.offsets, 2), put(a.route_pos, 3), put(a.sorted_route, 4), put(a.x_sorted, 5);
    a.tokens = 6, a.experts = 7, a.top_k = 8, a.hidden = 9, a.dtype = ScalarType::kFp16, a.x_dtype = ScalarType::kFp32;
    forwarded("sort_tokens", a, sort_tokens, get_sort_tokens_workspace_size, 11, [] {
      const auto& c = g_sort_tokens;
      return is(c.x, 0) && is(c.expert_ids, 1) && is(c.offsets, 2) && is(c.route_pos, 3) && is(c.sorted_route, 4) && is(c.x_sorted, 5) &&
             c.tokens == 6 && c.experts == 7 && c.top_k == 8 && c.hidden == 9 && c.dtype == RR_DTYPE_FP16 && c.x_dtype == RR_DTYPE_FP32 &&
             kernel_is(c);
    });
  }
  {
    SortTokensBackwardArgs a;
    expect(a.top_k == 2 && a.dtype == ScalarType::kBf16 && a.x_dtype == ScalarType::kBf16, "sort_tokens_backward's defaults");
    put(a.dx_sorted, 0), put(a.route_pos, 1), put(a.dx, 2);
    a.tokens = 3, a.top_k = 4, a.hidden = 5, a.dtype = ScalarType::kFp16, a.x_dtype = ScalarType::kFp32;
    forwarded("sort_tokens_backward", a, sort_tokens_backward, get_sort_tokens_backward_workspace_size, 12, [] {
      const auto& c = g_sort_tokens_backward;
      return is(c.dx_sorted, 0) && is(c.route_pos, 1) && is(c.dx, 2) && c.tokens == 3 && c.top_k == 4 && c.hidden == 5 &&
             c.dtype == RR_DTYPE_FP16 && c.x_dtype == RR_DTYPE_FP32 && kernel_is(c);
    });
  }
  {
    CombineTokensArgs a;
    expect(a.top_k == 2 && a.dtype == ScalarType::kBf16 && a.y_dtype == ScalarType::kBf16, "combine_tokens' defaults");
    put(a.y_sorted, 0), put(a.route_pos, 1), put(a.route_weights, 2), put(a.y, 3);
    a.tokens = 4, a.top_k = 5, a.hidden = 6, a.dtype = ScalarType::kFp16, a.y_dtype = ScalarType::kFp32;
    forwarded("combine_tokens", a, combine_tokens, get_combine_tokens_workspace_size, 13, [] {
      const auto& c = g_combine_tokens;
      return is(c.y_sorted, 0) && is(c.route_pos, 1) && is(c.route_weights, 2) && is(c.y, 3) && c.tokens == 4 && c.top_k == 5 &&
             c.hidden == 6 && c.dtype == RR_DTYPE_FP16 && c.y_dtype == RR_DTYPE_FP32 && kernel_is(c);
    });
  }
  {
    CombineTokensBackwardArgs a;
    expect(a.top_k == 2 && a.dtype == ScalarType::kBf16 && a.y_dtype == ScalarType::kBf16, "combine_tokens_backward's defaults");
    put(a.dy, 0), put(a.y_sorted, 1), put(a.route_pos, 2), put(a.route_weights, 3), put(a.dy_sorted, 4), put(a.droute_weights, 5);
    a.tokens = 6, a.top_k = 7, a.hidden = 8, a.dtype = ScalarType::kFp16, a.y_dtype = ScalarType::kFp32;
    forwarded("combine_tokens_backward", a, combine_tokens_backward, get_combine_tokens_backward_workspace_size, 14, [] {
      const auto& c = g_combine_tokens_backward;
      return is(c.dy, 0) && is(c.y_sorted, 1) && is(c.route_pos, 2) && is(c.route_weights, 3) && is(c.dy_sorted, 4) &&
             is(c.droute_weights, 5) && c.tokens == 6 && c.top_k == 7 && c.hidden == 8 && c.dtype == RR_DTYPE_FP16 &&
             c.y_dtype == RR_DTYPE_FP32 && kernel_is(c);
    });
  }
  {
    TopKGateBackwardArgs a;
    expect(a.top_k == 2, "topk_gate_backward's defaults");
    put(a.expert_ids, 0), put(a.weights, 1), put(a.dweights, 2), put(a.dlogits, 3);
    a.tokens = 4, a.experts = 5, a.top_k = 6;
    forwarded("topk_gate_backward", a, topk_gate_backward, get_topk_gate_backward_workspace_size, 15, [] {
      const auto& c = g_topk_gate_backward;
      return is(c.expert_ids, 0) && is(c.weights, 1) && is(c.dweights, 2) && is(c.dlogits, 3) && c.tokens == 4 && c.experts == 5 &&
             c.top_k == 6 && kernel_is(c);
    });
  }
  {
    QuantizeRowsMxfp4Args a;
    expect(a.top_k == 2 && a.dtype == ScalarType::kBf16, "quantize_rows_mxfp4's defaults");
    put(a.x, 0), put(a.sorted_route, 1), put(a.q, 2), put(a.scale, 3);
    a.rows = 4, a.hidden = 5, a.tokens = 6, a.top_k = 7, a.dtype = ScalarType::kFp32;
    forwarded("quantize_rows_mxfp4", a, quantize_rows_mxfp4, get_quantize_rows_mxfp4_workspace_size, 16, [] {
      const auto& c = g_quantize_rows_mxfp4;
      return is(c.x, 0) && is(c.sorted_route, 1) && is(c.q, 2) && is(c.scale, 3) && c.rows == 4 && c.hidden == 5 && c.tokens == 6 &&
             c.top_k == 7 && c.dtype == RR_DTYPE_FP32 && kernel_is(c);
    });
  }
  {
    Mxfp4GroupedGemmArgs a;
    expect(a.activation == Activation::kSilu && a.dtype == ScalarType::kBf16, "mxfp4_grouped_gemm's defaults");
    put(a.q, 0), put(a.q_scale, 1), put(a.w, 2), put(a.w_scale, 3), put(a.w_up, 4), put(a.w_up_scale, 5), put(a.offsets, 6), put(a.y, 7);
    a.rows = 8, a.experts = 9, a.hidden = 10, a.output = 11, a.activation = Activation::kGeluTanh, a.dtype = ScalarType::kFp32;
    forwarded("mxfp4_grouped_gemm", a, mxfp4_grouped_gemm, get_mxfp4_grouped_gemm_workspace_size, 17, [] {
      const auto& c = g_mxfp4_grouped_gemm;
      return is(c.q, 0) && is(c.q_scale, 1) && is(c.w, 2) && is(c.w_scale, 3) && is(c.w_up, 4) && is(c.w_up_scale, 5) &&
             is(c.offsets, 6) && is(c.y, 7) && c.rows == 8 && c.experts == 9 && c.hidden == 10 && c.output == 11 &&
             c.activation == RR_ACT_GELU_TANH && c.dtype == RR_DTYPE_FP32 && kernel_is(c);
    });
  }
  if (g_failures == 0) std::printf("token calls OK\n");
  return g_failures;
}
