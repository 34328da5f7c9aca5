// Rows to blocks of 32 E2M1 elements with an E8M0 scale each.
//
// A lane takes eight elements, four lanes a block: the largest magnitude is found on the bits
// (a NaN is above an infinity, an infinity above the rest), the scale's exponent is that of the
// magnitude less 2, and the conversion divides by the scale, rounds to even and cuts at 6.
// 16 lanes put four scales together to a word. What bounds it is memory: 16384 rows of 4096 BF16
// numbers gathered from 8192 tokens 28 us, 134 MB read (half of it again, from the caches) and 36
// written.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "block_device.h"
#include "mxfp4.h"
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

constexpr int kThreads = 256;
constexpr int kPiece = 8;  // elements of a lane

// DPP lane moves inside rows of 16 lanes
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E;    // lanes 1 0 3 2, lanes 2 3 0 1 of every four
constexpr int kTurn4 = 0x124, kTurn8 = 0x128;  // rows turned by four and eight lanes

// G threads a row, U pieces of a thread on their way together. WHOLE: rows are made of whole
// pieces.
template <typename T, int G, int U, bool WHOLE>
__global__ __launch_bounds__(kThreads) void rr_quantize_mxfp4_kernel(MxQuantizeParams p) {
  typedef T vec __attribute__((ext_vector_type(kPiece), aligned(sizeof(T))));
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (G - 1);
  const int blocks = mx_blocks(p.hidden);
  const int pieces = 4 * blocks, padded = 32 * mx_slices(p.hidden);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + tid / G; r < p.rows;
       r += static_cast<int64_t>(gridDim.x) * (kThreads / G)) {
    std::size_t source = r;
    if (p.sorted_route != nullptr) {
      const int route = p.sorted_route[r];
      if (route < 0 || route >= static_cast<int64_t>(p.tokens) * p.top_k) continue;
      source = static_cast<unsigned>(route) / static_cast<unsigned>(p.top_k);
    }
    const T* x = static_cast<const T*>(p.x) + source * p.hidden;
    for (int c0 = lane; c0 < padded; c0 += G * U) {
      vec piece[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int c = c0 + k * G;
        const int left = p.hidden - c * kPiece;
        if (WHOLE ? left > 0 : left >= kPiece) {
          piece[k] = *reinterpret_cast<const vec*>(x + c * kPiece);
        } else {
#pragma unroll
          for (int i = 0; i < kPiece; ++i) piece[k][i] = !WHOLE && i < left ? x[c * kPiece + i] : static_cast<T>(0.0F);
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int c = c0 + k * G;
        if (c >= padded) continue;  // (by 32 lanes: the moves stay inside 16)
        float v[kPiece];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
          v[i] = static_cast<float>(piece[k][i]);
          m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFU);
        }
        m = max(m, rr::dev::dpp_move<kSwap1>(m));
        m = max(m, rr::dev::dpp_move<kSwap2>(m));
        const bool finite = m < 0x7F800000U;
        // 2^(byte - 127), the least of them subnormal
        const uint32_t byte = m < (3U << 23) ? 0U : (m >> 23) - 2U;
        const float scale = __uint_as_float(byte == 0 ? 1U << 22 : byte << 23);
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
        if (c < pieces) reinterpret_cast<uint32_t*>(p.q)[static_cast<std::size_t>(r) * pieces + c] = finite ? q : 0U;
        uint32_t scales = (c < pieces ? (finite ? byte : 255U) : 0U) << (8 * ((c >> 2) & 3));
        scales |= rr::dev::dpp_move<kTurn4>(scales);
        scales |= rr::dev::dpp_move<kTurn8>(scales);
        if ((c & 15) == 0) {
          reinterpret_cast<uint32_t*>(p.scale)[(static_cast<std::size_t>(c >> 5) * p.rows + r) * 2 + ((c >> 4) & 1)] = scales;
        }
      }
    }
  }
}

template <typename T>
hipError_t quantize(const MxQuantizeParams& p, hipStream_t stream) {
  auto run = [&](auto g, auto u) {
    constexpr int G = decltype(g)::value, U = decltype(u)::value;
    const int64_t groups = (static_cast<int64_t>(p.rows) + kThreads / G - 1) / (kThreads / G);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(groups, 16384));
    if (p.hidden % kPiece == 0) {
      rr_quantize_mxfp4_kernel<T, G, U, true><<<grid, kThreads, 0, stream>>>(p);
    } else {
      rr_quantize_mxfp4_kernel<T, G, U, false><<<grid, kThreads, 0, stream>>>(p);
    }
    return hipGetLastError();
  };
  const int slices = mx_slices(p.hidden);  // of 32 pieces each
  if (slices == 1) return run(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  if (slices == 2) return run(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  // (a wave a row: 16384 rows of 4096, BF16, 29 us with two pieces a thread on their way, 32 with
  // 256 threads; few rows take all the threads that a workgroup has)
  if (p.rows < 1024) return run(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  return run(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
}

}  // namespace

hipError_t quantize_rows_mxfp4(const MxQuantizeParams& p, hipStream_t stream) {
  if (p.dtype == RR_DTYPE_FP32) return quantize<float>(p, stream);
  if (p.dtype == RR_DTYPE_BF16) return quantize<bf16>(p, stream);
  return quantize<f16>(p, stream);
}

}  // namespace rr::kern
