// 4-bit products for few rows an expert (decoding): the weights are read once from memory,
// straight into registers in matrix-operand order.
//
// A workgroup of W waves takes 64 columns (of each right operand) of one expert and 16 of its
// rows; the waves share the blocks of a row and add up through LDS in a fixed order. A step is
// a slice of 256 elements: 128 bytes of every row and eight scales. Lane group g multiplies
// blocks g and 4 + g of it (the two loads of a row's 128 bytes follow each other); its scales
// are the bytes g of the row's two words. What bounds it is memory.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "mxfp4.h"
#include "mxfp4_rows.h"
#include "row_groups.h"
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

typedef int i2 __attribute__((ext_vector_type(2)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kBufferFlags = 0x00027000;  // raw 32-bit buffer
constexpr uint32_t kPast = 0x80000000U;   // an offset past every record count
constexpr int kSliceBytes = 128;  // of every row

__device__ __forceinline__ f4 multiply(i4 a, i4 b, f4 c, int a_scale, int b_scale) {
  typedef int i8 __attribute__((ext_vector_type(8)));
  const i8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  constexpr int kE2M1 = 4;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, kE2M1, kE2M1, 0, a_scale, 0, b_scale);
}

// W waves, F fragments of 16 columns of each right operand, D slices on their way
template <class Epi, int W, int F, int D>
__global__ __launch_bounds__(64 * W, 2) void rr_mxfp4_rows_kernel(Product prm, int blocks) {
  constexpr int B = Epi::kDual ? 2 : 1;
  constexpr int kCols = 16 * F;
  __shared__ __align__(16) f4 s_sums[W > 1 ? W / 2 : 1][B * F][64];
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int block = static_cast<int>(blockIdx.x % static_cast<unsigned>(blocks));
  int first, count;
  const int e = find_group(prm, static_cast<int>(blockIdx.x / static_cast<unsigned>(blocks)), &first, &count);
  if (e < 0) return;
  const int n0 = block * kCols;
  const int N = prm.N, row_bytes = prm.lda;
  // this wave's slices
  const int slices = (prm.K + 7) / 8;
  const int s0 = static_cast<int>(static_cast<int64_t>(slices) * wave / W);
  const int s1 = static_cast<int>(static_cast<int64_t>(slices) * (wave + 1) / W);

  const int columns = min(N - n0, kCols);
  const int64_t channel = static_cast<int64_t>(e) * N + n0;
  const int64_t x_slice = static_cast<int64_t>(prm.rows) * 8, w_slice = static_cast<int64_t>(prm.experts) * N * 8;
  auto buffer_of = [](const void* base, int64_t at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base) + at), 0, bytes, kBufferFlags);
  };
  // rows past the last and columns past N repeat the last one: their results are not stored
  const uint32_t x_lane = static_cast<uint32_t>(min(li, count - 1)) * row_bytes + 16 * g;
  const uint32_t xs_lane = static_cast<uint32_t>(min(li, count - 1)) * 8;
  uint32_t w_lane[F], ws_lane[F];
#pragma unroll
  for (int j = 0; j < F; ++j) {
    const uint32_t c = min(16 * j + li, columns - 1);
    w_lane[j] = c * row_bytes + 16 * g;
    ws_lane[j] = c * 8;
  }
  // What a slice multiplies. Of a slice past the wave's last nothing is read (zeros).
  struct Slice {
    i4 x[2], w[B][F][2];
    i2 x_scale, w_scale[B][F];
  };
  auto load = [&](Slice& o, int s) {
    const bool on = s < s1;
    const int left = prm.K - 8 * s;  // blocks of a row from the slice on
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const auto w = buffer_of(b == 0 ? prm.b : prm.b_up, channel * row_bytes, on ? columns * row_bytes : 0);
#pragma unroll
      for (int j = 0; j < F; ++j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          o.w[b][j][h] = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(w, w_lane[j] + 64 * h + s * kSliceBytes, 0, 0));
        }
      }
    }
    const auto x = buffer_of(prm.a, static_cast<int64_t>(first) * row_bytes, on ? count * row_bytes : 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // (blocks past the last are zeros: what the weights have there, the next channel's, does not count)
      const uint32_t at = 4 * h + g < left ? x_lane + 64 * h + s * kSliceBytes : kPast;
      o.x[h] = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(x, at, 0, 0));
    }
    const auto xs = buffer_of(prm.a2, static_cast<int64_t>(first) * 8 + s * x_slice, on ? count * 8 : 0);
    o.x_scale = __builtin_bit_cast(i2, __builtin_amdgcn_raw_buffer_load_b64(xs, xs_lane, 0, 0));
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const auto ws = buffer_of(b == 0 ? prm.in : prm.in_up, channel * 8 + s * w_slice, on ? columns * 8 : 0);
#pragma unroll
      for (int j = 0; j < F; ++j) o.w_scale[b][j] = __builtin_bit_cast(i2, __builtin_amdgcn_raw_buffer_load_b64(ws, ws_lane[j], 0, 0));
    }
  };
  f4 acc[B][F] = {};
  auto multiply_slice = [&](const Slice& o, int s) {
    const int left = prm.K - 8 * s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool is = 4 * h + g < left;  // (scales past the last block are not looked at)
      const int x_scale = is ? (o.x_scale[h] >> (8 * g)) & 255 : 0;
#pragma unroll
      for (int b = 0; b < B; ++b) {
#pragma unroll
        for (int j = 0; j < F; ++j) {
          acc[b][j] = multiply(o.w[b][j][h], o.x[h], acc[b][j], is ? (o.w_scale[b][j][h] >> (8 * g)) & 255 : 0, x_scale);
        }
      }
    }
  };
  Slice set[D];
#pragma unroll
  for (int d = 0; d < D; ++d) load(set[d], s0 + d);
#pragma unroll 1
  for (int s = s0; s < s1; s += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      __builtin_amdgcn_sched_barrier(0);  // (loads hoisted over the products would need registers of their own)
      multiply_slice(set[d], s + d);
      __builtin_amdgcn_sched_barrier(0);
      load(set[d], s + d + D);
    }
  }

  // the waves' sums, halved round by round
#pragma unroll
  for (int half = W / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int q = 0; q < B * F; ++q) s_sums[wave - half][q][lane] = acc[q / F][q % F];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int q = 0; q < B * F; ++q) acc[q / F][q % F] += s_sums[wave][q][lane];
    }
    __syncthreads();
  }
  if (wave != 0 || li >= count) return;
  // lane: row li, columns 16 j + 4 g + 0..3
  const std::size_t row = static_cast<std::size_t>(first) + li;
#pragma unroll
  for (int j = 0; j < F; ++j) {
    const int n = n0 + 16 * j + 4 * g;
    if (n >= N) continue;
    float v[B][4];
#pragma unroll
    for (int b = 0; b < B; ++b) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[b][q] = acc[b][j][q];
    }
    if constexpr (Epi::kDual) {
      Epi::template emit<4>(prm, e, row, n, N - n, v[0], v[1]);
    } else {
      Epi::template emit<4>(prm, e, row, n, N - n, v[0]);
    }
  }
}

template <class Epi, int W, int F, int D>
hipError_t launch(const Product& prm, hipStream_t stream) {
  const int blocks = (prm.N + 16 * F - 1) / (16 * F);
  const std::size_t grid = most_groups(prm.rows, prm.experts) * blocks;
  rr_mxfp4_rows_kernel<Epi, W, F, D><<<dim3(static_cast<unsigned>(grid)), 64 * W, 0, stream>>>(prm, blocks);
  return hipGetLastError();
}

}  // namespace

bool mxfp4_rows_ok(int rows, int experts) { return rows <= 16 || rows <= 3 * std::min(rows, experts); }

template <class Epi>
hipError_t mxfp4_rows(const Product& prm, hipStream_t stream) {
  return launch<Epi, 4, 4, 1>(prm, stream);
}

template hipError_t mxfp4_rows<EpiStore<float>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiStore<bf16>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiStore<f16>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiGate<float>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiGate<bf16>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiGate<f16>>(const Product&, hipStream_t);

}  // namespace rr::kern
