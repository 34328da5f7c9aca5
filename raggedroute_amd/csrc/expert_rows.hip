// Grouped products of the expert block for few rows an expert (decoding): the weights are
// read once from memory, straight into registers in matrix-operand order.
//
// A workgroup of W waves takes 128 columns of one expert (of each right operand) and its
// rows in blocks of 16 MR; the waves share the sum's length and add up through LDS in a
// fixed order. What bounds it is memory: a wave has 8 to 16 loads of 1 KB in flight and
// never passes weights through LDS.
//  - 16-bit weights lie [K, N]: a lane (i, g) loads 8 columns 8 i .. + 7 of the k rows 8 g .. + 7
//    of a 32-k step and turns that 8 x 8 block (32 byte permutes); register c then holds
//    eight k of column 8 i + c, the operand of one v_mfma_f32_16x16x32: the order of the
//    columns among the instruction's rows is free.
//  - int8 weights lie [N, K]: a lane loads 16 k of one column.
//  - The weights are the instruction's first operand, so that a lane ends with adjacent
//    columns of one row.
// Where an expert's columns make fewer workgroups than the card has CUs, the sum is also
// split over workgroups (`splits`), whose FP32 parts a second launch adds in order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "expert_gemm.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kCols = 128;
constexpr int kCus = 256;  // MI355X

template <typename T>
struct Step;  // one matrix instruction: k of it, accumulator, product
template <>
struct Step<bf16> {
  static constexpr int kK = 32;
  typedef f4 acc;
  typedef bf16 frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
};
template <>
struct Step<f16> {
  static constexpr int kK = 32;
  typedef f4 acc;
  typedef f16 frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
};
template <>
struct Step<int8_t> {
  static constexpr int kK = 64;
  typedef i4 acc;
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// 16 bytes at p (of any alignment), of which the first `count` elements exist
template <typename T>
__device__ __forceinline__ i4 load16(const T* p, int count) {
  constexpr int V = 16 / sizeof(T);
  typedef T chunk __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  chunk v = {};
  if (count >= V) {
    v = *reinterpret_cast<const chunk*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i < count) v[i] = p[i];
    }
  }
  return __builtin_bit_cast(i4, v);
}

// The `index`-th expert that has rows (-1: there are fewer), by one wave's lanes.
__device__ __forceinline__ int find_expert(const Product& p, int index, int* first, int* count) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  for (int e0 = 0; e0 < p.experts; e0 += 64) {
    const int e = e0 + lane;
    int from = 0, rows = 0;
    if (e < p.experts) {
      from = rr::dev::offset_at(p.offsets, e, p.rows);
      rows = rr::dev::offset_at(p.offsets, e + 1, p.rows) - from;
    }
    uint64_t some = __ballot(rows > 0);
    const int here = __popcll(some);
    if (index < here) {
      for (int i = 0; i < index; ++i) some &= some - 1;
      const int at = __builtin_ctzll(some);
      *first = __builtin_amdgcn_readlane(from, at);
      *count = __builtin_amdgcn_readlane(rows, at);
      return e0 + at;
    }
    index -= here;
  }
  return -1;
}

template <typename T, class Epi, int MR, int W>
__global__ __launch_bounds__(64 * W) void rr_expert_rows_kernel(Product prm, float* parts, int splits, int blocks) {
  using M = Step<T>;
  using Acc = typename M::acc;
  constexpr bool kKC = sizeof(T) == 1;  // k along the weights' rows
  constexpr int B = Epi::kDual ? 2 : 1;
  extern __shared__ __align__(16) char smem[];
  i4* lds = reinterpret_cast<i4*>(smem);  // [W / 2][B * 8 * MR][64]
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int block = static_cast<int>(blockIdx.x) % blocks;
  const int split = static_cast<int>(blockIdx.x) / blocks % splits;
  int first, count;
  const int e = find_expert(prm, static_cast<int>(blockIdx.x) / blocks / splits, &first, &count);
  if (e < 0) return;
  const int n0 = block * kCols;
  const int K = prm.K, N = prm.N;
  // this wave's steps
  const int steps = (K + M::kK - 1) / M::kK;
  const int share = split * W + wave, shares = splits * W;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * share / shares);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (share + 1) / shares);
  const T* weights[2] = {static_cast<const T*>(prm.b) + static_cast<std::size_t>(e) * K * N,
                         static_cast<const T*>(Epi::kDual ? prm.b_up : prm.b) + static_cast<std::size_t>(e) * K * N};

#pragma unroll 1
  for (int r0 = 0; r0 < count; r0 += 16 * MR) {
    Acc acc[B][8][MR] = {};
    const T* x[MR];
#pragma unroll
    for (int i = 0; i < MR; ++i) x[i] = static_cast<const T*>(prm.a) + static_cast<std::size_t>(first + min(r0 + 16 * i + li, count - 1)) * K;
    // One step: `whole` says that neither the columns nor the step are cut.
    auto step = [&](int s, auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      const int k = s * M::kK + g * (16 / static_cast<int>(sizeof(T)));  // the lane's first k
      i4 xv[MR];
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        // (rows past the last repeat it: their results are not stored)
        xv[i] = load16(x[i] + k, kWhole ? 16 : K - k);
      }
      if constexpr (kKC) {
        i4 w[B][8];
#pragma unroll
        for (int b = 0; b < B; ++b) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int n = n0 + 16 * j + li;
            w[b][j] = load16(weights[b] + static_cast<std::size_t>(kWhole ? n : min(n, N - 1)) * K + k, kWhole ? 16 : K - k);
          }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int i = 0; i < MR; ++i) acc[b][j][i] = M::mul(w[b][j], xv[i], acc[b][j][i]);
          }
        }
      } else {
        i4 w[B][8];
        const int n = n0 + 8 * li;
#pragma unroll
        for (int b = 0; b < B; ++b) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const T* row = weights[b] + static_cast<std::size_t>(s * M::kK + q) * N;  // uniform
            const std::size_t at = static_cast<std::size_t>(8 * g) * N + n;
            w[b][q] = load16(row + at, kWhole ? 8 : k + q < K ? N - n : 0);
          }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            i4 column;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              column[m] = static_cast<int>(__builtin_amdgcn_perm(static_cast<uint32_t>(w[b][2 * m + 1][c >> 1]),
                                                                 static_cast<uint32_t>(w[b][2 * m][c >> 1]),
                                                                 (c & 1) != 0 ? 0x07060302U : 0x05040100U));
            }
#pragma unroll
            for (int i = 0; i < MR; ++i) acc[b][c][i] = M::mul(column, xv[i], acc[b][c][i]);
          }
        }
      }
    };
    const bool cut = n0 + kCols > N;
    const int whole_end = cut ? s0 : min(s1, K / M::kK);
#pragma unroll 1
    for (int s = s0; s < whole_end; ++s) step(s, std::integral_constant<bool, true>{});
#pragma unroll 1
    for (int s = whole_end; s < s1; ++s) step(s, std::integral_constant<bool, false>{});

    // the waves' sums, halved round by round
#pragma unroll
    for (int half = W / 2; half >= 1; half /= 2) {
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int q = 0; q < B * 8 * MR; ++q) {
          lds[((wave - half) * B * 8 * MR + q) * 64 + lane] = __builtin_bit_cast(i4, acc[q / (8 * MR)][q / MR % 8][q % MR]);
        }
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int q = 0; q < B * 8 * MR; ++q) {
          acc[q / (8 * MR)][q / MR % 8][q % MR] += __builtin_bit_cast(Acc, lds[(wave * B * 8 * MR + q) * 64 + lane]);
        }
      }
      __syncthreads();
    }
    if (wave != 0) continue;
    // lane: row 16 i + li; columns 32 g + 8 r + 0..7 (KC: 16 j + 4 g + 0..3)
#pragma unroll
    for (int i = 0; i < MR; ++i) {
      const int r = r0 + 16 * i + li;
      if (r >= count) continue;
      const std::size_t row = static_cast<std::size_t>(first) + r;
      constexpr int V = kKC ? 4 : 8;
#pragma unroll
      for (int p = 0; p < 32 / V; ++p) {
        const int n = n0 + (kKC ? 16 * p + 4 * g : 32 * g + 8 * p);
        if (n >= N) continue;
        float v[B][V];
#pragma unroll
        for (int b = 0; b < B; ++b) {
#pragma unroll
          for (int q = 0; q < V; ++q) v[b][q] = static_cast<float>(kKC ? acc[b][p][i][q] : acc[b][q][i][p]);
        }
        if (parts != nullptr) {
#pragma unroll
          for (int b = 0; b < B; ++b) {
            Cols<float, V>::store(parts + (static_cast<std::size_t>(b * splits + split) * prm.rows + row) * N + n, v[b], N - n);
          }
        } else if constexpr (Epi::kDual) {
          Epi::template emit<V>(prm, e, row, n, N - n, v[0], v[1]);
        } else {
          Epi::template emit<V>(prm, e, row, n, N - n, v[0]);
        }
      }
    }
  }
}

// The splits' parts added in order, eight columns a thread.
template <class Epi>
__global__ __launch_bounds__(256) void rr_expert_rows_sum_kernel(Product prm, const float* parts, int splits) {
  constexpr int B = Epi::kDual ? 2 : 1;
  const int eights = (prm.N + 7) / 8;
  const int rows = rr::dev::offset_at(prm.offsets, prm.experts, prm.rows);
  const std::size_t total = static_cast<std::size_t>(rows) * eights;
  for (std::size_t t = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x; t < total;
       t += static_cast<std::size_t>(gridDim.x) * 256) {
    const std::size_t row = t / eights;
    const int n = static_cast<int>(t % eights) * 8;
    float v[B][8] = {};
    for (int s = 0; s < splits; ++s) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        float part[8];
        Cols<float, 8>::load(parts + (static_cast<std::size_t>(b * splits + s) * prm.rows + row) * prm.N + n, part, prm.N - n);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[b][q] += part[q];
      }
    }
    if constexpr (Epi::kDual) {
      Epi::template emit<8>(prm, 0, row, n, prm.N - n, v[0], v[1]);
    } else {
      Epi::template emit<8>(prm, 0, row, n, prm.N - n, v[0]);
    }
  }
}

template <typename T, class Epi, int MR, int W>
hipError_t launch(const Product& prm, float* parts, int splits, hipStream_t stream) {
  constexpr std::size_t lds = static_cast<std::size_t>(W / 2) * (Epi::kDual ? 2 : 1) * 8 * MR * 64 * sizeof(i4);
  if constexpr (lds > 64 * 1024) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(rr_expert_rows_kernel<T, Epi, MR, W>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (attr != hipSuccess) return attr;
  }
  const int blocks = (prm.N + kCols - 1) / kCols;
  const std::size_t grid = static_cast<std::size_t>(std::min(prm.experts, prm.rows)) * blocks * splits;
  rr_expert_rows_kernel<T, Epi, MR, W><<<dim3(static_cast<unsigned>(grid)), 64 * W, lds, stream>>>(prm, parts, splits, blocks);
  if (splits > 1) {
    if constexpr (sizeof(T) == 2) {
      const std::size_t threads = static_cast<std::size_t>(prm.rows) * ((prm.N + 7) / 8);
      const unsigned sums = static_cast<unsigned>(std::min<std::size_t>((threads + 255) / 256, 2048));
      rr_expert_rows_sum_kernel<Epi><<<dim3(sums), 256, 0, stream>>>(prm, parts, splits);
    }
  }
  return hipGetLastError();
}

template <typename T, class Epi, int MR>
hipError_t launch_waves(const Product& prm, float* parts, int splits, hipStream_t stream) {
  const int steps = prm.K / Step<T>::kK / splits;
  if (steps >= 48) return launch<T, Epi, MR, 8>(prm, parts, splits, stream);
  return steps >= 8 ? launch<T, Epi, MR, 4>(prm, parts, splits, stream) : launch<T, Epi, MR, 2>(prm, parts, splits, stream);
}

}  // namespace

bool expert_rows_ok(int rows, int experts) {
  const int active = std::min(rows, experts);
  return rows <= 16 || rows <= 24 * active;
}

int expert_rows_splits(int rows, int experts, int columns, int length) {
  if (!expert_rows_ok(rows, experts)) return 1;
  const int groups = std::min(rows, experts) * ((columns + kCols - 1) / kCols);
  const int most = std::min(length / 1024, 8);
  return std::max(1, std::min(most, kCus / groups));
}

template <typename T, class Epi>
hipError_t expert_rows(const Product& prm, float* parts, int splits, hipStream_t stream) {
  const int active = std::min(prm.rows, prm.experts);
  if (prm.rows <= 16 || prm.rows <= 5 * active) return launch_waves<T, Epi, 1>(prm, parts, splits, stream);
  return launch_waves<T, Epi, 2>(prm, parts, splits, stream);
}

template hipError_t expert_rows<bf16, EpiGate<bf16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<bf16, EpiStore<bf16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<f16, EpiGate<f16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<f16, EpiStore<f16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8<float>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8<bf16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8<f16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8Gate<float>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8Gate<bf16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8Gate<f16>>(const Product&, float*, int, hipStream_t);

}  // namespace rr::kern
