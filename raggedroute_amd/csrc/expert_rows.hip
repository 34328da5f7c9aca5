// Grouped products of the expert block for few rows an expert (decoding): the weights are
// read once from memory, straight into registers in matrix-operand order.
//
// A workgroup of W waves takes 128 columns (int8: 64) of one expert (of each right operand) and 16 of
// its rows; the waves share the sum's length and add up through LDS in a fixed order. An
// expert's groups of 16 rows are side by side, so that rows which crowd on one expert
// share the card (one workgroup after the other: 640 rows on one of 128 experts, K = 2048, F =
// 768, 1130 us; here 41, and on tiles the same). What bounds it is memory: a wave has 8 to 16
// loads of 1 KB in flight and never passes weights through LDS (one token, two experts, K =
// 4096, F = 14336: 470 MB of gate and up in 81 us = 5.8 TB/s, of a pure read's 7.1; two rows on
// each of eight experts, forward: 454 us, on tiles of 128 rows 558). Rows of odd widths, and
// the last 128 columns of others, are loaded a step at a time with nothing in flight (the
// token at K = 4095, F = 14335: 873 us, at the even widths 121).
//  - 16-bit weights lie [K, N]: a lane (i, g) loads 8 columns 8 i .. + 7 of the k rows 8 g .. + 7
//    of a 32-k step and turns that 8 x 8 block (32 byte permutes); register c then holds
//    eight k of column 8 i + c, the operand of one v_mfma_f32_16x16x32: the order of the
//    columns among the instruction's rows is free.
//  - int8 weights lie [N, K]: a lane loads 16 k of one column (64 columns a workgroup, 128 k
//    a step, so that the two loads of a row's 128 bytes follow each other).
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
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kBufferFlags = 0x00027000;  // raw 32-bit buffer
// Policies of the weights' loads: past the caches where the weights are larger than the
// caches keep from one call to the next (one token of E = 8, K = 4096, F = 14336 134 -> 123 us;
// but E = 64, K = 256, F = 128 11.0 -> 11.7). int8 rows are loaded 64 bytes at a time, whose
// lines the next load needs again (E = 128, K = 2048, N = 768, 128 rows, with their
// quantisation: 52.4 us, past the caches 53.0), 16-bit rows a whole line and more.
constexpr int kStreamed = 2, kCached = 0;
constexpr std::size_t kStreamedBytes = std::size_t{64} << 20;

constexpr int kCus = 256;  // MI355X

// A step: its k, the workgroup's columns, whether k runs along the weights' rows,
// accumulator and product of the matrix instruction (int8 steps are two of them: 128 bytes
// of every weight row).
template <typename T>
struct Step;
template <>
struct Step<bf16> {
  static constexpr int kK = 32, kCols = 128;
  static constexpr bool kKC = false;
  typedef f4 acc;
  typedef bf16 frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
};
template <>
struct Step<f16> {
  static constexpr int kK = 32, kCols = 128;
  static constexpr bool kKC = false;
  typedef f4 acc;
  typedef f16 frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
};
template <>
struct Step<int8_t> {
  static constexpr int kK = 128, kCols = 64;
  static constexpr bool kKC = true;
  typedef i4 acc;
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// 16 bytes at base (uniform) + offset + lane offset. `WHOLE`: all of them exist and lie on
// a 4-byte boundary; else any alignment, the first `count` elements exist. POLICY:
// of whole loads.
template <bool WHOLE, int POLICY, typename T>
__device__ __forceinline__ i4 load16(const T* base, uint32_t offset, uint32_t lane_offset, int count) {
  if constexpr (WHOLE) {
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, -1, kBufferFlags);
    return __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(buffer, lane_offset, offset, POLICY));
  }
  constexpr int V = 16 / sizeof(T);
  typedef T chunk __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  const char* at = reinterpret_cast<const char*>(base) + offset + lane_offset;
  chunk v = {};
  if (count >= V) {
    v = *reinterpret_cast<const chunk*>(at);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i < count) v[i] = reinterpret_cast<const T*>(at)[i];
    }
  }
  return __builtin_bit_cast(i4, v);
}

constexpr int kGroup = 16;  // rows of a workgroup

// The `index`-th group of rows, counted through the experts (-1: there are fewer): its expert,
// first row and rows. By one wave's lanes.
__device__ __forceinline__ int find_group(const Product& p, int index, int* first, int* count) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int most = 0;  // bound of the experts before
  for (int e0 = 0; e0 < p.experts; e0 += 64) {
    const int e = e0 + lane;
    int from = 0, to = 0;
    if (e < p.experts) {
      from = rr::dev::offset_at(p.offsets, e, p.rows);
      to = rr::dev::offset_at(p.offsets, e + 1, p.rows);
    }
    from = max(most, rr::dev::wave_inclusive_max(from));
    to = max(from, to);
    most = __builtin_amdgcn_readlane(to, 63);
    const int groups = (to - from + kGroup - 1) / kGroup;
    const int through = rr::dev::wave_inclusive_scan(groups);
    const int here = __builtin_amdgcn_readlane(through, 63);
    if (index < here) {
      const int at = __builtin_ctzll(__ballot(through > index));
      const int r0 = (index - __builtin_amdgcn_readlane(through - groups, at)) * kGroup;
      *first = __builtin_amdgcn_readlane(from, at) + r0;
      *count = min(__builtin_amdgcn_readlane(to, at) - *first, kGroup);
      return e0 + at;
    }
    index -= here;
  }
  return -1;
}

// (waves a SIMD: what the accumulators and the two sets of weights leave room for)
template <typename T, class Epi, int W, int POLICY>
__global__ __launch_bounds__(64 * W, Epi::kDual ? 2 : 3) void rr_expert_rows_kernel(Product prm, float* parts, int splits, int blocks) {
  using M = Step<T>;
  using Acc = typename M::acc;
  constexpr bool kKC = M::kKC;
  constexpr int B = Epi::kDual ? 2 : 1;
  constexpr int C = kKC ? 4 : 8;       // accumulators of 16 columns
  constexpr int X = kKC ? 2 : 1;       // matrix instructions of a step for each
  constexpr int V = 16 / sizeof(T);    // elements of a load
  extern __shared__ __align__(16) char smem[];
  i4* lds = reinterpret_cast<i4*>(smem);  // [W / 2][B * C][64]
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int block = static_cast<int>(blockIdx.x) % blocks;
  const int split = static_cast<int>(blockIdx.x) / blocks % splits;
  int first, count;
  const int e = find_group(prm, static_cast<int>(blockIdx.x) / blocks / splits, &first, &count);
  if (e < 0) return;
  const int n0 = block * M::kCols;
  const int K = prm.K, N = prm.N;
  // this wave's steps
  const int steps = (K + M::kK - 1) / M::kK;
  const int share = split * W + wave, shares = splits * W;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * share / shares);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (share + 1) / shares);
  const T* weights[2] = {static_cast<const T*>(prm.b) + static_cast<std::size_t>(e) * K * N,
                         static_cast<const T*>(Epi::kDual ? prm.b_up : prm.b) + static_cast<std::size_t>(e) * K * N};
  // every row that is loaded starts on a 4-byte boundary
  const bool aligned = ((reinterpret_cast<uintptr_t>(prm.a) | reinterpret_cast<uintptr_t>(weights[0]) |
                         reinterpret_cast<uintptr_t>(weights[1]) | sizeof(T) * K | (kKC ? 0 : sizeof(T) * N)) & 3) == 0;

  Acc acc[B][C] = {};
  // byte offsets of the lane: of its rows (rows past the last repeat it: their results
  // are not stored) and in the weights
  constexpr uint32_t S = sizeof(T);
  const T* x = static_cast<const T*>(prm.a) + static_cast<std::size_t>(first) * K;
  const uint32_t x_at = S * (static_cast<uint32_t>(min(li, count - 1)) * static_cast<uint32_t>(K) + g * V);
  uint32_t w_at[kKC ? 4 : 1];
#pragma unroll
  for (int j = 0; j < (kKC ? 4 : 1); ++j) {
    w_at[j] = kKC ? S * (static_cast<uint32_t>(min(16 * j + li, N - 1 - n0)) * static_cast<uint32_t>(K) + g * V)
                  : S * (static_cast<uint32_t>(8 * g) * static_cast<uint32_t>(N) + 8 * li);
  }
  struct Rows {
    i4 v[X];
  };
  struct Weights {
    i4 v[8];
  };
  // what a step multiplies; `whole`: neither the columns nor the step are cut
  auto load_rows = [&](Rows& o, int s, auto whole) {
#pragma unroll
    for (int h = 0; h < X; ++h) {
      o.v[h] = load16<decltype(whole)::value, kCached>(x + s * M::kK, S * 4 * h * V, x_at, K - s * M::kK - (4 * h + g) * V);
    }
  };
  auto load_weights = [&](Weights& o, int b, int s, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    if constexpr (kKC) {  // [fragment][half]: columns 16 j + li, k of half h
      const T* at = weights[b] + static_cast<std::size_t>(n0) * K + s * M::kK;  // (uniform, as below)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        o.v[q] = load16<kWhole, POLICY>(at, S * 4 * (q & 1) * V, w_at[q >> 1], K - s * M::kK - (4 * (q & 1) + g) * V);
        if (!kWhole) __builtin_amdgcn_sched_barrier(0);  // (the pieces of all eight at once would fill the registers)
      }
    } else {  // k 8 g + q: columns 8 li .. + 7
      const T* at = weights[b] + static_cast<std::size_t>(s * M::kK) * N + n0;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        o.v[q] = load16<kWhole, POLICY>(at, S * static_cast<uint32_t>(q) * static_cast<uint32_t>(N), w_at[0],
                                s * M::kK + 8 * g + q < K ? N - n0 - 8 * li : 0);
        if (!kWhole) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto multiply = [&](const Weights& w, const Rows& r, int b) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if constexpr (kKC) {
#pragma unroll
        for (int h = 0; h < X; ++h) acc[b][c] = M::mul(w.v[2 * c + h], r.v[h], acc[b][c]);
      } else {
        i4 column;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          column[m] = static_cast<int>(__builtin_amdgcn_perm(static_cast<uint32_t>(w.v[2 * m + 1][c >> 1]),
                                                             static_cast<uint32_t>(w.v[2 * m][c >> 1]),
                                                             (c & 1) != 0 ? 0x07060302U : 0x05040100U));
        }
        acc[b][c] = M::mul(column, r.v[0], acc[b][c]);
      }
    }
  };
  // Two sets of weights in registers: while one is multiplied the other is on its way.
  // Dual products hold one step's gate and up weights, others two steps.
  const std::integral_constant<bool, true> whole;
  const std::integral_constant<bool, false> cut;
  int s = s0;
  const int end = n0 + M::kCols > N || !aligned ? s0 : max(s0, min(s1, K / M::kK));  // of the whole steps
  constexpr int D = Epi::kDual ? 1 : 2;                                 // steps in the two sets
  if (s + D <= end) {
    Weights w0, w1;
    Rows r0v, r1v;
    load_rows(r0v, s, whole);
    load_weights(w0, 0, s, whole);
    if constexpr (!Epi::kDual) load_rows(r1v, s + 1, whole);
    load_weights(w1, B - 1, s + D - 1, whole);
#pragma unroll 1
    for (; s + 2 * D <= end; s += D) {
      __builtin_amdgcn_sched_barrier(0);
      Rows next;
      multiply(w0, r0v, 0);
      __builtin_amdgcn_sched_barrier(0);  // (loads hoisted over the products would need registers of their own)
      if constexpr (Epi::kDual) {
        load_rows(next, s + 1, whole);
      } else {
        load_rows(r0v, s + 2, whole);
      }
      load_weights(w0, 0, s + D, whole);
      __builtin_amdgcn_sched_barrier(0);
      multiply(w1, Epi::kDual ? r0v : r1v, B - 1);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (Epi::kDual) {
        r0v = next;
      } else {
        load_rows(r1v, s + 3, whole);
      }
      load_weights(w1, B - 1, s + 2 * D - 1, whole);
    }
    multiply(w0, r0v, 0);
    multiply(w1, Epi::kDual ? r0v : r1v, B - 1);
    s += D;
  }
#pragma unroll 1
  for (; s < s1; ++s) {
    Rows r;
    Weights w;
    load_rows(r, s, cut);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      load_weights(w, b, s, cut);
      multiply(w, r, b);
    }
  }

  // the waves' sums, halved round by round
#pragma unroll
  for (int half = W / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int q = 0; q < B * C; ++q) {
        lds[((wave - half) * B * C + q) * 64 + lane] = __builtin_bit_cast(i4, acc[q / C][q % C]);
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int q = 0; q < B * C; ++q) {
        acc[q / C][q % C] += __builtin_bit_cast(Acc, lds[(wave * B * C + q) * 64 + lane]);
      }
    }
    __syncthreads();
  }
  if (wave != 0) return;
  // lane: row li; columns 32 g + 8 r + 0..7 (KC: 16 j + 4 g + 0..3)
  if (li >= count) return;
  const std::size_t row = static_cast<std::size_t>(first) + li;
  constexpr int E = kKC ? 4 : 8;  // columns of a store
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int n = n0 + (kKC ? 16 * p + 4 * g : 32 * g + 8 * p);
    if (n >= N) continue;
    float v[B][E];
#pragma unroll
    for (int b = 0; b < B; ++b) {
#pragma unroll
      for (int q = 0; q < E; ++q) v[b][q] = static_cast<float>(kKC ? acc[b][p][q] : acc[b][q][p]);
    }
    if (parts != nullptr) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        Cols<float, E>::store(parts + (static_cast<std::size_t>(b * splits + split) * prm.rows + row) * N + n, v[b], N - n);
      }
    } else if constexpr (Epi::kDual) {
      Epi::template emit<E>(prm, e, row, n, N - n, v[0], v[1]);
    } else {
      Epi::template emit<E>(prm, e, row, n, N - n, v[0]);
    }
  }
}

// The splits' parts added in order, eight columns a thread, for the rows from the first
// expert's to the last one's.
template <class Epi>
__global__ __launch_bounds__(256) void rr_expert_rows_sum_kernel(Product prm, const float* parts, int splits) {
  constexpr int B = Epi::kDual ? 2 : 1;
  const int eights = (prm.N + 7) / 8;
  const int first = rr::dev::offset_at(prm.offsets, 0, prm.rows);
  int end = 0;
  for (int e = static_cast<int>(threadIdx.x) & 63; e <= prm.experts; e += 64) end = max(end, rr::dev::offset_at(prm.offsets, e, prm.rows));
  end = __builtin_amdgcn_readlane(rr::dev::wave_inclusive_max(end), 63);
  const std::size_t total = static_cast<std::size_t>(end - first) * eights;
  for (std::size_t t = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x; t < total;
       t += static_cast<std::size_t>(gridDim.x) * 256) {
    const std::size_t row = first + t / eights;
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

template <typename T, class Epi, int W, int POLICY>
hipError_t launch(const Product& prm, float* parts, int splits, hipStream_t stream) {
  constexpr std::size_t lds = static_cast<std::size_t>(W / 2) * (Epi::kDual ? 2 : 1) * (Step<T>::kKC ? 4 : 8) * 64 * sizeof(i4);
  static_assert(lds <= 64 * 1024, "no attribute raises the limit");
  const int blocks = (prm.N + Step<T>::kCols - 1) / Step<T>::kCols;
  // (the most groups: of n rows an expert has (n - 1) / kGroup + 1 at most)
  const int busy = std::min(prm.experts, prm.rows);
  const std::size_t grid = static_cast<std::size_t>((prm.rows - busy) / kGroup + busy) * blocks * splits;
  rr_expert_rows_kernel<T, Epi, W, POLICY><<<dim3(static_cast<unsigned>(grid)), 64 * W, lds, stream>>>(prm, parts, splits, blocks);
  if (splits > 1) {
    if constexpr (sizeof(T) == 2) {
      const std::size_t threads = static_cast<std::size_t>(prm.rows) * ((prm.N + 7) / 8);
      const unsigned sums = static_cast<unsigned>(std::min<std::size_t>((threads + 255) / 256, 2048));
      rr_expert_rows_sum_kernel<Epi><<<dim3(sums), 256, 0, stream>>>(prm, parts, splits);
    }
  }
  return hipGetLastError();
}

// Waves that share a sum: so that each has six steps and more, but four where there are
// four steps.
template <typename T, class Epi, int POLICY>
hipError_t launch_waves(const Product& prm, float* parts, int splits, hipStream_t stream) {
  const int steps = (prm.K + Step<T>::kK - 1) / Step<T>::kK / splits;
  return steps >= 48 ? launch<T, Epi, 8, POLICY>(prm, parts, splits, stream)
                     : launch<T, Epi, 4, POLICY>(prm, parts, splits, stream);
}

}  // namespace

// Five rows an expert on average, of int8 three: tiles then multiply 64 rows for every few,
// but read an expert's weights once however many rows it has, and here every 16 rows read them
// again (E = 128, K = 2048, F = 768: 640 rows 194 us without skew and 216 with Zipf's 1, 641
// on tiles 209 and 210; E = 8, K = 4096, F = 14336: 40 rows 457, 41 on tiles 522; int8, E = 128,
// K = 2048, N = 768: 384 rows 37 to 39, 385 on tiles 37). Rows that all go to one expert cost up to
// twice the tiles' time (5120 rows on one of 1024 experts, K = 1024, F = 256: 89 us, 5121 on
// tiles 41).
bool expert_rows_ok(int rows, int experts, bool int8) {
  return rows <= 16 || rows <= (int8 ? 3 : 5) * std::min(rows, experts);
}

int expert_rows_splits(int rows, int experts, int columns, int length) {
  if (!expert_rows_ok(rows, experts, false)) return 1;
  const int groups = std::min(rows, experts) * ((columns + Step<bf16>::kCols - 1) / Step<bf16>::kCols);
  const int most = std::min(length / 1024, 8);
  return std::max(1, std::min(most, kCus / groups));
}

template <typename T, class Epi>
hipError_t expert_rows(const Product& prm, float* parts, int splits, hipStream_t stream) {
  if constexpr (!Step<T>::kKC) {
    const std::size_t bytes = static_cast<std::size_t>(std::min(prm.experts, prm.rows)) * prm.K * prm.N * sizeof(T);
    if (bytes > kStreamedBytes) return launch_waves<T, Epi, kStreamed>(prm, parts, splits, stream);
  }
  return launch_waves<T, Epi, kCached>(prm, parts, splits, stream);
}

template hipError_t expert_rows<bf16, EpiGate<bf16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<bf16, EpiStore<bf16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<f16, EpiGate<f16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<f16, EpiStore<f16>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8<float, true>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8<bf16, true>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8<f16, true>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8Gate<float, true>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8Gate<bf16, true>>(const Product&, float*, int, hipStream_t);
template hipError_t expert_rows<int8_t, EpiInt8Gate<f16, true>>(const Product&, float*, int, hipStream_t);

}  // namespace rr::kern
