// 4-bit products for few rows an expert (decoding): the weights are read once from memory,
// a line at a time.
//
// A workgroup of W waves takes R = 64 or 32 weight rows (of one operand, or half of them of each of
// two) of one expert and 16 of its rows; the waves share the blocks of a row and add up through LDS in a
// fixed order. A step is a slice of 256 elements: 128 bytes of every row, which eight lanes
// bring as one line straight into the wave's own part of LDS, and eight scales. It is read
// from there in operand order, and the next slice is on its way before it is multiplied. What bounds it is memory: two rows
// of two experts, K = 4096, N = 14336, gated: 125 MB in 22.7 us (5.5 TB/s; lanes that load their
// operands themselves, 64 bytes of a row at a time, 28 us; cached 25.7).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "large_lds.h"
#include "mxfp4.h"
#include "mxfp4_rows.h"
#include "row_groups.h"
#include "tile_stream.h"
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

typedef float f4 __attribute__((ext_vector_type(4)));

// Weights that are larger than the caches keep from one call to the next are loaded past them.
constexpr std::size_t kStreamedBytes = std::size_t{64} << 20;
constexpr int kScaleBytes = 8;  // of a row's slice

// A wave's part of LDS for R weight rows: weights, rows, their scales.
template <int R>
struct Part {
  static constexpr int kRows = R * kSliceBytes;
  static constexpr int kWeightScales = kRows + 16 * kSliceBytes;
  static constexpr int kRowScales = kWeightScales + R * kScaleBytes;
  static constexpr int kBytes = kRowScales + 16 * kScaleBytes;
};

// HALF: which of the scales' two low bytes counts.
template <int HALF>
__device__ __forceinline__ f4 multiply(i4 a, i4 b, f4 c, int a_scale, int b_scale) {
  typedef int i8 __attribute__((ext_vector_type(8)));
  const i8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  constexpr int kE2M1 = 4;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, kE2M1, kE2M1, HALF, a_scale, HALF, b_scale);
}

template <class Epi, int W, int R, bool STREAMED>
__global__ __launch_bounds__(64 * W, 3) void rr_mxfp4_rows_kernel(Product prm, int blocks) {
  constexpr int B = Epi::kDual ? 2 : 1;
  constexpr int F = R / 16 / B;  // fragments of 16 columns of each right operand
  using L = Part<R>;
  constexpr int kCols = 16 * F;
  extern __shared__ __align__(128) char smem[];  // [W][L::kBytes]
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int block = static_cast<int>(blockIdx.x % static_cast<unsigned>(blocks));
  int first, count;
  const int e = find_group(prm, static_cast<int>(blockIdx.x / static_cast<unsigned>(blocks)), &first, &count);
  if (e < 0) return;
  const int n0 = block * kCols;
  const int N = prm.N;
  const int64_t row_bytes = prm.lda;
  // this wave's slices
  const int slices = (prm.K + 7) / 8;
  const int s0 = static_cast<int>(static_cast<int64_t>(slices) * wave / W);
  const int s1 = static_cast<int>(static_cast<int64_t>(slices) * (wave + 1) / W);

  const int columns = min(N - n0, kCols);
  const int64_t channel = static_cast<int64_t>(e) * N + n0;
  const int64_t x_slice = static_cast<int64_t>(prm.rows) * kScaleBytes, w_slice = static_cast<int64_t>(prm.experts) * N * kScaleBytes;
  // Rows past the last and columns past N are past the buffers' records: zeros. (What lies past
  // a row's end in its last slice is the next row's: its scales count as 2^-127.)
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((RR_LDS char*)smem)) + wave * L::kBytes;
  const uint32_t at_lane = static_cast<uint32_t>((lane >> 3) * prm.lda) + (static_cast<uint32_t>((lane & 7) ^ (lane >> 3)) << 4);
  auto load = [&](int s) {
    const int64_t from = static_cast<int64_t>(s) * kSliceBytes;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const char* w = static_cast<const char*>(b == 0 ? prm.b : prm.b_up) + channel * row_bytes + from;
      const int64_t left = columns * row_bytes - from;
#pragma unroll
      for (int q = 0; q < 2 * F; ++q) {
        const i4 buffer = make_buffer(w + 8 * q * row_bytes, left - 8 * q * row_bytes);
        const uint32_t to = lds + (b * 2 * F + q) * 1024;
        if constexpr (STREAMED) {
          stream_to_lds(buffer, at_lane, to);
        } else {
          load_to_lds(buffer, at_lane, to);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t skip = (first + 8 * q) * row_bytes + from;
      load_to_lds(make_buffer(static_cast<const char*>(prm.a) + skip, (count - 8 * q) * row_bytes - from), at_lane, lds + L::kRows + q * 1024);
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const char* scales = static_cast<const char*>(b == 0 ? prm.in : prm.in_up) + channel * kScaleBytes + s * w_slice;
#pragma unroll
      for (int q = 0; q < (F + 1) / 2; ++q) {
        if (F > 1 || lane < 32) {
          load_words_to_lds(make_buffer(scales + q * 256, columns * kScaleBytes - q * 256), lane * 4,
                            lds + L::kWeightScales + b * F * 128 + q * 256);
        }
      }
    }
    if (lane < 32) {
      load_words_to_lds(make_buffer(static_cast<const char*>(prm.a2) + first * static_cast<int64_t>(kScaleBytes) + s * x_slice, count * kScaleBytes),
                        lane * 4, lds + L::kRowScales);
    }
  };
  // block 2 g + h of a row's slice
  uint32_t at_row[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) at_row[h] = lds + li * kSliceBytes + (static_cast<uint32_t>((2 * g + h) ^ (li & 7)) << 4);
  const uint32_t at_scale = lds + li * kScaleBytes + 2 * g;
  auto read_scales = [&](uint32_t at) { return static_cast<int>(*reinterpret_cast<RR_LDS const uint16_t*>(at)); };

  f4 acc[B][F] = {};
  if (s0 < s1) load(s0);
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    wait_loads<0>();
    i4 w[B * F][2], x[2];
    int w_scale[B * F];
    const int left = prm.K - 8 * s - 2 * g;  // blocks of a row from the lane's on; scales past them are not looked at
    const int mask = left >= 2 ? 0xFFFF : left == 1 ? 0xFF : 0;
#pragma unroll
    for (int j = 0; j < B * F; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) w[j][h] = read16(at_row[h] + j * 16 * kSliceBytes);
      w_scale[j] = read_scales(at_scale + L::kWeightScales + j * 16 * kScaleBytes);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) x[h] = read16(at_row[h] + L::kRows);
    const int x_scale = read_scales(at_scale + L::kRowScales) & mask;
    wait_lds();
    if (s + 1 < s1) load(s + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < B * F; ++j) {
      acc[j / F][j % F] = multiply<0>(w[j][0], x[0], acc[j / F][j % F], w_scale[j] & mask, x_scale);
      acc[j / F][j % F] = multiply<1>(w[j][1], x[1], acc[j / F][j % F], w_scale[j] & mask, x_scale);
    }
  }
  // (the parts of LDS become the sums')
  f4(*s_sums)[B * F][64] = reinterpret_cast<f4(*)[B * F][64]>(smem);
  static_assert(W / 2 * B * F * 64 * sizeof(f4) <= W * L::kBytes);
  __syncthreads();

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

// Workgroups that share an expert's columns, `weight_rows` each.
std::size_t blocks_of(int columns, bool dual, int weight_rows = 64) {
  const int of_one = weight_rows / (dual ? 2 : 1);
  return static_cast<std::size_t>((columns + of_one - 1) / of_one);
}

template <class Epi, int W, int R, bool STREAMED>
hipError_t launch(const Product& prm, hipStream_t stream) {
  constexpr int kLds = W * Part<R>::kBytes;
  if constexpr (kLds > 64 * 1024) {
    static std::atomic<uint64_t> allowed{0};
    const hipError_t error = allow_lds(reinterpret_cast<const void*>(rr_mxfp4_rows_kernel<Epi, W, R, STREAMED>), kLds, &allowed);
    if (error != hipSuccess) return error;
  }
  const std::size_t blocks = blocks_of(prm.N, Epi::kDual, R);
  const std::size_t grid = most_groups(prm.rows, prm.experts) * blocks;
  rr_mxfp4_rows_kernel<Epi, W, R, STREAMED><<<dim3(static_cast<unsigned>(grid)), 64 * W, kLds, stream>>>(prm, static_cast<int>(blocks));
  return hipGetLastError();
}

// Few waves that have many slices each, but enough of them in all (two rows, two experts: K =
// 4096, N = 14336, gated, two waves 23 us, four 24, eight 29; K = 14336, N = 4096 34, 22 and 16). One
// where a row is one slice (1302 rows of 166 experts, K = 64, N = 5280: 36 -> 20 us).
// Workgroups of half the weight rows where whole ones would leave CUs idle, with eight waves for long
// sums and four for others (two rows, two experts: K = 14336, N = 4096 15.2 -> 12.6 us, by sixteen waves
// 12.8; K = N = 4096 6.6 -> 5.9; 128 rows of one expert, K = N = 1024 5.1 -> 4.4, by eight 4.6), but not for
// sums of a few slices (40 rows of three experts, K = 512, N = 520, gated: 4.3 and 4.8).
constexpr std::size_t kFewWorkgroups = 256;

template <class Epi, bool STREAMED>
hipError_t launch_waves(const Product& prm, hipStream_t stream) {
  const int slices = (prm.K + 7) / 8;
  const std::size_t workgroups = most_groups(prm.rows, prm.experts) * blocks_of(prm.N, Epi::kDual);
  if (workgroups < kFewWorkgroups && slices >= 16) return launch<Epi, 8, 32, STREAMED>(prm, stream);
  // (the weights of so few workgroups' columns of less than 16 slices are 31 MB at most)
  static_assert(kFewWorkgroups * 64 * 15 * kSliceBytes < kStreamedBytes);
  if (workgroups < kFewWorkgroups && slices >= 4) return launch<Epi, 4, 32, false>(prm, stream);
  if (slices >= 16 && workgroups < 384) return launch<Epi, 8, 64, STREAMED>(prm, stream);
  if (slices >= 8 && workgroups < 768) return launch<Epi, 4, 64, STREAMED>(prm, stream);
  if (slices >= 2) return launch<Epi, 2, 64, STREAMED>(prm, stream);
  return launch<Epi, 1, 64, STREAMED>(prm, stream);
}

}  // namespace

// Rows an expert on average: a tile multiplies 64 rows for every few but reads an expert's weights
// once, here every 16 rows read them again. Long sums: twelve (16 slices, E = 8, N = 14336: 8 rows an
// expert 39 us, on tiles 49; 12: 46 and 49; 16: 52 and 50), 16 for eight slices (E = 128, N = 768,
// gated: 44 and 46). Of short ones a tile is mostly prologue and epilogue: 40 (four slices, E =
// 64, N = 1024, gated: 32 rows 22 and 25, 48: 27 and 28, 64: 33 and 28; two, N = 2048: 32 rows 16 and 19, 48: 21
// and 20; one, E = 167, N = 4816: 32 rows 48 and 52, 48: 62 and 57).
// And with more where there are few tiles, whose slices follow each other while most of the
// card is idle: K = N = 4096, one expert, 128 rows (512 workgroups here) 9.3 us, on tiles 18.8; K =
// 2784, N = 672, one expert, 256 rows (176) 6.3 and 17.9. The limit of 640 workgroups leaves to tiles what is
// faster on them from some 2000 on (K = 4096, N = 14336, one expert, 160 rows, 2240: 31 and 25.5; K = 2048,
// N = 4096, eight experts, 512 rows, 2496: 19.4 and 14.2), and some that is not below that (K = N = 4096,
// one expert, 256 rows, 1024: 13.9 and 21; K = N = 1024, eight experts, 1024 rows, 1136: 7.4 and 10.4).
bool mxfp4_rows_ok(const Product& prm, bool dual) {
  const std::size_t workgroups = most_groups(prm.rows, prm.experts) * blocks_of(prm.N, dual);
  if (workgroups >= std::size_t{1} << 23) return false;  // (a launch has less than 2^32 threads)
  const int slices = (prm.K + 7) / 8;
  const long rows = slices <= 4 ? 40 : slices <= 8 ? 16 : 12;
  return prm.rows <= 16 || prm.rows <= rows * std::min(prm.rows, prm.experts) || workgroups <= 640;
}

template <class Epi>
hipError_t mxfp4_rows(const Product& prm, hipStream_t stream) {
  const std::size_t bytes = static_cast<std::size_t>(std::min(prm.experts, prm.rows)) * prm.N * prm.lda * (Epi::kDual ? 2 : 1);
  return bytes > kStreamedBytes ? launch_waves<Epi, true>(prm, stream) : launch_waves<Epi, false>(prm, stream);
}

template hipError_t mxfp4_rows<EpiMxStore<float>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiMxStore<bf16>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiMxStore<f16>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiMxGate<float>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiMxGate<bf16>>(const Product&, hipStream_t);
template hipError_t mxfp4_rows<EpiMxGate<f16>>(const Product&, hipStream_t);

}  // namespace rr::kern
