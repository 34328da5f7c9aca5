// Grouped products of the expert block: 256-column tiles of 256 or 128 rows on the 16-bit
// and int8 matrix instructions (v_mfma_f32_16x16x32_bf16 / _f16, v_mfma_i32_16x16x64_i8).
//
//   rows of expert e:      C = A[rows] B[e]  (one or two B, or two pairs A, B added up)
//   weights of expert e:   C[e] = A[rows]^T B[rows]
// sums in FP32 (int32), rounded once by the epilogue.
//
// One workgroup of eight waves a CU walks over output tiles; a k slice is 128 bytes of
// every row (64 16-bit or 128 int8 elements). Both operands' slices go straight from
// memory into one of two LDS stages of 64 KB (tiles of 128 rows: three of 48 KB; buffer
// loads, 16 bytes a lane), that many slices ahead of the products and across the end of a
// tile: the stream of slices does not stop for an epilogue.
//  - Left operand and right operand may each have k along rows (KC: 128-byte rows in
//    LDS, read with ds_read_b128) or down columns (KS: rows of 128 columns, read with
//    ds_read_b64_tr_b16, which hands each lane four k of one column), so that no product
//    of the block, forward or backward, needs a transposed copy.
//  - 16-byte chunks are placed at chunk ^ f(row) by loading permuted chunks: the lanes
//    that read together then reach all 64 banks.
//  - What lies past a row's, segment's or expert's end is cut off by the buffer's record
//    count (reads past it give zeros), what lies past the sum's length inside a row by
//    an offset past it.
//  - Wave (wm, wn) sums 128 rows x 64 columns (dual products: 32 columns of each right
//    operand, so that gate and up of an element meet in one lane). The right operand is
//    the instruction's first one and its columns are dealt so that a lane ends with 16 (8
//    and 8) adjacent columns of a row: wide stores, no exchange.
//  - A wave fetches the operands of its next 16 products while it issues the present
//    ones; the workgroup meets once or twice a slice.
//
// What bounds it: large products the slices' loads that miss an XCD's L2 (8192 skewed rows of
// eight experts, K = 4096, F = 14336: gate and up 1922 us = 1.00 PFLOP/s, 0.67 of a dense
// library product of that size; without its loads 1426, the products alone 1052; data
// gradients 2072, weight gradients 1973 and 937 us); int8 the power that the products draw
// (16384 rows of eight experts, K = 4096, N = 14336: 917 us = 2.1 POP/s, a dense library product
// of that size 819); experts of a hundred rows the weights from HBM and what a few tiles a
// CU leave idle (8192 rows of 64 experts, K = 1024, F = 512, forward and backward: 275 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "expert_gemm.h"
#include "launchers.h"
#include "tile_stream.h"
#include "tiles.h"
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512;

template <typename T>
struct Matrix;
template <>
struct Matrix<bf16> {
  typedef bf16 frag __attribute__((ext_vector_type(8)));
  typedef f4 acc;
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
};
template <>
struct Matrix<f16> {
  typedef f16 frag __attribute__((ext_vector_type(8)));
  typedef f4 acc;
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
};
template <>
struct Matrix<int8_t> {
  typedef i4 acc;
  static __device__ __forceinline__ acc mul(i4 a, i4 b, acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};

// A kernel: element type, whether A and B have k along rows (KC), weight gradients or row
// products, epilogue, how slices come (DIRECT into LDS, or through registers), and the
// rows of a tile. Tiles of 128 rows leave room for a third stage of LDS.
template <typename T_, bool A_KC, bool B_KC, bool WEIGHTS, class Epi_, bool DIRECT, int ROWS>
struct Kind {
  using T = T_;
  using Epi = Epi_;
  static constexpr bool kAKC = A_KC, kBKC = B_KC, kWeights = WEIGHTS, kDual = Epi_::kDual, kDirect = DIRECT;
  static constexpr int kTileRows = ROWS;
  static constexpr int kStages = DIRECT && ROWS == 128 ? 3 : 2;
  static constexpr int kABytes = ROWS * kSliceBytes;  // A's slice
  static constexpr int kStageBytes = kABytes + kTileCols * kSliceBytes;
  static_assert(ROWS == 128 || (DIRECT && ROWS == 256), "through registers a tile has 128 rows");
  static constexpr int kSlice = kSliceBytes / sizeof(T_);  // k of a slice
  static constexpr int kCols = kDual ? kTileCols / 2 : kTileCols;
  static_assert(A_KC || sizeof(T_) == 2, "transposing reads are 16-bit");
  static_assert(B_KC || sizeof(T_) == 2, "transposing reads are 16-bit");
};

// The chunk permutations f(row): KC by eight chunks of a 128-byte row, KS by 16 of a
// 256-byte row (k). The rows (and pieces) that 16 lanes read together differ in the bits
// used: KC A rows 16 i + 0..15; KC B columns 4 J a + 4 j + b (a, b in 0..3); KS k 8 g + 4 q + 0..3.
template <bool DUAL>
__device__ __forceinline__ int swizzle_b_row(int r) {
  return (r & 3) | ((r >> (DUAL ? 3 : 4)) & 1) << 2;
}
__device__ __forceinline__ int swizzle_a_k(int k) { return (k & 3) << 1 | ((k >> 3) & 1) << 3; }
template <bool DUAL>
__device__ __forceinline__ int swizzle_b_k(int k) {
  return DUAL ? (k & 3) << 2 : (k & 1) | ((k >> 1) & 1) << 3;
}

// Two transposing reads: eight k of one column, `at` and four rows further.
__device__ __forceinline__ i4 read_columns(uint32_t at) {
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<RR_LDS s4*>(at));
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<RR_LDS s4*>(at + 4 * 256));
  typedef int i2 __attribute__((ext_vector_type(2)));
  const i2 l = __builtin_bit_cast(i2, lo), h = __builtin_bit_cast(i2, hi);
  return i4{l[0], l[1], h[0], h[1]};
}

// Slices of `rows` rows, one at least.
__host__ __device__ constexpr int slices_of(int rows, int slice) { return rows > 0 ? (rows - 1) / slice + 1 : 1; }
static_assert(slices_of(0, 64) == 1 && slices_of(64, 64) == 1 && slices_of(65, 64) == 2);
static_assert(slices_of(0x7FFFFFFF, 64) == 1 << 25, "a sum with the slice would pass 31 bits");

// An output tile (uniform).
struct Tile {
  int e;           // expert
  int first;       // its first row
  int row0, rows;  // row products: first row and rows; weight gradients: first row of the result and rows there
  int n0;          // first column
  int slices;      // k slices, of all parts
};

template <class P>
__global__ __launch_bounds__(kThreads, 2) void rr_expert_gemm_kernel(Product prm) {
  using T = typename P::T;
  using M = Matrix<T>;
  using Acc = typename M::acc;
  constexpr int S = sizeof(T);
  extern __shared__ __align__(16) char smem[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((RR_LDS char*)smem));
  int32_t* s_off = reinterpret_cast<int32_t*>(smem + P::kStages * P::kStageBytes);  // [E + 1]
  int32_t* s_pre = s_off + prm.experts + 1;                             // [E + 1] full row tiles before expert e
  int32_t* s_pre2 = s_pre + prm.experts + 1;                            // [E + 1] short row tiles before expert e
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int li = lane & 15, g = lane >> 4;
  const int experts = prm.experts;

  for (int e = tid; e <= experts; e += kThreads) s_off[e] = rr::dev::offset_at(prm.offsets, e, prm.rows);
  __syncthreads();
  if (wave == 0) {
    raise_offsets(s_off, experts, lane);
    if constexpr (!P::kWeights) build_tile_prefix<P::kTileRows, true>(s_off, s_pre, s_pre2, experts, lane);
  }
  __syncthreads();
  const int col_tiles = (prm.N + P::kCols - 1) / P::kCols;
  const int m_tiles = P::kWeights ? (prm.M + P::kTileRows - 1) / P::kTileRows : 0;
  const int full_rows = P::kWeights ? 0 : __builtin_amdgcn_readfirstlane(s_pre[experts]);
  const int short_rows = P::kWeights ? 0 : __builtin_amdgcn_readfirstlane(s_pre2[experts]);
  const int total_full = full_rows * col_tiles;
  const int total = P::kWeights ? experts * m_tiles * col_tiles : total_full + short_rows * col_tiles;
  const int grid = static_cast<int>(gridDim.x);
  const int worker = tile_worker(static_cast<int>(blockIdx.x), grid);
  const int part_slices = P::kWeights ? 0 : (prm.K + P::kSlice - 1) / P::kSlice;
  const int parts = P::kWeights || prm.a2 == nullptr || S == 1 ? 1 : 2;

  // The last whole round holds full and short tiles: the workgroups of the short ones are
  // done first.
  const int whole_rounds = total / grid * grid;
  const bool mixed = !P::kWeights && whole_rounds != 0 && total_full < whole_rounds && total_full > whole_rounds - grid;
  // The workgroup's tile of a round; false where there is none. The last, partial round
  // goes to the workgroups in dispatch order, over all XCDs (or from the last one, see mixed);
  // its tiles are cut into two or four by their rows where that many workgroups are left (8192 rows of eight experts, K =
  // 28672, N = 4096: 2.25 rounds).
  auto decode = [&](int dealt, Tile& tl) {
    const int left = total - dealt;
    if (left <= 0) return false;
    int t = dealt + worker, sub = 0, span = P::kTileRows;
    if (left < grid) {
      const int cuts = P::kTileRows == 256 && 4 * left <= grid ? 4 : 2 * left <= grid ? 2 : 1;
      const int mine = mixed ? grid - 1 - worker : static_cast<int>(blockIdx.x);
      sub = mine / left;
      if (sub >= cuts) return false;
      t = dealt + mine - sub * left;
      span = P::kTileRows / cuts;
    }
    int rt, ct;
    if constexpr (P::kWeights) {
      tl.e = t / (m_tiles * col_tiles);
      place_tile(t - tl.e * m_tiles * col_tiles, m_tiles, col_tiles, &rt, &ct);
      tl.first = __builtin_amdgcn_readfirstlane(s_off[tl.e]);
      const int count = __builtin_amdgcn_readfirstlane(s_off[tl.e + 1]) - tl.first;
      tl.row0 = rt * P::kTileRows;
      tl.rows = min(prm.M - tl.row0, P::kTileRows);
      // (an expert without rows takes one slice of zeros)
      tl.slices = slices_of(count, P::kSlice);
    } else {
      // (an expert's tiles lie together, so that those which run side by side share weights)
      const bool is_short = t >= total_full;
      const int32_t* pre = is_short ? s_pre2 : s_pre;
      if (is_short) t -= total_full;
      tl.e = __builtin_amdgcn_readfirstlane(tile_expert(pre, experts, t / col_tiles));
      const int before = __builtin_amdgcn_readfirstlane(pre[tl.e]);
      place_tile(t - before * col_tiles, __builtin_amdgcn_readfirstlane(pre[tl.e + 1]) - before, col_tiles, &rt, &ct);
      tl.first = __builtin_amdgcn_readfirstlane(s_off[tl.e]);
      const int end = __builtin_amdgcn_readfirstlane(s_off[tl.e + 1]);
      tl.row0 = tl.first + (is_short ? (end - tl.first) / P::kTileRows : rt) * P::kTileRows;
      tl.rows = min(end - tl.row0, P::kTileRows);
      tl.slices = part_slices * parts;
    }
    tl.n0 = ct * P::kCols;
    tl.row0 += sub * span;
    tl.rows = min(tl.rows - sub * span, span);
    return tl.rows > 0;
  };

  // ---- the stream of slices into LDS ----
  // Wave w brings rows 32 w .. + 31 (KC) or k rows 16 (w % 4) .. + 15 of half w / 4 (KS) of
  // each operand in four loads; half w / 4 is the columns (of KS A: rows of the result)
  // from 128 on, or in a dual product the right operand b_up. KC A goes in 16 rows of half
  // w / 4 from 16 (w % 4) and from 64 + 16 (w % 4), in the order in which the products use
  // them. A of a 128-row tile is one half, brought by all waves in two loads.
  constexpr int QA = P::kTileRows / 64;  // loads of A
  const int half = wave >> 2;
  const int a_half = P::kTileRows == 256 ? half : 0;
  const int a_share = P::kTileRows == 256 ? wn : wave;  // among the waves of a half
  // (lane offsets carry everything that varies: a range check must see the whole offset)
  uint32_t a_lane[QA], b_lane[4], a_chunk = 0, b_chunk[2] = {};
  constexpr int b_bit = P::kDual ? 0 : 1;  // the bit of q that B's chunk depends on (KC)
  auto a_row = [&](int q) {  // KC: row, KS: k
    if constexpr (!P::kAKC) return 4 * QA * a_share + 4 * q + (lane >> 4);
    const int first = QA == 4 ? 128 * half + 64 * (q >> 1) + 16 * wn + 8 * (q & 1) : 16 * wave + 8 * q;
    return first + (lane >> 3);
  };
  auto b_row = [&](int q) { return P::kBKC ? 32 * wn + 8 * q + (lane >> 3) : 16 * wn + 4 * q + (lane >> 4); };
#pragma unroll
  for (int q = 0; q < QA; ++q) {
    const int r = a_row(q);
    const uint32_t chunk = static_cast<uint32_t>(P::kAKC ? (lane & 7) ^ (r & 7) : (lane & 15) ^ swizzle_a_k(r)) << 4;
    if (P::kAKC) a_chunk = chunk;
    a_lane[q] = static_cast<uint32_t>(r) * static_cast<uint32_t>(prm.lda) * S + chunk;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = b_row(q);
    const uint32_t chunk = static_cast<uint32_t>(P::kBKC ? (lane & 7) ^ swizzle_b_row<P::kDual>(r)
                                                         : (lane & 15) ^ swizzle_b_k<P::kDual>(r)) << 4;
    if (P::kBKC) b_chunk[(q >> b_bit) & 1] = chunk;
    b_lane[q] = static_cast<uint32_t>(r) * static_cast<uint32_t>(prm.ldb) * S + chunk;
  }
  // bytes between slices
  const int64_t a_slice = P::kAKC ? kSliceBytes : static_cast<int64_t>(P::kSlice) * prm.lda * S;
  const int64_t b_slice = P::kBKC ? kSliceBytes : static_cast<int64_t>(P::kSlice) * prm.ldb * S;
  const uint32_t to_a = lds0 + (P::kAKC && QA == 4 ? half * kHalfBytes + wn * 2048 : wave * (QA * 1024));
  auto a_to = [&](int q) -> uint32_t { return P::kAKC ? (q >> 1) * 8192 + (q & 1) * 1024 : q * 1024; };
  const uint32_t to_b = lds0 + P::kABytes + wave * 4096;

  Tile next;               // the tile whose slices are being loaded
  int dealt = 0;           // its round
  bool open;               // there is one
  int slice = 0;           // its slice to be loaded
  const char *a_at, *b_at;  // the slice of each operand, and the bytes to the operand's end from there
  int64_t a_left, b_left;
  int k_left;      // bytes of a row's sum from the slice on
  int k_rows = 0;  // through registers: k rows of KS operands from the slice on
  auto start_part = [&](int part) {
    const char* a = static_cast<const char*>(part == 0 ? prm.a : prm.a2);
    const char* b = static_cast<const char*>(P::kDual ? (half == 0 ? prm.b : prm.b_up) : part == 0 ? prm.b : prm.b_up);
    const int n = next.n0 + (P::kDual ? 0 : half * 128);
    if constexpr (P::kWeights) {
      const int64_t rows = __builtin_amdgcn_readfirstlane(s_off[next.e + 1] - next.first);
      const int m = next.row0 + a_half * 128;
      a_at = a + (static_cast<int64_t>(next.first) * prm.lda + m) * S;
      a_left = m < prm.M ? (rows * prm.lda - m) * S : 0;
      b_at = b + (static_cast<int64_t>(next.first) * prm.ldb + n) * S;
      b_left = n < prm.N ? (rows * prm.ldb - n) * S : 0;
      k_rows = static_cast<int>(rows);
    } else {
      a_at = a + static_cast<int64_t>(next.row0) * prm.lda * S;
      a_left = static_cast<int64_t>(next.rows) * prm.lda * S;
      if constexpr (P::kBKC) {
        b_at = b + (static_cast<int64_t>(next.e) * prm.N + n) * prm.ldb * S;
        b_left = static_cast<int64_t>(min(prm.N - n, 128)) * prm.ldb * S;
      } else {
        b_at = b + (static_cast<int64_t>(next.e) * prm.K * prm.ldb + n) * S;
        b_left = n < prm.N ? (static_cast<int64_t>(prm.K) * prm.ldb - n) * S : 0;
      }
      k_left = prm.K * S;
      k_rows = prm.K;
    }
  };
  auto start_tile = [&]() {
    open = decode(dealt, next);
    slice = 0;
    if (open) {
      start_part(0);
    } else {
      a_left = b_left = 0;
    }
  };
  auto cut = [&](uint32_t offset, uint32_t chunk) { return static_cast<int>(chunk) < k_left ? offset : kPast; };
  // (record counts in whole words do not end a KS operand exactly)
  auto cut_row = [&](uint32_t offset, int k) { return P::kDirect || k < k_rows ? offset : kPast; };
  // The wave's load q of each operand's slice. Direct: into the stage. Through registers:
  // `put` writes what the last `load` of the same q brought. Chunks of any alignment come as
  // the five aligned words that they touch, shifted together when they are put (one load of
  // 16 bytes off a word boundary takes the address unit several times as long: 6002 rows of
  // eight experts, K = 1023, F = 1535: 393 us); the last chunk of a row's sum, which a row's
  // end may cut (KC), is cleared behind it there.
  struct Held {
    i4 v;
    int more;
  };
  Held a_held[P::kDirect ? 1 : QA], b_held[P::kDirect ? 1 : 4];
  uint32_t a_skew = 0, b_skew = 0;  // of the held slice: its start past a word's,
  int k_held = 0;                   // and the bytes of a row's sum from it on
  auto load_words = [&](const char* at, int64_t left, uint32_t offset) {
    const uint32_t skew = reinterpret_cast<uintptr_t>(at) & 3;
    // (records to the end of the word that holds the operand's last element)
    const int64_t records = left <= 0 ? 0 : (left + skew + 3) & ~static_cast<int64_t>(3);
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at - skew), 0,
                                                          static_cast<int>(records < 0x7FFFFFFC ? records : 0x7FFFFFFC), kBufferFlags);
    const int from = static_cast<int>((offset + skew) & ~3U);
    Held h;
    h.v = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(buffer, from, 0, 0));
    h.more = static_cast<int>(__builtin_amdgcn_raw_buffer_load_b32(buffer, from + 16, 0, 0));
    return h;
  };
  auto joined = [&](const Held& h, uint32_t offset, uint32_t chunk, bool along_k) {
    const uint32_t shift = (offset & 3) * 8;
    i4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = static_cast<int>(__builtin_amdgcn_alignbit(static_cast<uint32_t>(i < 3 ? h.v[i < 3 ? i + 1 : 3] : h.more), static_cast<uint32_t>(h.v[i]), shift));
    }
    if (along_k && k_held < kSliceBytes) {
      const int bytes = k_held - static_cast<int>(chunk);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = bytes - 4 * i;
        o[i] = n >= 4 ? o[i] : n <= 0 ? 0 : o[i] & ((1 << (8 * n)) - 1);
      }
    }
    return o;
  };
  auto load_a = [&](uint32_t stage, int q) {
    const uint32_t offset = P::kAKC ? cut(a_lane[q], a_chunk) : cut_row(a_lane[q], a_row(q));
    if constexpr (P::kDirect) {
      load_to_lds(make_buffer(a_at, a_left), offset, to_a + stage + a_to(q));
    } else {
      a_held[q] = load_words(a_at, a_left, offset);
    }
  };
  auto load_b = [&](uint32_t stage, int q) {
    const uint32_t offset = P::kBKC ? cut(b_lane[q], b_chunk[(q >> b_bit) & 1]) : cut_row(b_lane[q], b_row(q));
    if constexpr (P::kDirect) {
      load_to_lds(make_buffer(b_at, b_left), offset, to_b + stage + q * 1024);
    } else {
      b_held[q] = load_words(b_at, b_left, offset);
    }
  };
  auto put_a = [&](uint32_t stage, int q) {
    if constexpr (!P::kDirect) {
      *reinterpret_cast<RR_LDS i4*>(to_a + stage + a_to(q) + lane * 16) = joined(a_held[q], a_lane[q] + a_skew, a_chunk, P::kAKC);
    }
  };
  auto put_b = [&](uint32_t stage, int q) {
    if constexpr (!P::kDirect) {
      *reinterpret_cast<RR_LDS i4*>(to_b + stage + q * 1024 + lane * 16) =
          joined(b_held[q], b_lane[q] + b_skew, b_chunk[(q >> b_bit) & 1], P::kBKC);
    }
  };
  auto hold = [&]() {  // notes what `put` has to know of the slice just loaded
    a_skew = reinterpret_cast<uintptr_t>(a_at) & 3;
    b_skew = reinterpret_cast<uintptr_t>(b_at) & 3;
    k_held = k_left;
  };
  auto advance = [&]() {  // to the next slice
    if constexpr (!P::kDirect) hold();
    if (!open) return;
    a_at += a_slice;
    a_left -= a_slice;
    b_at += b_slice;
    b_left -= b_slice;
    k_left -= kSliceBytes;
    k_rows -= P::kSlice;
    ++slice;
    if (slice == next.slices) {
      dealt += grid;
      start_tile();
    } else if (!P::kWeights && parts == 2 && slice == part_slices) {
      start_part(1);
    }
  };

  // ---- operand reads ----
  uint32_t b_read[2];  // per k half (KC), per fragment pair (KS)
  if constexpr (P::kBKC) {
    const int r = (P::kDual ? 32 * wn + 8 * (li >> 2) : 64 * (wn & 1) + 16 * (li >> 2)) + (li & 3);
    const uint32_t base = lds0 + P::kABytes + (P::kDual ? 0 : (wn >> 1) * kHalfBytes) + r * kSliceBytes;
#pragma unroll
    for (int h = 0; h < 2; ++h) b_read[h] = base + (static_cast<uint32_t>((4 * h + g) ^ swizzle_b_row<P::kDual>(r)) << 4);
  } else {
    const int k = 8 * g + (li >> 2);
    const uint32_t base = lds0 + P::kABytes + (P::kDual ? 0 : (wn >> 1) * kHalfBytes) + k * 256;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int chunk = P::kDual ? 4 * wn + (li & 3) : 8 * (wn & 1) + 2 * (li & 3) + v;
      b_read[v] = base + (static_cast<uint32_t>(chunk ^ swizzle_b_k<P::kDual>(k)) << 4);
    }
  }
  // fragment j (0..3; dual: gate 0, 1, up 2, 3) of k half h
  auto read_b = [&](uint32_t stage, int j, int h) -> i4 {
    if constexpr (P::kBKC) {
      return read16(b_read[h] + stage + (P::kDual ? (j >> 1) * kHalfBytes + (j & 1) * 4 * kSliceBytes : j * 4 * kSliceBytes));
    } else if constexpr (P::kDual) {
      return read_columns(b_read[0] + stage + (j >> 1) * kHalfBytes + (j & 1) * 8 + h * 32 * 256);
    } else {
      return read_columns(b_read[j >> 1] + stage + (j & 1) * 8 + h * 32 * 256);
    }
  };

  start_tile();
  if (!open) return;
  Tile tl = next;
#pragma unroll
  for (int st = 0; st < P::kStages; ++st) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q < QA) load_a(st * P::kStageBytes, q);
      load_b(st * P::kStageBytes, q);
    }
    if constexpr (!P::kDirect) hold();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q < QA) put_a(st * P::kStageBytes, q);
      put_b(st * P::kStageBytes, q);
    }
    advance();
  }
  if constexpr (P::kDirect) {
    wait_loads<(P::kStages - 1) * (QA + 4)>();
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // (the third slice, on its way)
      if (q < QA) load_a(0, q);
      load_b(0, q);
    }
    advance();
    wait_lds();
  }
  wave_barrier();
  uint32_t stage = 0;  // of the slice to be multiplied
  int round = 0;

  auto run_tile = [&](auto mi) {
    constexpr int MI = decltype(mi)::value;  // 16-row fragments of a wave
    constexpr int MA = MI < 4 ? MI : 4;      // of them in a phase
    constexpr int PH = 2 * MI / MA;          // phases of a slice: k half p % 2, fragments from MA (p / 2)
    Acc acc[MI][4] = {};
    const int wrow = wm * 16 * MI;
    uint32_t a_read[P::kAKC ? 2 : MI];
    if constexpr (P::kAKC) {
      const uint32_t base = lds0 + (wrow + li) * kSliceBytes;
#pragma unroll
      for (int h = 0; h < 2; ++h) a_read[h] = base + (static_cast<uint32_t>((4 * h + g) ^ (li & 7)) << 4);
    } else {
      const int k = 8 * g + (li >> 2);
      const uint32_t base = lds0 + (wrow >> 7) * kHalfBytes + k * 256 + (li & 1) * 8;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int chunk = ((wrow & 127) >> 3) + 2 * i + ((li & 3) >> 1);
        a_read[i] = base + (static_cast<uint32_t>(chunk ^ swizzle_a_k(k)) << 4);
      }
    }
    auto read_a = [&](uint32_t stage, int i, int h) -> i4 {
      if constexpr (P::kAKC) {
        return read16(a_read[h] + stage + i * 16 * kSliceBytes);
      } else {
        return read_columns(a_read[i] + stage + h * 32 * 256);
      }
    };
    i4 a[2][MA], b[2][4];  // of this phase and the next, of both k halves
    // the operands of phase p, in two parts
    auto fetch = [&](uint32_t stage, int p, int part) {
      const int h = p % 2, i0 = MA * (p / 2);
      if (p < 2) {
#pragma unroll
        for (int j = 2 * part; j < 2 * part + 2; ++j) b[h][j] = read_b(stage, j, h);
      }
#pragma unroll
      for (int i = part * (MA / 2); i < (part + 1) * (MA / 2); ++i) a[p & 1][i] = read_a(stage, i0 + i, h);
    };
    fetch(stage, 0, 0);
    fetch(stage, 0, 1);
    // A slice takes PH phases of MA x 4 products, each under the fetch of the next one's
    // operands. Before its last phase the slice has been read whole by every wave and the
    // next slice, loaded since that point of the slice before, has landed: a barrier, then
    // the next slice's operands are fetched and the slice after it is loaded into the stage
    // that came free. Of four phases the second no longer reads B of the slice nor, KC, the
    // first half of A's rows: a barrier there frees them half a slice earlier, and the loads
    // spread over three phases (all loads at once take the address unit, 28 cycles each,
    // longer than a phase's products).
    constexpr bool kSpread = P::kDirect && PH == 4;
    auto a_phase = [](int q) { return kSpread && P::kAKC && q < 2 ? 2 : PH - 1; };
    auto b_phase = [](int q) { return !kSpread ? PH - 1 : q < (P::kAKC ? 3 : 2) ? 1 : 2; };
#pragma unroll 1
    for (int kt = 0; kt < tl.slices; ++kt) {
      const bool last = kt + 1 == tl.slices;  // (the next tile fetches its own operands)
      const uint32_t st = stage;
#pragma unroll
      for (int p = 0; p < PH; ++p) {
        const int h = p % 2, i0 = MA * (p / 2);
        if (p == PH - 1 || (kSpread && p == 1)) {
          wait_lds();
          if constexpr (P::kDirect) {
            if (p == PH - 1) wait_loads<kSpread ? (P::kAKC ? 6 : 4) : (P::kStages - 2) * (QA + 4)>();  // the next slice's
          }
          wave_barrier();
          if (p == PH - 1) stage = stage == (P::kStages - 1) * P::kStageBytes ? 0 : stage + P::kStageBytes;
        }
#pragma unroll
        for (int i = 0; i < MA; ++i) {
          if (i < 2) {
            if (p < PH - 1) {
              fetch(stage, p + 1, i);
            } else if (!last) {
              fetch(stage, 0, i);
            }
          }
#pragma unroll
          for (int q = i * 4 / MA; q < (i + 1) * 4 / MA; ++q) {
            if (q < QA && p == a_phase(q)) put_a(st, q);
            if (p == b_phase(q)) put_b(st, q);
            if (q < QA && p == a_phase(q)) load_a(st, q);
            if (p == b_phase(q)) load_b(st, q);
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i0 + i][j] = M::mul(b[h][j], a[p & 1][i], acc[i0 + i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      advance();
    }
    // lane: rows wrow + 16 i + li, 16 columns from 16 g (dual: 8 from 8 g) of the wave's
    const std::size_t row0 = (P::kWeights ? static_cast<std::size_t>(tl.e) * prm.M : 0) + tl.row0;
    const int n = tl.n0 + (P::kDual ? 32 * wn + 8 * g : 64 * wn + 16 * g);
    auto whole = [&](int col) { return S == 2 && P::kDirect ? 8 : prm.N - col; };  // (widths of 16-bit direct products are whole eights)
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = wrow + 16 * i + li;
      if (r >= tl.rows) continue;
      if constexpr (P::kDual) {
        if (n >= prm.N) continue;
        float v[8], u[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          v[q] = static_cast<float>(acc[i][q >> 2][q & 3]);
          u[q] = static_cast<float>(acc[i][2 + (q >> 2)][q & 3]);
        }
        P::Epi::template emit<8>(prm, tl.e, row0 + r, n, whole(n), v, u);
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (n + 8 * c >= prm.N) continue;
          float v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = static_cast<float>(acc[i][2 * c + (q >> 2)][q & 3]);
          P::Epi::template emit<8>(prm, tl.e, row0 + r, n + 8 * c, whole(n + 8 * c), v);
        }
      }
    }
  };

#pragma unroll 1
  for (;;) {
    if (P::kTileRows == 256 && tl.rows > 128) {
      if constexpr (P::kTileRows == 256) run_tile(std::integral_constant<int, 8>{});
    } else if (tl.rows > 64) {
      run_tile(std::integral_constant<int, 4>{});
    } else {
      run_tile(std::integral_constant<int, 2>{});
    }
    round += grid;
    if (!decode(round, tl)) break;
  }
  if constexpr (P::kDirect) wait_loads<0>();  // (the stream's last loads bring nothing, but they write LDS)
}

template <class P>
hipError_t launch(const Product& prm, hipStream_t stream) {
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(rr_expert_gemm_kernel<P>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (attr != hipSuccess) return attr;
  const long cols = (prm.N + P::kCols - 1) / P::kCols;
  const long rows = P::kWeights ? static_cast<long>(prm.experts) * ((prm.M + 63) / 64)
                                : prm.rows / 64 + std::min<long>(prm.experts, prm.rows);
  long grid = std::min<long>(cols * rows, device_cu_count());
  if (grid >= kXcds) grid = grid / kXcds * kXcds;
  const std::size_t lds = P::kStages * P::kStageBytes + 3 * static_cast<std::size_t>(prm.experts + 1) * sizeof(int32_t);
  rr_expert_gemm_kernel<P><<<dim3(static_cast<unsigned>(grid)), kThreads, lds, stream>>>(prm);
  return hipGetLastError();
}

template <typename T, bool DIRECT, int ROWS>
using GateUp = Kind<T, true, false, false, EpiGate<T>, DIRECT, ROWS>;  // x [Wg | Wu]
template <typename T, bool DIRECT, int ROWS>
using Down = Kind<T, true, false, false, EpiStore<T>, DIRECT, ROWS>;  // a Wd
template <typename T, bool DIRECT, int ROWS>
using DGateUp = Kind<T, true, true, false, EpiDGate<T>, DIRECT, ROWS>;  // dy Wd^T
template <typename T, bool DIRECT, int ROWS>
using Dx = Kind<T, true, true, false, EpiStore<T>, DIRECT, ROWS>;  // dg Wg^T + du Wu^T
template <typename T, bool DIRECT, int ROWS>
using DwPair = Kind<T, false, false, true, EpiPair<T>, DIRECT, ROWS>;  // x^T [dg | du]
template <typename T, bool DIRECT, int ROWS>
using Dw = Kind<T, false, false, true, EpiStore<T>, DIRECT, ROWS>;  // a^T dy
template <typename T, bool DIRECT, int ROWS>
using Int8 = Kind<int8_t, true, true, false, EpiInt8<T, !DIRECT>, DIRECT, ROWS>;
template <typename T, bool DIRECT, int ROWS>
using Int8Gate = Kind<int8_t, true, true, false, EpiInt8Gate<T, !DIRECT>, DIRECT, ROWS>;

// Loads straight into LDS need every row of every operand on a 16-byte boundary.
bool aligned16(std::initializer_list<const void*> pointers) {
  for (const void* p : pointers) {
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  }
  return true;
}

// Tiles of 128 rows and a third stage where an expert has 160 rows or fewer on average (int8:
// 96): fewer rows of zeros are multiplied, tiles divide better among the CUs, and slices
// that come from HBM have twice the time to land (8192 rows of 64 experts, K = 1024, N =
// 512: the four row products of a training step 166 us against 207, the gradient of Wd 39
// against 43; a forward pass of 8192 rows of 128 experts, K = 2048, F = 768, 311 us against
// 345). With more rows weights would be read again for every 128 of them (32768 rows of
// those experts: gate and up 314 us against 288; int8, K = 2048, N = 768: 8192 rows 146 us
// against 163, but 1024 rows of eight experts, K = 4096, N = 14336, 206 against 184). The
// paired weight gradients, whose tiles are mostly stores, keep 256 rows (64 us against 70).
template <typename T, bool DIRECT, template <typename, bool, int> class K>
hipError_t launch_kind(const Product& p, hipStream_t stream) {
  if constexpr (!DIRECT) {
    return launch<K<T, false, 128>>(p, stream);
  } else if constexpr (K<T, true, 256>::kWeights && K<T, true, 256>::kDual) {
    return launch<K<T, true, 256>>(p, stream);
  } else {
    constexpr long kFew = sizeof(typename K<T, true, 256>::T) == 1 ? 96 : 160;
    return p.rows <= kFew * p.experts ? launch<K<T, true, 128>>(p, stream) : launch<K<T, true, 256>>(p, stream);
  }
}

Product base_of(const FfnParams& f) {
  Product p{};
  p.offsets = f.offsets;
  p.experts = f.experts;
  p.rows = f.rows;
  p.activation = f.activation;
  return p;
}

template <typename T, bool DIRECT>
hipError_t forward(const FfnParams& f, hipStream_t stream) {
  Product p = base_of(f);
  p.a = f.x;
  p.b = f.w_gate;
  p.b_up = f.w_up;
  p.out = f.gate;
  p.out_up = f.up;
  p.out_act = f.act;
  p.N = f.inner;
  p.K = f.hidden;
  p.lda = f.hidden;
  p.ldb = f.inner;
  const bool few = expert_rows_ok(f.rows, f.experts, false);
  int splits = expert_rows_splits(f.rows, f.experts, f.inner, f.hidden);
  const hipError_t error = few ? expert_rows<T, EpiGate<T>>(p, splits > 1 ? f.parts : nullptr, splits, stream)
                               : launch_kind<T, DIRECT, GateUp>(p, stream);
  if (error != hipSuccess) return error;
  p = base_of(f);
  p.a = f.act;
  p.b = f.w_down;
  p.out = f.y;
  p.out_f32 = f.y_f32;
  p.N = f.output;
  p.K = f.inner;
  p.lda = f.inner;
  p.ldb = f.output;
  if (!few) return launch_kind<T, DIRECT, Down>(p, stream);
  splits = expert_rows_splits(f.rows, f.experts, f.output, f.inner);
  return expert_rows<T, EpiStore<T>>(p, splits > 1 ? f.parts : nullptr, splits, stream);
}

template <typename T, bool DIRECT>
hipError_t backward(const FfnParams& f, hipStream_t stream) {
  hipError_t error = hipSuccess;
  if (f.rows != 0) {
    Product p = base_of(f);
    p.a = f.dy;
    p.b = f.w_down;
    p.in = f.gate;
    p.in_up = f.up;
    p.out = f.d_gate;
    p.out_up = f.d_up;
    p.N = f.inner;
    p.K = f.output;
    p.lda = p.ldb = f.output;
    error = launch_kind<T, DIRECT, DGateUp>(p, stream);
  }
  if (error == hipSuccess && f.rows != 0 && f.dx != nullptr) {
    Product p = base_of(f);
    p.a = f.d_gate;
    p.a2 = f.d_up;
    p.b = f.w_gate;
    p.b_up = f.w_up;
    p.out = f.dx;
    p.N = f.hidden;
    p.K = f.inner;
    p.lda = p.ldb = f.inner;
    error = launch_kind<T, DIRECT, Dx>(p, stream);
  }
  if (error == hipSuccess && f.dw_gate != nullptr) {
    Product p = base_of(f);
    p.a = f.x;
    p.b = f.d_gate;
    p.b_up = f.d_up;
    p.out = f.dw_gate;
    p.out_up = f.dw_up;
    p.M = f.hidden;
    p.N = f.inner;
    p.lda = f.hidden;
    p.ldb = f.inner;
    error = launch_kind<T, DIRECT, DwPair>(p, stream);
  }
  if (error == hipSuccess && f.dw_down != nullptr) {
    Product p = base_of(f);
    p.a = f.act;
    p.b = f.dy;
    p.out = f.dw_down;
    p.M = f.inner;
    p.N = f.output;
    p.lda = f.inner;
    p.ldb = f.output;
    error = launch_kind<T, DIRECT, Dw>(p, stream);
  }
  return error;
}

template <typename T, bool DIRECT>
hipError_t int8_product(const Int8Params& f, hipStream_t stream) {
  Product p{};
  p.offsets = f.offsets;
  p.experts = f.experts;
  p.rows = f.rows;
  p.activation = f.activation;
  p.a = f.q;
  p.a2 = f.q_scale;
  p.b = f.w;
  p.b_up = f.w_up;
  p.in = f.w_scale;
  p.in_up = f.w_up_scale;
  p.out = f.y;
  p.N = f.output;
  p.K = f.hidden;
  p.lda = p.ldb = f.hidden;
  if (expert_rows_ok(f.rows, f.experts, true)) {
    return f.w_up != nullptr ? expert_rows<int8_t, EpiInt8Gate<T, true>>(p, nullptr, 1, stream)
                             : expert_rows<int8_t, EpiInt8<T, true>>(p, nullptr, 1, stream);
  }
  return f.w_up != nullptr ? launch_kind<T, DIRECT, Int8Gate>(p, stream)
                           : launch_kind<T, DIRECT, Int8>(p, stream);
}

}  // namespace

std::size_t gated_ffn_parts(int rows, int experts, int hidden, int inner, int output) {
  const std::size_t up = static_cast<std::size_t>(expert_rows_splits(rows, experts, inner, hidden));
  const std::size_t down = static_cast<std::size_t>(expert_rows_splits(rows, experts, output, inner));
  return static_cast<std::size_t>(rows) * std::max(up > 1 ? 2 * up * inner : 0, down > 1 ? down * output : 0);
}

hipError_t gated_ffn(const FfnParams& f, hipStream_t stream) {
  const bool direct =
      f.hidden % 8 == 0 && f.inner % 8 == 0 && f.output % 8 == 0 && aligned16({f.x, f.w_gate, f.w_up, f.w_down, f.act});
  if (f.bf16) return direct ? forward<bf16, true>(f, stream) : forward<bf16, false>(f, stream);
  return direct ? forward<f16, true>(f, stream) : forward<f16, false>(f, stream);
}

hipError_t gated_ffn_backward(const FfnParams& f, hipStream_t stream) {
  const bool direct = f.hidden % 8 == 0 && f.inner % 8 == 0 && f.output % 8 == 0 &&
                      aligned16({f.x, f.w_gate, f.w_up, f.w_down, f.act, f.dy, f.d_gate, f.d_up});
  if (f.bf16) return direct ? backward<bf16, true>(f, stream) : backward<bf16, false>(f, stream);
  return direct ? backward<f16, true>(f, stream) : backward<f16, false>(f, stream);
}

hipError_t int8_grouped_gemm(const Int8Params& f, hipStream_t stream) {
  // (the longest sums need the other form's epilogue)
  const bool direct = f.hidden % 16 == 0 && f.hidden != kMostInt8Hidden && aligned16({f.q, f.w, f.w_up});
  if (f.dtype == RR_DTYPE_FP32) return direct ? int8_product<float, true>(f, stream) : int8_product<float, false>(f, stream);
  if (f.dtype == RR_DTYPE_BF16) return direct ? int8_product<bf16, true>(f, stream) : int8_product<bf16, false>(f, stream);
  return direct ? int8_product<f16, true>(f, stream) : int8_product<f16, false>(f, stream);
}

}  // namespace rr::kern
