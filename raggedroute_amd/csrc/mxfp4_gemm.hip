// Grouped products of 4-bit rows and weights with a power of two for every 32 elements:
// 256-column tiles of 256 or 128 rows on v_mfma_scale_f32_32x32x64_f8f6f4, sums in FP32.
//
//   C[r, n] = sum over blocks b of 2^(Xa[r, b] + Xw[n, b]) sum over k of A[r, k] W[n, k]
//
// The instruction takes 16 bytes a lane of each operand, 32 elements and thus one block, and a
// scale a lane, so that the products need nothing beside it: it multiplies twice what the
// int8 instruction does of as many bytes in the same time. The stream of slices is that of
// the other expert products (expert_gemm.hip): one workgroup of eight waves a CU, slices of
// 128 bytes (256 elements, eight blocks) of every row of both operands straight from memory into
// LDS, that many slices ahead of the products and across the end of a tile. A slice's scales
// (eight bytes a row, side by side in memory) come the same way, a word a lane.
//  - Lane group g (of 32 lanes) multiplies blocks 4 g .. 4 g + 3 of a slice, so that its four
//    scales are one register, of which the instruction's selector takes a byte.
//  - The weights are the instruction's first operand and their rows are dealt to its 32 so
//    that a lane ends with 16 adjacent columns of a row.
//  - Scales of blocks past the row's last, whatever their bytes are, are replaced by 0 on both
//    sides: the elements there, the next row's, then add 2^-254 times 36 at most, nothing.
//
// What bounds it: large products the power that the instructions draw, LDS, which is read and
// written as long as they run (264 KB a slice), and the slices' loads (16384 rows of eight experts, K =
// 4096, N = 14336: 555 us = 3.5 PFLOP/s; without its loads 438, without its LDS reads, too, 379, of
// which the stores of 470 MB are 70); small ones the prologue and the epilogue of one or two
// tiles a CU (6002 rows of nine experts, K = 1023, N = 1535, gated: 30 us, at K = 64 21).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "expert_gemm.h"
#include "large_lds.h"
#include "launchers.h"
#include "mxfp4.h"
#include "mxfp4_rows.h"
#include "tile_stream.h"
#include "tiles.h"
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kThreads = 512;
constexpr int kScaleBytes = 8;  // of a row's slice

// A kernel: epilogue and rows of a tile. Tiles of 128 rows leave room for a third stage.
template <class Epi_, int ROWS>
struct MxKind {
  using Epi = Epi_;
  static constexpr bool kDual = Epi_::kDual;
  static constexpr int kTileRows = ROWS;
  static constexpr int kStages = ROWS == 128 ? 3 : 2;
  static constexpr int kABytes = ROWS * kSliceBytes;
  static constexpr int kBBytes = kTileCols * kSliceBytes;
  static constexpr int kAScales = kABytes + kBBytes;  // A's scales in a stage, then B's
  static constexpr int kBScales = kAScales + ROWS * kScaleBytes;
  static constexpr int kStageBytes = kBScales + kTileCols * kScaleBytes;
  static constexpr int kCols = kDual ? kTileCols / 2 : kTileCols;
  static_assert(kStageBytes % kSliceBytes == 0, "a chunk's number is bits 4 to 6 of its LDS address");
};

// Column of a fragment's row m: the sums of rows 8 i + 4 g + r are registers 4 i + r of lane group g.
__device__ __forceinline__ int dealt_column(int m) { return ((m >> 2) & 1) << 4 | (m >> 3) << 2 | (m & 3); }

// Chunk permutation of a weight row's eight chunks: the rows that lanes read together differ
// in the bits used.
__device__ __forceinline__ int swizzle_b(int r) { return ((r >> 1) & 3) | ((r >> 4) & 1) << 2; }

// BYTE: which of the scales' counts.
template <int BYTE>
__device__ __forceinline__ f16v multiply(i4 a, i4 b, f16v c, int a_scale, int b_scale) {
  typedef int i8 __attribute__((ext_vector_type(8)));
  const i8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  constexpr int kE2M1 = 4;
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, kE2M1, kE2M1, BYTE, a_scale, BYTE, b_scale);
}

__device__ __forceinline__ int read_word(uint32_t at) { return *reinterpret_cast<RR_LDS const int*>(at); }

// An output tile (uniform).
struct MxTile {
  int e;           // expert
  int row0, rows;  // first row and rows
  int n0;          // first column
};

// p.a, p.b, p.b_up: packed rows, lda = ldb: bytes between them. p.in, p.in_up: scales of the
// weights, p.a2: of the rows. p.K: blocks of a row.
template <class P>
__global__ __launch_bounds__(kThreads, 2) void rr_mxfp4_gemm_kernel(Product prm) {
  extern __shared__ __align__(128) char smem[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((RR_LDS char*)smem));
  int32_t* s_off = reinterpret_cast<int32_t*>(smem + P::kStages * P::kStageBytes);  // [E + 1]
  int32_t* s_pre = s_off + prm.experts + 1;                             // [E + 1] full row tiles before expert e
  int32_t* s_pre2 = s_pre + prm.experts + 1;                            // [E + 1] short row tiles before expert e
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int li = lane & 31, g = lane >> 5;
  const int experts = prm.experts;

  for (int e = tid; e <= experts; e += kThreads) s_off[e] = rr::dev::offset_at(prm.offsets, e, prm.rows);
  __syncthreads();
  if (wave == 0) {
    raise_offsets(s_off, experts, lane);
    build_tile_prefix<P::kTileRows, true>(s_off, s_pre, s_pre2, experts, lane);
  }
  __syncthreads();
  const int col_tiles = (prm.N + P::kCols - 1) / P::kCols;
  const int full_rows = __builtin_amdgcn_readfirstlane(s_pre[experts]);
  const int short_rows = __builtin_amdgcn_readfirstlane(s_pre2[experts]);
  const int total_full = full_rows * col_tiles;
  const int total = total_full + short_rows * col_tiles;
  const int grid = static_cast<int>(gridDim.x);
  const int worker = tile_worker(static_cast<int>(blockIdx.x), grid);
  const int slices = (prm.K + 7) / 8;

  // Tiles in rounds of the grid, the last partial one cut, as in expert_gemm.hip.
  const int whole_rounds = total / grid * grid;
  const bool mixed = whole_rounds != 0 && total_full < whole_rounds && total_full > whole_rounds - grid;
  auto decode = [&](int dealt, MxTile& tl) {
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
    const bool is_short = t >= total_full;
    const int32_t* pre = is_short ? s_pre2 : s_pre;
    if (is_short) t -= total_full;
    tl.e = __builtin_amdgcn_readfirstlane(tile_expert(pre, experts, t / col_tiles));
    const int before = __builtin_amdgcn_readfirstlane(pre[tl.e]);
    int rt, ct;
    place_tile(t - before * col_tiles, __builtin_amdgcn_readfirstlane(pre[tl.e + 1]) - before, col_tiles, &rt, &ct);
    const int first = __builtin_amdgcn_readfirstlane(s_off[tl.e]);
    const int end = __builtin_amdgcn_readfirstlane(s_off[tl.e + 1]);
    tl.row0 = first + (is_short ? (end - first) / P::kTileRows : rt) * P::kTileRows;
    tl.rows = min(end - tl.row0, P::kTileRows);
    tl.n0 = ct * P::kCols;
    tl.row0 += sub * span;
    tl.rows = min(tl.rows - sub * span, span);
    return tl.rows > 0;
  };

  // ---- the stream of slices into LDS ----
  // Wave w brings rows 32 w .. + 31 of B in four loads (half w / 4 is the columns from 128 on, or
  // in a dual product the weights b_up), 16 rows of half w / 4 of A from 16 (w % 4) and from 64 +
  // 16 (w % 4), in the order in which the products use them (a tile of 128 rows: rows 16 w .. + 15
  // in two loads), and the scales of rows 32 w .. + 31 of each (of A's 128: of 16 w .. + 15) in one
  // load each.
  constexpr int QA = P::kTileRows / 64;  // loads of A
  constexpr int kLoads = QA + 6;         // of a slice
  const int half = wave >> 2;
  // Lane offsets inside eight rows; which eight is the buffer's start.
  uint32_t a_lane, b_lane[2];
  const int64_t row_bytes = prm.lda;
  {
    const int r = lane >> 3;
    a_lane = static_cast<uint32_t>(r * prm.lda) + (static_cast<uint32_t>((lane & 7) ^ r) << 4);
#pragma unroll
    for (int q = 0; q < 2; ++q) b_lane[q] = static_cast<uint32_t>(r * prm.lda) + (static_cast<uint32_t>((lane & 7) ^ swizzle_b(16 * q + r)) << 4);
  }
  const int a_first = QA == 4 ? 128 * half + 16 * wn : 16 * wave;  // the wave's first rows
  const int b_first = 32 * wn;
  const uint32_t a_scale_lane = static_cast<uint32_t>((QA == 4 ? 32 : 16) * wave * kScaleBytes + lane * 4);
  const uint32_t b_scale_lane = static_cast<uint32_t>(32 * wn * kScaleBytes + lane * 4);
  const uint32_t to_a = lds0 + (QA == 4 ? half * kHalfBytes + wn * 2048 : wave * 2048);
  auto a_to = [](int q) -> uint32_t { return (q >> 1) * 8192 + (q & 1) * 1024; };
  const uint32_t to_b = lds0 + P::kABytes + wave * 4096;
  const uint32_t to_a_scale = lds0 + P::kAScales + (QA == 4 ? 32 : 16) * wave * kScaleBytes;
  const uint32_t to_b_scale = lds0 + P::kBScales + 32 * wave * kScaleBytes;

  MxTile next;          // the tile whose slices are being loaded
  int dealt = 0;        // its round
  bool open;            // there is one
  int slice = 0;        // its slice to be loaded
  const char *a_at, *b_at, *as_at, *bs_at;  // the slice of each operand, and the bytes to the operand's end from there
  int64_t a_left, b_left;
  int as_left, bs_left;
  const int64_t a_scale_slice = static_cast<int64_t>(prm.rows) * kScaleBytes;  // bytes between slices
  const int64_t b_scale_slice = static_cast<int64_t>(experts) * prm.N * kScaleBytes;
  auto start_tile = [&]() {
    open = decode(dealt, next);
    slice = 0;
    if (!open) {
      a_left = b_left = as_left = bs_left = 0;
      return;
    }
    const char* b = static_cast<const char*>(P::kDual && half != 0 ? prm.b_up : prm.b);
    const char* bs = static_cast<const char*>(P::kDual && half != 0 ? prm.in_up : prm.in);
    const int n = next.n0 + (P::kDual ? 0 : half * 128);
    const int64_t channel = static_cast<int64_t>(next.e) * prm.N + n;
    const int columns = min(prm.N - n, 128);
    a_at = static_cast<const char*>(prm.a) + static_cast<int64_t>(next.row0) * prm.lda;
    a_left = static_cast<int64_t>(next.rows) * prm.lda;
    as_at = static_cast<const char*>(prm.a2) + static_cast<int64_t>(next.row0) * kScaleBytes;
    as_left = next.rows * kScaleBytes;
    b_at = b + channel * prm.lda;
    b_left = static_cast<int64_t>(columns) * prm.lda;
    bs_at = bs + channel * kScaleBytes;
    bs_left = columns * kScaleBytes;
  };
  // (what lies past a row's end in its last slice is the next row's: its scales count as 2^-127)
  auto load_a = [&](uint32_t stage, int q) {
    const int64_t from = (a_first + 64 * (q >> 1) + 8 * (q & 1)) * row_bytes;
    load_to_lds(make_buffer(a_at + from, a_left - from), a_lane, to_a + stage + a_to(q));
  };
  auto load_b = [&](uint32_t stage, int q) {
    const int64_t from = (b_first + 8 * q) * row_bytes;
    load_to_lds(make_buffer(b_at + from, b_left - from), b_lane[q >> 1], to_b + stage + q * 1024);
  };
  auto load_scales = [&](uint32_t stage) {
    if (QA == 4 || lane < 32) load_words_to_lds(make_buffer(as_at, as_left), a_scale_lane, to_a_scale + stage);
    load_words_to_lds(make_buffer(bs_at, bs_left), b_scale_lane, to_b_scale + stage);
  };
  auto advance = [&]() {  // to the next slice
    if (!open) return;
    a_at += kSliceBytes;
    a_left -= kSliceBytes;
    b_at += kSliceBytes;
    b_left -= kSliceBytes;
    as_at += a_scale_slice;
    bs_at += b_scale_slice;
    ++slice;
    if (slice == slices) {
      dealt += grid;
      start_tile();
    }
  };

  // ---- operand reads ----
  uint32_t b_read;  // block 4 g; t blocks further: the address ^ (t << 4)
  uint32_t b_scale;
  {
    const int r = (P::kDual ? 32 * wn : 64 * (wn & 1)) + dealt_column(li);
    const uint32_t base = lds0 + P::kABytes + (P::kDual ? 0 : (wn >> 1) * kHalfBytes) + r * kSliceBytes;
    b_read = base + (static_cast<uint32_t>((4 * g) ^ swizzle_b(r)) << 4);
    b_scale = lds0 + P::kBScales + (r + (P::kDual ? 0 : (wn >> 1) * 128)) * kScaleBytes + 4 * g;
  }
  // fragment j (dual: of gate, of up)
  auto read_b = [&](uint32_t stage, int j, int t) -> i4 {
    return read16(((b_read + stage) ^ (t << 4)) + j * (P::kDual ? kHalfBytes : 32 * kSliceBytes));
  };
  auto read_b_scale = [&](uint32_t stage, int j) { return read_word(b_scale + stage + j * (P::kDual ? 128 : 32) * kScaleBytes); };

  start_tile();
  if (!open) return;
  MxTile tl = next;
#pragma unroll
  for (int st = 0; st < P::kStages; ++st) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q < QA) load_a(st * P::kStageBytes, q);
      load_b(st * P::kStageBytes, q);
    }
    load_scales(st * P::kStageBytes);
    advance();
  }
  wait_loads<(P::kStages - 1) * kLoads>();
  wave_barrier();
  uint32_t stage = 0;  // of the slice to be multiplied
  int round = 0;

  auto run_tile = [&](auto mi) {
    constexpr int MI = decltype(mi)::value;  // 32-row fragments of a wave
    constexpr int MA = MI < 2 ? MI : 2;      // of them in a phase
    constexpr int PH = 2 * MI / MA;          // phases of a slice: blocks 2 (p % 2) and one more, fragments from MA (p / 2)
    constexpr int U = 2 * MA;                // pairs of products of a phase
    f16v acc[MI][2] = {};
    const int wrow = wm * 32 * MI;
    const uint32_t a_read = lds0 + (wrow + li) * kSliceBytes + (static_cast<uint32_t>((4 * g) ^ (li & 7)) << 4);
    const uint32_t a_scale = lds0 + P::kAScales + (wrow + li) * kScaleBytes + 4 * g;
    i4 a[2][U], b[4][2];  // a of this phase and the next, b of the slice (the next one's from the last phase on)
    int as[2][MA], bs[2][2];  // scales: [0] in use, [1] fetched for the next fragments and the next slice
    int k_blocks = prm.K;     // of a row from the slice on that is multiplied
    auto mask_of = [&](int blocks) {
      const int n = blocks - 4 * g;
      return n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
    };
    int mask = mask_of(k_blocks);
    // the operands of phase p, in two parts
    auto fetch = [&](uint32_t stage, int p, int part) {
      const int t = 2 * (p % 2) + part, i0 = MA * (p / 2);
      if (p < 2) {
#pragma unroll
        for (int j = 0; j < 2; ++j) b[t][j] = read_b(stage, j, t);
        if (p == 0) bs[1][part] = read_b_scale(stage, part);
      }
#pragma unroll
      for (int i = 0; i < MA; ++i) {
        a[p & 1][part * MA + i] = read16(((a_read + stage) ^ (t << 4)) + (i0 + i) * 32 * kSliceBytes);
        if (p % 2 == 0 && part == 0) as[1][i] = read_word(a_scale + stage + (i0 + i) * 32 * kScaleBytes);
      }
    };
    fetch(stage, 0, 0);
    fetch(stage, 0, 1);
    // The phases of a slice, its barriers and its loads are those of expert_gemm.hip; the
    // scales of the slice after the next are loaded in the last phase, when those of this one
    // have been read.
    constexpr bool kSpread = PH == 4;
    auto a_phase = [](int q) { return kSpread && q < 2 ? 2 : PH - 1; };
    auto b_phase = [](int q) { return !kSpread ? PH - 1 : q < 3 ? 1 : 2; };
#pragma unroll 1
    for (int kt = 0; kt < slices; ++kt) {
      const bool last = kt + 1 == slices;  // (the next tile fetches its own operands)
      const uint32_t st = stage;
#pragma unroll
      for (int p = 0; p < PH; ++p) {
        const int i0 = MA * (p / 2);
        if (p == 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) bs[0][j] = bs[1][j] & mask;
        }
        if (p % 2 == 0) {
#pragma unroll
          for (int i = 0; i < MA; ++i) as[0][i] = as[1][i] & mask;
        }
        if (p == PH - 1 || (kSpread && p == 1)) {
          wait_lds();
          if (p == PH - 1) wait_loads<kSpread ? 6 : (P::kStages - 2) * kLoads>();  // the next slice's
          wave_barrier();
          if (p == PH - 1) stage = stage == (P::kStages - 1) * P::kStageBytes ? 0 : stage + P::kStageBytes;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u < 2) {
            if (p < PH - 1) {
              fetch(stage, p + 1, u);
            } else if (!last) {
              fetch(stage, 0, u);
            }
          }
#pragma unroll
          for (int q = u * 4 / U; q < (u + 1) * 4 / U; ++q) {
            if (q < QA && p == a_phase(q)) load_a(st, q);
            if (p == b_phase(q)) load_b(st, q);
            if (q == 3 && p == PH - 1) load_scales(st);
          }
          __builtin_amdgcn_sched_barrier(0);
          const int i = i0 + u % MA;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const i4 w = b[2 * (p % 2) + u / MA][j], x = a[p & 1][u];
            const int ws = bs[0][j], xs = as[0][u % MA];
            if (p % 2 == 0) {
              acc[i][j] = u / MA == 0 ? multiply<0>(w, x, acc[i][j], ws, xs) : multiply<1>(w, x, acc[i][j], ws, xs);
            } else {
              acc[i][j] = u / MA == 0 ? multiply<2>(w, x, acc[i][j], ws, xs) : multiply<3>(w, x, acc[i][j], ws, xs);
            }
            // (the compiler takes these products for pure and would move them all behind the
            // slice's loads, with their operands in registers until then)
            asm volatile("" : "+v"(acc[i][j]));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      k_blocks -= 8;
      mask = mask_of(k_blocks);
      advance();
    }
    // lane: rows wrow + 32 i + li, 16 columns from 16 g of each fragment's 32
    const std::size_t row0 = tl.row0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = wrow + 32 * i + li;
      if (r >= tl.rows) continue;
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // eight columns of both operands, or 16 of a fragment
        if constexpr (P::kDual) {
          const int n = tl.n0 + 32 * wn + 16 * g + 8 * c;
          if (n >= prm.N) continue;
          float v[8], u[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            v[q] = acc[i][0][8 * c + q];
            u[q] = acc[i][1][8 * c + q];
          }
          P::Epi::template emit<8>(prm, tl.e, row0 + r, n, prm.N - n, v, u);
        } else {
          const int n = tl.n0 + 64 * wn + 32 * c + 16 * g;
          if (n >= prm.N) continue;
          float v[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) v[q] = acc[i][c][q];
          P::Epi::template emit<16>(prm, tl.e, row0 + r, n, prm.N - n, v);
        }
      }
    }
  };

#pragma unroll 1
  for (;;) {
    if (P::kTileRows == 256 && tl.rows > 128) {
      if constexpr (P::kTileRows == 256) run_tile(std::integral_constant<int, 4>{});
    } else if (tl.rows > 64) {
      run_tile(std::integral_constant<int, 2>{});
    } else {
      run_tile(std::integral_constant<int, 1>{});
    }
    round += grid;
    if (!decode(round, tl)) break;
  }
  wait_loads<0>();  // (the stream's last loads bring nothing, but they write LDS)
}

template <class P>
hipError_t launch(const Product& prm, hipStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  const hipError_t error = allow_lds(reinterpret_cast<const void*>(rr_mxfp4_gemm_kernel<P>), 160 * 1024, &allowed);
  if (error != hipSuccess) return error;
  const long cols = (prm.N + P::kCols - 1) / P::kCols;
  const long rows = prm.rows / 64 + std::min<long>(prm.experts, prm.rows);
  long grid = std::min<long>(cols * rows, device_cu_count());
  if (grid >= kXcds) grid = grid / kXcds * kXcds;
  const std::size_t lds = P::kStages * P::kStageBytes + 3 * static_cast<std::size_t>(prm.experts + 1) * sizeof(int32_t);
  rr_mxfp4_gemm_kernel<P><<<dim3(static_cast<unsigned>(grid)), kThreads, lds, stream>>>(prm);
  return hipGetLastError();
}

template <class Epi>
hipError_t product(const Product& prm, hipStream_t stream) {
  if (mxfp4_rows_ok(prm, Epi::kDual)) return mxfp4_rows<Epi>(prm, stream);
  // (the LDS that three stages leave holds the bounds of 596 experts)
  constexpr int kMost = (160 * 1024 - MxKind<Epi, 128>::kStages * MxKind<Epi, 128>::kStageBytes) / (3 * static_cast<int>(sizeof(int32_t))) - 1;
  static_assert(kMost >= 512);
  static_assert(MxKind<Epi, 256>::kStages * MxKind<Epi, 256>::kStageBytes + 3 * (RR_MAX_EXPERTS + 1) * sizeof(int32_t) <= 160 * 1024);
  // Tiles of 128 rows where an expert has 128 rows or fewer on average (E = 128, K = 2048, N = 768,
  // gated: 16384 rows 75 us, on tiles of 256 rows 82; E = 8, K = N = 4096: 1024 rows 25.8 and 27.8, but N
  // = 14336 82 and 78; 2048 rows of those 117 and 108).
  const bool few = prm.rows <= 128L * prm.experts && prm.experts <= kMost;
  return few ? launch<MxKind<Epi, 128>>(prm, stream) : launch<MxKind<Epi, 256>>(prm, stream);
}

template <typename T>
hipError_t typed(const MxGemmParams& f, hipStream_t stream) {
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
  p.N = f.output;
  p.K = mx_blocks(f.hidden);
  p.lda = p.ldb = 16 * p.K;
  if (f.w_up != nullptr) {
    p.out_act = f.y;
    return product<EpiMxGate<T>>(p, stream);
  }
  p.out = f.y;
  return product<EpiMxStore<T>>(p, stream);
}

}  // namespace

hipError_t mxfp4_grouped_gemm(const MxGemmParams& f, hipStream_t stream) {
  if (f.dtype == RR_DTYPE_FP32) return typed<float>(f, stream);
  if (f.dtype == RR_DTYPE_BF16) return typed<bf16>(f, stream);
  return typed<f16>(f, stream);
}

}  // namespace rr::kern
