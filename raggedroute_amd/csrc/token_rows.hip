// Tokens to their experts and back, with gradients: the stable order of the routes, the rows'
// copies, their weighted sums, and the gate's gradient.
//
//   pos[r] = #{q: id_q < id_r} + #{q < r: id_q = id_r}     (ids outside 0..experts-1 left out)
//   out[t] = sum_j w[t, j] sorted[pos[t, j]]
//   d sorted[pos[r]] = w[r] dy[t],  dw[r] = <dy[t], sorted[pos[r]]>
//   dlogits[t, id_j] = w_j sum_i w_i (dw_j - dw_i)
//
// Nothing here is arithmetic to speak of: the rows are moved at the rate of HBM (65536 rows of 2048
// BF16 numbers: sorted in 59 us, 5.1 TB/s; combined in 55, 5.5; both gradients of that 99 to 114, 5.0
// to 5.8; a plain copy 5.15) and the maps take the latency of a launch or two, up to some hundred
// thousand routes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "block_device.h"
#include "launchers.h"
#include "tokens.h"
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

constexpr int kThreads = 256;

// Rows of any width, of whole pieces, or those with results past the caches: where they are
// larger than what the next kernel finds in an L2 (65536 rows of 2048 BF16 numbers: sorting 78
// -> 69 us, combining and its gradients, which read the rows again, 185 -> 165).
constexpr int kAny = 0, kWhole = 1, kStreamed = 2;
constexpr std::size_t kStreamedBytes = std::size_t{16} << 20;

// V elements of a row, any alignment that the type has; `left` of them exist.
template <typename T, int V>
struct Piece {
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec v;
  template <int MODE>
  __device__ __forceinline__ void load(const T* p, int left) {
    if (MODE != kAny || left >= V) {
      v = *reinterpret_cast<const vec*>(p);
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < left ? p[i] : static_cast<T>(0.0F);
  }
  template <int MODE>
  __device__ __forceinline__ void store(T* p, int left) const {
    if constexpr (MODE == kStreamed) {
      __builtin_nontemporal_store(v, reinterpret_cast<vec*>(p));
      return;
    }
    if (MODE != kAny || left >= V) {
      *reinterpret_cast<vec*>(p) = v;
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i < left) p[i] = v[i];
    }
  }
};

// The same elements in another type (bits are kept where it is the same).
template <typename T, typename TX, int V>
__device__ __forceinline__ Piece<T, V> converted(const Piece<TX, V>& x) {
  Piece<T, V> o;
  if constexpr (std::is_same_v<T, TX>) {
    o.v = x.v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = static_cast<T>(static_cast<float>(x.v[i]));
  }
  return o;
}

// Elements of a thread's piece: 16 bytes of the sorted rows' type.
template <typename T>
constexpr int kPiece = 16 / sizeof(T);
// Routes of a token whose positions, then rows are on their way together. Sums of up to four
// routes are held for four only, and where a thread has several whole pieces of a row, for two of
// them: BF16, top-2, the sum and its gradients, 8192 rows of 2048: 15.0, 38.9 us for eight ->
// 13.9, 27.2 for four; 8192 of 4096: 35.3, 59.5 for eight, 33.1, 52.5 for four, 31.5, 51.9 for
// four of two pieces. (Pieces of odd rows, 3001 of 4095: gradients 28.3 us by one, 32.1 by two.)
constexpr int kBatch = 8, kFewTopK = 4;

// ---- the routes' order ----

// Every route's position and the offsets, for few routes: every workgroup reads all ids. The
// first `tokens * chunks` workgroups rank the routes of a token (a wave for each in turn, 64
// ids at a time by ballots) and copy a chunk of its row; the others count the ids below every
// expert. (Rows of 2048 BF16 numbers of 128 experts, top-8: 64 routes 3.4 us, by the kernel for more
// routes 4.7; 256 routes 5.2 and 4.7, 1024 17 and 4.9.)
constexpr int kFewRoutes = 128;

template <typename TX, typename T, bool ROWS>
__global__ __launch_bounds__(kThreads) void rr_sort_few_kernel(SortParams p, int chunks) {
  __shared__ int32_t s_ids[kFewRoutes];
  __shared__ int32_t s_pos[64];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int routes = p.tokens * p.top_k;
  const int padded = (routes + 63) & ~63;
  const int token = static_cast<int>(blockIdx.x) / chunks;
  const int chunk = static_cast<int>(blockIdx.x) - token * chunks;
  for (int i = tid; i < padded; i += kThreads) {
    const int id = i < routes ? p.ids[i] : -1;
    s_ids[i] = static_cast<unsigned>(id) < static_cast<unsigned>(p.experts) ? id : -1;
  }
  __syncthreads();
  if (token >= p.tokens) {
    // ids below expert e, 256 experts a workgroup (-1 counts as none: unsigned)
    const int e0 = (static_cast<int>(blockIdx.x) - p.tokens * chunks) * kThreads;
    const int e = e0 + tid;
    int32_t below = 0;
    for (int i = 0; i < routes; ++i) below += static_cast<unsigned>(s_ids[i]) < static_cast<unsigned>(e);
    if (e <= p.experts) p.offsets[e] = below;
    if (e0 == 0 && p.sorted_route != nullptr) {
      int placed = 0;
      for (int i = 0; i < padded; i += 64) placed += __popcll(__ballot(s_ids[i + lane] >= 0));
      for (int i = placed + tid; i < routes; i += kThreads) p.sorted_route[i] = -1;
    }
    return;
  }
  const int first = token * p.top_k;
  for (int j = wave; j < p.top_k; j += kThreads / 64) {
    const int r = first + j;
    const int id = s_ids[r];
    int pos = 0;
    for (int i = 0; i < padded; i += 64) {
      const int other = s_ids[i + lane];
      const bool before = static_cast<unsigned>(other) < static_cast<unsigned>(id) || (other == id && i + lane < r);
      pos += __popcll(__ballot(before));
    }
    if (lane == 0) {
      s_pos[j] = id >= 0 ? pos : -1;
      if (chunk == 0) {
        p.route_pos[r] = id >= 0 ? pos : -1;
        if (id >= 0 && p.sorted_route != nullptr) p.sorted_route[pos] = r;
      }
    }
  }
  if constexpr (ROWS) {
    __syncthreads();
    constexpr int V = kPiece<T>;
    const int c = (chunk * kThreads + tid) * V;
    if (c >= p.hidden) return;
    Piece<TX, V> x;
    x.template load<kAny>(static_cast<const TX*>(p.x) + static_cast<std::size_t>(token) * p.hidden + c, p.hidden - c);
    const Piece<T, V> o = converted<T>(x);
    for (int j = 0; j < p.top_k; ++j) {
      if (s_pos[j] >= 0) o.template store<kAny>(static_cast<T*>(p.x_sorted) + static_cast<std::size_t>(s_pos[j]) * p.hidden + c, p.hidden - c);
    }
  }
}

// More routes: a workgroup owns the routes of some tokens. It counts the ids before its own and
// those from there on (LDS, an atomic addition for each: counts do not depend on their order),
// or, COUNTED, sums the counts of the chunks, which a launch before it made, and counts the ids of
// its own chunk alone; a scan over the experts then gives where each begins, and one wave
// ranks the workgroup's routes by ballots, 64 at a time in their order. No workgroup waits for
// another.
//  - Up to kCountedRoutes every workgroup counts all ids and copies its tokens' rows, too: one
//    launch (6002 routes of nine experts, rows of 1023: 10.5 us, in two launches 13.5; 12000 routes, rows of
//    1024 BF16 numbers: of eight experts 13.2, in three launches 14.3, of 512 13.5 and 17.5). With
//    kApartBytes of tokens or more (two thirds of it where rows are no whole pieces) the rows
//    are another launch's (FP32 to FP16, one launch and two: 8192 rows of 2048 25.1 and
//    22.6 us, 4096 51 and 43, 3001 of 7168, top-2, 39.8 and 37.3; BF16: 8192 of 2048 16.2 and 18.5,
//    of 2827 41 and 28.5, 3001 of 2827, top-2, 15.4 and 15.5), and with more than kCountedApart routes the
//    chunks' counts are, too (16384 rows of 4096 of eight experts 54.8, without 59.6).
//  - Above, the counts and the rows are other launches', the rows' a workgroup a token in the tokens'
//    order, which writes a row behind the other in every expert's segment (32768 rows of 4096 BF16
//    numbers of eight experts: 80 us; 512 workgroups that copy what they own, spread over the
//    segments, 88). Maps of 65536 routes of 128 experts 8.3 us; by workgroups that own an expert and read
//    all ids 15. A chunk is a 32nd of the routes, and a workgroup counts the ids of its own chunk up to
//    its own: past some hundred thousand routes the time grows with their square (of 1, 8, 128 and 1024
//    experts: 262144 routes 35, 15, 16 and 24 us; 2^20 407, 107, 77 and 91; 2^22 4300, 948, 512 and 538).
constexpr int kOwnedRoutes = 512;  // of a workgroup at most
constexpr int kOwners = 512;       // workgroups, or as many as routes make of kOwnedRoutes
constexpr int kCountedRoutes = 16384, kCountedApart = 8192;
constexpr std::size_t kApartBytes = std::size_t{48} << 20;
constexpr int kChunks = 32;

// Routes of a chunk: a multiple of 256, as few as make kChunks chunks or fewer.
__host__ __device__ inline int64_t chunk_routes(int64_t routes) { return (routes + kChunks * 256 - 1) / (kChunks * 256) * 256; }

// Counts in LDS lie in 2^shift copies side by side, which lanes use by turns: additions to one
// address follow each other, and of few experts many lanes have the same (maps of
// 16384 routes of one expert 31 -> 8.8 us, of eight 11.8 -> 8.6, of 32 8.9 and 8.7).
__device__ __forceinline__ int copies_shift(int experts) { return experts <= 32 ? 3 : 0; }
__device__ __forceinline__ int copy_of(int e, int shift, int tid) { return (e << shift) + (tid & ((1 << shift) - 1)); }
__device__ __forceinline__ int32_t sum_copies(const int32_t* counts, int e, int shift) {
  if (shift == 0) return counts[e];
  typedef int quad __attribute__((ext_vector_type(4)));
  const quad q = reinterpret_cast<const quad*>(counts)[2 * e] + reinterpret_cast<const quad*>(counts)[2 * e + 1];
  return q[0] + q[1] + q[2] + q[3];
}

// Adds the ids [begin, end) to the counts of LDS, `threads` at a time.
template <int THREADS>
__device__ __forceinline__ void count_ids(int32_t* counts, int shift, const int32_t* ids, int64_t begin, int64_t end, int experts, int tid) {
  constexpr int kBatchIds = 4;
  for (int64_t from = begin; from < end; from += THREADS * kBatchIds) {
    int id[kBatchIds];
#pragma unroll
    for (int i = 0; i < kBatchIds; ++i) {
      const int64_t at = from + i * THREADS + tid;
      id[i] = at < end ? ids[at] : -1;
    }
#pragma unroll
    for (int i = 0; i < kBatchIds; ++i) {
      if (static_cast<unsigned>(id[i]) < static_cast<unsigned>(experts)) atomicAdd(counts + copy_of(id[i], shift, tid), 1);
    }
  }
}

__global__ __launch_bounds__(1024) void rr_sort_count_kernel(SortParams p) {
  __shared__ __align__(16) int32_t s_counts[RR_MAX_EXPERTS];
  static_assert(RR_MAX_EXPERTS <= 1024, "a thread an expert");
  static_assert(32 << 3 <= kThreads, "the copies' counts");
  const int tid = static_cast<int>(threadIdx.x);
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k, chunk = chunk_routes(routes);
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * chunk;
  const int shift = copies_shift(p.experts);
  if (tid < p.experts << shift) s_counts[tid] = 0;
  __syncthreads();
  count_ids<1024>(s_counts, shift, p.ids, begin, begin + chunk < routes ? begin + chunk : routes, p.experts, tid);
  __syncthreads();
  if (tid < p.experts) p.counts[static_cast<int>(blockIdx.x) * p.experts + tid] = sum_copies(s_counts, tid, shift);
}

// P experts a thread.
template <typename TX, typename T, int MODE, bool COUNTED, bool ROWS, int P>
__global__ __launch_bounds__(kThreads) void rr_sort_owned_kernel(SortParams p, int owned) {
  __shared__ __align__(16) int32_t s_before[P * kThreads], s_from[P * kThreads];  // ids before the workgroup's own; from there on
  __shared__ int32_t s_wave[kThreads / 64];
  __shared__ int32_t s_pos[kOwnedRoutes];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * owned;
  const int tokens = static_cast<int>(p.tokens - t0 < owned ? p.tokens - t0 : owned);
  const int64_t r0 = t0 * p.top_k;
  const int count = tokens * p.top_k;
  const int shift = COUNTED ? 0 : copies_shift(p.experts);  // (COUNTED: no copies, a chunk's ids alone are counted)
  for (int i = tid; i < p.experts << shift; i += kThreads) s_before[i] = s_from[i] = 0;
  __syncthreads();
  if constexpr (COUNTED) {
    const int64_t chunk = chunk_routes(routes);
    const int mine = static_cast<int>(r0 / chunk), chunks = static_cast<int>((routes + chunk - 1) / chunk);
    // every expert's chunks shared among as many threads as there are for it
    const int shares = max(kThreads / p.experts, 1);
    for (int i = tid; i < shares * p.experts; i += kThreads) {
      const int e = i % p.experts, share = i / p.experts;
      int32_t before = 0, from = 0;
#pragma unroll 8
      for (int c = share; c < chunks; c += shares) {
        const int32_t n = p.counts[c * p.experts + e];
        before += c < mine ? n : 0;
        from += c < mine ? 0 : n;
      }
      atomicAdd(s_before + e, before);
      atomicAdd(s_from + e, from);
    }
    // (those of its own chunk counted as from there on so far)
    const int64_t begin = mine * chunk;
    for (int64_t at = begin + tid; at < r0; at += kThreads) {
      const int id = p.ids[at];
      if (static_cast<unsigned>(id) < static_cast<unsigned>(p.experts)) {
        atomicAdd(s_before + id, 1);
        atomicAdd(s_from + id, -1);
      }
    }
  } else {
    count_ids<kThreads>(s_before, shift, p.ids, 0, r0, p.experts, tid);
    count_ids<kThreads>(s_from, shift, p.ids, r0, routes, p.experts, tid);
  }
  __syncthreads();
  // where every expert begins, and this workgroup's first route of it
  {
    int32_t before[P], all[P], sum = 0;  // of experts P tid + 0..
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const int e = P * tid + q;
      before[q] = e < p.experts ? sum_copies(s_before, e, shift) : 0;
      all[q] = e < p.experts ? before[q] + sum_copies(s_from, e, shift) : 0;
      sum += all[q];
    }
    const int32_t through = rr::dev::wave_inclusive_scan(sum);
    if (lane == 63) s_wave[tid >> 6] = through;
    __syncthreads();
    int32_t start = through - sum;
    int32_t placed = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
      start += w < tid >> 6 ? s_wave[w] : 0;
      placed += s_wave[w];
    }
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const int e = P * tid + q;
      if (e >= p.experts) continue;
      s_before[e] = start + before[q];  // (read by all before the barrier)
      if (blockIdx.x == 0) p.offsets[e] = start;
      start += all[q];
    }
    if (blockIdx.x == 0 && tid == 0) p.offsets[p.experts] = placed;
    if (p.sorted_route != nullptr) {  // (the last entries, spread over the workgroups)
      for (int64_t i = placed + static_cast<int64_t>(blockIdx.x) * kThreads + tid; i < routes; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        p.sorted_route[i] = -1;
      }
    }
  }
  __syncthreads();
  if (tid < 64) {
    const int bits = rr::dev::bits_for(p.experts);
    for (int i = 0; i < count; i += 64) {
      const int at = i + lane;
      const int id = at < count ? p.ids[r0 + at] : -1;
      const bool valid = static_cast<unsigned>(id) < static_cast<unsigned>(p.experts);
      const uint64_t same = rr::dev::match_mask(valid ? id : 0, bits, __ballot(valid));
      const int rank = __popcll(same & rr::dev::lanemask_lt());
      int32_t pos = -1;
      if (valid) {
        pos = s_before[id] + rank;
        rr::dev::wave_lds_sync();
        if (rank == 0) s_before[id] += __popcll(same);
      }
      rr::dev::wave_lds_sync();
      if (at < count) {
        s_pos[at] = pos;
        p.route_pos[r0 + at] = pos;
        if (pos >= 0 && p.sorted_route != nullptr) p.sorted_route[pos] = static_cast<int32_t>(r0 + at);
      }
    }
  }
  if constexpr (ROWS) {
    __syncthreads();
    constexpr int V = kPiece<T>;
    const auto* x = static_cast<const TX*>(p.x);
    auto* out = static_cast<T*>(p.x_sorted);
    const std::size_t H = p.hidden;
    // Pieces of the tokens' rows in a row, several on their way together.
    constexpr int kAhead = 4;
    const int pieces = (p.hidden + V - 1) / V;
    int t = tid / pieces, c = tid % pieces;  // of the next piece
    const int t_step = kThreads / pieces, c_step = kThreads % pieces;
    while (t < tokens) {
      Piece<TX, V> piece[kAhead];
      int token[kAhead], column[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        token[k] = t;
        column[k] = c * V;
        if (t < tokens) piece[k].template load<MODE>(x + (t0 + t) * H + column[k], p.hidden - column[k]);
        t += t_step;
        c += c_step;
        if (c >= pieces) {
          c -= pieces;
          ++t;
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (token[k] >= tokens) continue;
        const Piece<T, V> o = converted<T>(piece[k]);
        for (int j = 0; j < p.top_k; ++j) {
          const int pos = s_pos[token[k] * p.top_k + j];
          if (pos >= 0) o.template store<MODE>(out + pos * H + column[k], p.hidden - column[k]);
        }
      }
    }
  }
}

// ---- rows ----

// A position of a map, or -1 where it is none of 0..routes-1.
__device__ __forceinline__ int checked(int32_t pos, int64_t routes) {
  return pos >= 0 && pos < routes ? pos : -1;
}

// The positions and weights of B routes of a token from route j0 on. Every load is on its way
// before one of them is looked at; past the last route it is loaded again and counts as none.
template <int B>
__device__ __forceinline__ void load_positions(const int32_t* of_token, int j0, int top_k, int64_t routes, int (&pos)[B]) {
#pragma unroll
  for (int j = 0; j < B; ++j) pos[j] = of_token[min(j0 + j, top_k - 1)];
#pragma unroll
  for (int j = 0; j < B; ++j) pos[j] = j0 + j < top_k ? checked(pos[j], routes) : -1;
}

template <int B>
__device__ __forceinline__ void load_weights(const float* weights, int64_t r0, int j0, int top_k, float (&w)[B]) {
#pragma unroll
  for (int j = 0; j < B; ++j) w[j] = 1.0F;
  if (weights == nullptr) return;
#pragma unroll
  for (int j = 0; j < B; ++j) w[j] = weights[r0 + min(j0 + j, top_k - 1)];
}

// G threads a token (and as many more as blockIdx.y counts, for wide rows of few tokens): its row
// read once and stored at the positions of its routes.
template <typename TX, typename T, int G, int MODE>
__global__ __launch_bounds__(kThreads) void rr_sort_rows_kernel(SortParams p) {
  constexpr int V = kPiece<T>;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (G - 1);
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  const auto* x = static_cast<const TX*>(p.x);
  auto* out = static_cast<T*>(p.x_sorted);
  const std::size_t H = p.hidden;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + tid / G; t < p.tokens;
       t += static_cast<int64_t>(gridDim.x) * (kThreads / G)) {
    for (int j0 = 0; j0 < p.top_k; j0 += kBatch) {
      int pos[kBatch];
      load_positions(p.route_pos + t * p.top_k, j0, p.top_k, routes, pos);
      for (int c = (static_cast<int>(blockIdx.y) * G + lane) * V; c < p.hidden; c += static_cast<int>(gridDim.y) * G * V) {
        Piece<TX, V> piece;
        piece.template load<MODE>(x + t * H + c, p.hidden - c);
        const Piece<T, V> o = converted<T>(piece);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (pos[j] >= 0) o.template store<MODE>(out + pos[j] * H + c, p.hidden - c);
        }
      }
    }
  }
}

// G threads a token (and as many more as blockIdx.y counts, for wide rows of few tokens): the sum of
// its routes' rows. B routes and C pieces of each are on their way together.
template <typename TY, typename T, int G, int MODE, int B, int C>
__global__ __launch_bounds__(kThreads) void rr_combine_kernel(CombineParams p) {
  constexpr int V = kPiece<T>;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (G - 1);
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  const auto* rows = static_cast<const T*>(p.sorted);
  auto* out = static_cast<TY*>(p.out);
  const std::size_t H = p.hidden;
  const int step = static_cast<int>(gridDim.y) * G * V;  // between a thread's pieces
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + tid / G; t < p.tokens;
       t += static_cast<int64_t>(gridDim.x) * (kThreads / G)) {
    for (int c0 = (static_cast<int>(blockIdx.y) * G + lane) * V; c0 < p.hidden; c0 += C * step) {
      float sum[C][V] = {};
      for (int j0 = 0; j0 < p.top_k; j0 += B) {
        int pos[B];
        float w[B];
        Piece<T, V> row[B][C];
        load_positions(p.route_pos + t * p.top_k, j0, p.top_k, routes, pos);
        load_weights(p.weights, t * p.top_k, j0, p.top_k, w);
#pragma unroll
        for (int j = 0; j < B; ++j) {
#pragma unroll
          for (int q = 0; q < C; ++q) {
            const int c = c0 + q * step;
            if (j0 + j < p.top_k && (q == 0 || c < p.hidden)) {
              row[j][q].template load<MODE>(rows + max(pos[j], 0) * H + c, p.hidden - c);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < B; ++j) {
          if (j0 + j < p.top_k && pos[j] >= 0) {
#pragma unroll
            for (int q = 0; q < C; ++q) {
#pragma unroll
              for (int i = 0; i < V; ++i) sum[q][i] = __builtin_fmaf(w[j], static_cast<float>(row[j][q].v[i]), sum[q][i]);
            }
          }
        }
      }
      // (no loop: out of a loop of one step the compiler moves the store and loses that it is nontemporal)
      auto store = [&](int q, int c) {
        Piece<TY, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = static_cast<TY>(sum[q][i]);
        o.template store<MODE>(out + t * H + c, p.hidden - c);
      };
      store(0, c0);
      if constexpr (C == 2) {
        if (c0 + step < p.hidden) store(1, c0 + step);
      }
    }
  }
}

// G threads a token: the gradients of its routes' rows and weights, B routes and C pieces of each
// together. The columns' products are added by lane, then over the lanes in a fixed order.
template <typename TY, typename T, int G, int MODE, int B, int C>
__global__ __launch_bounds__(kThreads) void rr_combine_backward_kernel(CombineParams p) {
  constexpr int V = kPiece<T>;
  __shared__ float s_dot[2][kThreads / 64][B];  // by turns
  int turn = 0;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (G - 1);
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  const auto* dy = static_cast<const TY*>(p.dy);
  const auto* rows = static_cast<const T*>(p.sorted);
  auto* back = static_cast<T*>(p.dy_sorted);
  const std::size_t H = p.hidden;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / G);
  // (every thread of a workgroup takes every turn: sums of more than a wave meet at barriers)
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * (kThreads / G); t0 < p.tokens; t0 += step) {
    const int64_t t = t0 + tid / G;
    const bool here = t < p.tokens;
    for (int j0 = 0; j0 < p.top_k; j0 += B) {
      int pos[B];
      float w[B], dot[B] = {};
      const int64_t r0 = (here ? t : 0) * p.top_k;
      load_positions(p.route_pos + r0, j0, p.top_k, here ? routes : 0, pos);
      load_weights(p.weights, r0, j0, p.top_k, w);
      for (int c0 = lane * V; here && c0 < p.hidden; c0 += C * G * V) {
        Piece<TY, V> g[C];
#pragma unroll
        for (int q = 0; q < C; ++q) {
          const int c = c0 + q * G * V;
          if (q == 0 || c < p.hidden) g[q].template load<MODE>(dy + t * H + c, p.hidden - c);
        }
        if (p.dweights != nullptr) {
          Piece<T, V> row[B][C];
#pragma unroll
          for (int j = 0; j < B; ++j) {
            if (pos[j] < 0) continue;
#pragma unroll
            for (int q = 0; q < C; ++q) {
              const int c = c0 + q * G * V;
              if (q == 0 || c < p.hidden) row[j][q].template load<MODE>(rows + pos[j] * H + c, p.hidden - c);
            }
          }
#pragma unroll
          for (int j = 0; j < B; ++j) {
            if (pos[j] < 0) continue;
#pragma unroll
            for (int q = 0; q < C; ++q) {
              if (q > 0 && c0 + q * G * V >= p.hidden) continue;
#pragma unroll
              for (int i = 0; i < V; ++i) {
                dot[j] = __builtin_fmaf(static_cast<float>(g[q].v[i]), static_cast<float>(row[j][q].v[i]), dot[j]);
              }
            }
          }
        }
        if (p.dy_sorted != nullptr) {
          auto store = [&](int j, int q, int c) {  // (as in the kernel above)
            Piece<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = static_cast<T>(w[j] * static_cast<float>(g[q].v[i]));
            o.template store<MODE>(back + pos[j] * H + c, p.hidden - c);
          };
#pragma unroll
          for (int j = 0; j < B; ++j) {
            if (pos[j] < 0) continue;
            store(j, 0, c0);
            if constexpr (C == 2) {
              if (c0 + G * V < p.hidden) store(j, 1, c0 + G * V);
            }
          }
        }
      }
      if (p.dweights == nullptr) continue;
#pragma unroll
      for (int j = 0; j < B; ++j) {
#pragma unroll
        for (int m = 1; m < (G < 64 ? G : 64); m *= 2) dot[j] += __shfl_xor(dot[j], m, 64);
      }
      if constexpr (G > 64) {
        if ((tid & 63) == 0) {
#pragma unroll
          for (int j = 0; j < B; ++j) s_dot[turn][tid >> 6][j] = dot[j];
        }
        __syncthreads();  // (the other turn's sums were read before it)
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < B; ++j) {
            dot[j] = 0.0F;
            for (int q = 0; q < G / 64; ++q) dot[j] += s_dot[turn][(tid >> 6) + q][j];
          }
        }
        turn ^= 1;
      }
      if (here && lane == 0) {
#pragma unroll
        for (int j = 0; j < B; ++j) {
          if (j0 + j < p.top_k) p.dweights[t * p.top_k + j0 + j] = pos[j] >= 0 ? dot[j] : 0.0F;
        }
      }
    }
  }
}

// A wave a token: lane j has the gradient of its route's logit, then every lane its experts'.
// Differences of the weights' gradients are taken before they are weighted: of a weight near 1
// they are what is left.
__global__ __launch_bounds__(kThreads) void rr_gate_backward_kernel(GateBackwardParams p) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6); t < p.tokens;
       t += static_cast<int64_t>(gridDim.x) * (kThreads / 64)) {
    int id = -1;
    float w = 0.0F, d = 0.0F;
    if (lane < p.top_k) {
      const int64_t r = t * p.top_k + lane;
      id = p.ids[r];
      if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.experts)) id = -1;
      if (id >= 0) {
        w = p.weights[r];
        d = p.dweights[r];
      }
    }
    float g = 0.0F;
    for (int i = 0; i < p.top_k; ++i) {
      const int other = __builtin_amdgcn_readlane(id, i);
      const float wi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), i));
      const float di = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(d), i));
      if (other >= 0) g = __builtin_fmaf(wi, d - di, g);
    }
    g *= w;
    // (every lane stays active: the others read its registers)
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
      const int e = e0 + lane;
      float sum = 0.0F;
      for (int j = 0; j < p.top_k; ++j) {
        const int other = __builtin_amdgcn_readlane(id, j);
        const float gj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), j));
        sum += other == e ? gj : 0.0F;
      }
      if (e < p.experts) p.dlogits[t * p.experts + e] = sum;
    }
  }
}

// Workgroups of `per` tokens each.
unsigned token_grid(int tokens, int per) {
  return static_cast<unsigned>(std::min<int64_t>((static_cast<int64_t>(tokens) + per - 1) / per, 16384));
}

// Workgroups that share a token's columns, for few tokens with wide rows (six tokens of 4864 FP32
// numbers, top-8, combined: 8.3 us by one each, 4.4 by five).
template <int G>
dim3 token_grid(int tokens, int hidden, int piece) {
  const unsigned x = token_grid(tokens, kThreads / G);
  const int most = (hidden + G * piece - 1) / (G * piece);
  return dim3(x, static_cast<unsigned>(std::max(1, std::min(most, static_cast<int>(1024 / x)))));
}

// Threads of a token: as many as its row has pieces, up to a workgroup's (a wave for a row of 256
// pieces: combining 65536 rows of 2048 BF16 numbers 79 us against 59, its gradients 131 against
// 115). BACKWARD: a wave up to 128 pieces, whose sums then meet at no barrier (gradients of 6002
// rows of 1023 10 us, with two waves a token 14).
// `bytes`: of the rows that are written.
template <bool BACKWARD, typename F>
hipError_t with_group(int hidden, int piece, std::size_t bytes, F f) {
  const int pieces = (hidden + piece - 1) / piece;
  auto with_mode = [&](auto g) {
    if (hidden % piece != 0) return f(g, std::integral_constant<int, kAny>{});
    if constexpr (decltype(g)::value >= 64) {
      if (bytes >= kStreamedBytes) return f(g, std::integral_constant<int, kStreamed>{});
    }
    return f(g, std::integral_constant<int, kWhole>{});
  };
  if (pieces <= 8) return with_mode(std::integral_constant<int, 8>{});
  if (pieces <= 16) return with_mode(std::integral_constant<int, 16>{});
  if (pieces <= 32) return with_mode(std::integral_constant<int, 32>{});
  if (pieces <= (BACKWARD ? 128 : 64)) return with_mode(std::integral_constant<int, 64>{});
  if constexpr (!BACKWARD) {
    if (pieces <= 128) return with_mode(std::integral_constant<int, 128>{});
  }
  return with_mode(std::integral_constant<int, 256>{});
}

template <typename TX, typename T>
hipError_t sort_rows(const SortParams& p, hipStream_t stream) {
  const std::size_t bytes = sizeof(T) * p.tokens * p.top_k * p.hidden;
  return with_group<false>(p.hidden, kPiece<T>, bytes, [&](auto g, auto mode) {
    constexpr int G = decltype(g)::value;
    // (whole rows of more than 64 pieces that have this launch are more than kStreamedBytes: they are
    // more than kCountedRoutes, or kApartBytes of tokens, which 16 bits halve)
    static_assert((kCountedRoutes + 1) * std::size_t{65 * 16} >= kStreamedBytes && kApartBytes / 2 >= kStreamedBytes);
    constexpr int M = G > 64 && decltype(mode)::value == kWhole ? kStreamed : decltype(mode)::value;
    rr_sort_rows_kernel<TX, T, G, M><<<token_grid<G>(p.tokens, p.hidden, kPiece<T>), kThreads, 0, stream>>>(p);
    return hipGetLastError();
  });
}

template <typename TX, typename T, int P>
hipError_t sort_owned(const SortParams& p, hipStream_t stream) {
  const int64_t tokens = p.tokens, routes = tokens * p.top_k;
  const int owned = static_cast<int>(std::min<int64_t>((tokens + kOwners - 1) / kOwners, kOwnedRoutes / p.top_k));
  const unsigned grid = static_cast<unsigned>((tokens + owned - 1) / owned);
  const bool whole = p.hidden % kPiece<T> == 0;
  const bool large = p.x_sorted != nullptr && sizeof(TX) * tokens * p.hidden >= (whole ? kApartBytes : kApartBytes / 3 * 2);
  const bool counted = routes > (large ? kCountedApart : kCountedRoutes);
  const bool apart = counted || large;
  if (p.x_sorted == nullptr || apart) {
    if (counted) {
      const int64_t chunk = chunk_routes(routes);
      rr_sort_count_kernel<<<static_cast<unsigned>((routes + chunk - 1) / chunk), 1024, 0, stream>>>(p);
      const hipError_t error = hipGetLastError();
      if (error != hipSuccess) return error;
      rr_sort_owned_kernel<TX, T, kAny, true, false, P><<<grid, kThreads, 0, stream>>>(p, owned);
    } else {
      rr_sort_owned_kernel<TX, T, kAny, false, false, P><<<grid, kThreads, 0, stream>>>(p, owned);
    }
    const hipError_t error = hipGetLastError();
    return error != hipSuccess || p.x_sorted == nullptr ? error : sort_rows<TX, T>(p, stream);
  }
  if (!whole) {
    rr_sort_owned_kernel<TX, T, kAny, false, true, P><<<grid, kThreads, 0, stream>>>(p, owned);
  } else if (sizeof(T) * routes * p.hidden < kStreamedBytes) {
    rr_sort_owned_kernel<TX, T, kWhole, false, true, P><<<grid, kThreads, 0, stream>>>(p, owned);
  } else {
    rr_sort_owned_kernel<TX, T, kStreamed, false, true, P><<<grid, kThreads, 0, stream>>>(p, owned);
  }
  return hipGetLastError();
}

template <typename TX, typename T>
hipError_t sort_typed(const SortParams& p, hipStream_t stream) {
  if (static_cast<int64_t>(p.tokens) * p.top_k > kFewRoutes) {
    static_assert(RR_MAX_EXPERTS <= 4 * kThreads);
    return p.experts <= kThreads ? sort_owned<TX, T, 1>(p, stream) : sort_owned<TX, T, 4>(p, stream);
  }
  const int counters = (p.experts + 1 + kThreads - 1) / kThreads;
  if (p.x_sorted == nullptr) {
    rr_sort_few_kernel<TX, T, false><<<p.tokens + counters, kThreads, 0, stream>>>(p, 1);
  } else {
    const int chunks = (p.hidden + kThreads * kPiece<T> - 1) / (kThreads * kPiece<T>);
    rr_sort_few_kernel<TX, T, true><<<p.tokens * chunks + counters, kThreads, 0, stream>>>(p, chunks);
  }
  return hipGetLastError();
}

template <typename TY, typename T>
hipError_t combine_typed(const CombineParams& p, hipStream_t stream) {
  return with_group<false>(p.hidden, kPiece<T>, sizeof(TY) * p.tokens * p.hidden, [&](auto g, auto mode) {
    constexpr int G = decltype(g)::value;
    constexpr int M = decltype(mode)::value;
    const dim3 grid = token_grid<G>(p.tokens, p.hidden, kPiece<T>);
    if constexpr (M != kAny && G == kThreads) {  // (of fewer threads each has one piece)
      if (p.top_k <= kFewTopK && static_cast<std::size_t>(p.hidden) > static_cast<std::size_t>(grid.y) * G * kPiece<T>) {
        rr_combine_kernel<TY, T, G, M, kFewTopK, 2><<<grid, kThreads, 0, stream>>>(p);
        return hipGetLastError();
      }
    }
    if (p.top_k <= kFewTopK) {
      rr_combine_kernel<TY, T, G, M, kFewTopK, 1><<<grid, kThreads, 0, stream>>>(p);
    } else {
      rr_combine_kernel<TY, T, G, M, kBatch, 1><<<grid, kThreads, 0, stream>>>(p);
    }
    return hipGetLastError();
  });
}

template <typename TY, typename T>
hipError_t backward_typed(const CombineParams& p, hipStream_t stream) {
  return with_group<true>(p.hidden, kPiece<T>, sizeof(T) * p.tokens * p.top_k * p.hidden, [&](auto g, auto mode) {
    constexpr int G = decltype(g)::value;
    constexpr int M = decltype(mode)::value;
    const unsigned grid = token_grid(p.tokens, kThreads / G);
    if constexpr (M != kAny && G >= 64) {  // (of fewer threads each has one piece)
      if (p.top_k <= kFewTopK && p.hidden > G * kPiece<T>) {
        rr_combine_backward_kernel<TY, T, G, M, kFewTopK, 2><<<grid, kThreads, 0, stream>>>(p);
        return hipGetLastError();
      }
    }
    if (p.top_k <= kFewTopK) {
      rr_combine_backward_kernel<TY, T, G, M, kFewTopK, 1><<<grid, kThreads, 0, stream>>>(p);
    } else {
      rr_combine_backward_kernel<TY, T, G, M, kBatch, 1><<<grid, kThreads, 0, stream>>>(p);
    }
    return hipGetLastError();
  });
}

}  // namespace

std::size_t sort_tokens_counts(int64_t routes, int experts) {
  return routes > kCountedApart ? static_cast<std::size_t>(kChunks) * experts : 0;
}

hipError_t sort_tokens(const SortParams& p, hipStream_t stream) {
  if (p.dtype == RR_DTYPE_FP32) return sort_typed<float, float>(p, stream);
  if (p.dtype == RR_DTYPE_BF16) return p.x_f32 ? sort_typed<float, bf16>(p, stream) : sort_typed<bf16, bf16>(p, stream);
  return p.x_f32 ? sort_typed<float, f16>(p, stream) : sort_typed<f16, f16>(p, stream);
}

hipError_t combine_tokens(const CombineParams& p, hipStream_t stream) {
  if (p.dtype == RR_DTYPE_FP32) return combine_typed<float, float>(p, stream);
  if (p.dtype == RR_DTYPE_BF16) return p.tokens_f32 ? combine_typed<float, bf16>(p, stream) : combine_typed<bf16, bf16>(p, stream);
  return p.tokens_f32 ? combine_typed<float, f16>(p, stream) : combine_typed<f16, f16>(p, stream);
}

hipError_t combine_tokens_backward(const CombineParams& p, hipStream_t stream) {
  if (p.dtype == RR_DTYPE_FP32) return backward_typed<float, float>(p, stream);
  if (p.dtype == RR_DTYPE_BF16) return p.tokens_f32 ? backward_typed<float, bf16>(p, stream) : backward_typed<bf16, bf16>(p, stream);
  return p.tokens_f32 ? backward_typed<float, f16>(p, stream) : backward_typed<f16, f16>(p, stream);
}

hipError_t topk_gate_backward(const GateBackwardParams& p, hipStream_t stream) {
  rr_gate_backward_kernel<<<token_grid(p.tokens, kThreads / 64), kThreads, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace rr::kern
