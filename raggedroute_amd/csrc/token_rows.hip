// Tokens to their experts and back, with gradients: the stable order of the routes, the rows'
// copies, their weighted sums, and the gate's gradient.
//
//   pos[r] = #{q: id_q < id_r} + #{q < r: id_q = id_r}     (ids outside 0..experts-1 left out)
//   out[t] = sum_j w[t, j] sorted[pos[t, j]]
//   d sorted[pos[r]] = w[r] dy[t],  dw[r] = <dy[t], sorted[pos[r]]>
//   dlogits[t, id_j] = w_j sum_i w_i (dw_j - dw_i)
//
// Nothing here is arithmetic to speak of: the rows are moved at the rate of HBM and the maps
// take the latency of a launch or two.
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

// V elements of a row, any alignment that the type has; `left` of them exist.
template <typename T, int V>
struct Piece {
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec v;
  __device__ __forceinline__ void load(const T* p, int left) {
    if (left >= V) {
      v = *reinterpret_cast<const vec*>(p);
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < left ? p[i] : static_cast<T>(0.0F);
  }
  __device__ __forceinline__ void store(T* p, int left) const {
    if (left >= V) {
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
constexpr int kBatch = 8;  // routes of a token whose positions are loaded together

// ---- the routes' order ----

// Every route's position and the offsets, for few routes: every workgroup reads all ids. The
// first `tokens * chunks` workgroups rank the routes of a token (a wave for each in turn, 64
// ids at a time by ballots) and copy a chunk of its row; the others count the ids below every
// expert.
constexpr int kFewRoutes = 1024;

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
    x.load(static_cast<const TX*>(p.x) + static_cast<std::size_t>(token) * p.hidden + c, p.hidden - c);
    const Piece<T, V> o = converted<T>(x);
    for (int j = 0; j < p.top_k; ++j) {
      if (s_pos[j] >= 0) o.store(static_cast<T*>(p.x_sorted) + static_cast<std::size_t>(s_pos[j]) * p.hidden + c, p.hidden - c);
    }
  }
}

// Any number of routes: a workgroup owns G experts and reads all ids twice, its 16 waves a
// contiguous share each, four ids a lane. The first pass counts the ids below the workgroup's
// experts and those of each; the second gives the routes of its experts their positions. No
// workgroup waits for another and nothing is added atomically.
constexpr int kRankWaves = 16;

template <int G>
__global__ __launch_bounds__(64 * kRankWaves) void rr_sort_rank_kernel(SortParams p) {
  __shared__ int32_t s_count[G + 1][kRankWaves];  // of a wave's ids: [0] below, [1 + g] of expert e0 + g
  typedef int quad __attribute__((ext_vector_type(4), aligned(4)));
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int e0 = static_cast<int>(blockIdx.x) * G;
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  const int64_t share = ((routes + kRankWaves * 256 - 1) / (kRankWaves * 256)) * 256;
  const int64_t begin = share * wave, end = begin + share < routes ? begin + share : routes;
  // (an id that is none of 0..experts-1 becomes -1: as an unsigned number above all)
  auto load = [&](int64_t at) {
    quad v;
    const int64_t left = end - at;
    if (left >= 4) {
      v = *reinterpret_cast<const quad*>(p.ids + at);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = i < left ? p.ids[at + i] : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<unsigned>(v[i]) < static_cast<unsigned>(p.experts) ? v[i] : -1;
    return v;
  };
  int32_t below = 0, mine[G] = {};
  for (int64_t at = begin + 4 * lane; at - 4 * lane < end; at += 256) {
    const quad v = load(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      below += __popcll(__ballot(static_cast<unsigned>(v[i]) < static_cast<unsigned>(e0)));
#pragma unroll
      for (int g = 0; g < G; ++g) mine[g] += __popcll(__ballot(v[i] == e0 + g));
    }
  }
  if (lane == 0) {
    s_count[0][wave] = below;
#pragma unroll
    for (int g = 0; g < G; ++g) s_count[1 + g][wave] = mine[g];
  }
  __syncthreads();
  // where expert e0 + g begins, and this wave's first route of it
  int32_t start = 0, at_wave[G];
  for (int w = 0; w < kRankWaves; ++w) start += s_count[0][w];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    at_wave[g] = start;
    int32_t all = 0;
    for (int w = 0; w < kRankWaves; ++w) {
      if (w < wave) at_wave[g] += s_count[1 + g][w];
      all += s_count[1 + g][w];
    }
    if (tid == 0 && e0 + g < p.experts) p.offsets[e0 + g] = start;
    start += all;
  }
  if (e0 + G >= p.experts) {  // the last workgroup: start is the number of placed routes
    if (tid == 0) p.offsets[p.experts] = start;
    if (p.sorted_route != nullptr) {
      for (int64_t i = start + tid; i < routes; i += 64 * kRankWaves) p.sorted_route[i] = -1;
    }
  }
  for (int64_t at = begin + 4 * lane; at - 4 * lane < end; at += 256) {
    const quad v = load(at);
    auto place = [&](int i, int32_t pos) {
      const int64_t r = at + i;
      if (r >= end) return;
      p.route_pos[r] = pos;
      if (pos >= 0 && p.sorted_route != nullptr) p.sorted_route[pos] = static_cast<int32_t>(r);
    };
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint64_t m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = __ballot(v[i] == e0 + g);
      if ((m[0] | m[1] | m[2] | m[3]) == 0) continue;
      int32_t pos = at_wave[g];
      const uint64_t lower = rr::dev::lanemask_lt();
#pragma unroll
      for (int i = 0; i < 4; ++i) pos += __popcll(m[i] & lower);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (v[i] == e0 + g) place(i, pos++);
        at_wave[g] += __popcll(m[i]);
      }
    }
    if (blockIdx.x == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (v[i] < 0) place(i, -1);
      }
    }
  }
}

// ---- rows ----

// A position of a map, or -1 where it is none of 0..routes-1.
__device__ __forceinline__ int checked(int32_t pos, int64_t routes) {
  return pos >= 0 && pos < routes ? pos : -1;
}

// G threads a token: its row read once and stored at the positions of its routes.
template <typename TX, typename T, int G>
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
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        pos[j] = j0 + j < p.top_k ? checked(p.route_pos[t * p.top_k + j0 + j], routes) : -1;
      }
      for (int c = lane * V; c < p.hidden; c += G * V) {
        Piece<TX, V> piece;
        piece.load(x + t * H + c, p.hidden - c);
        const Piece<T, V> o = converted<T>(piece);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (pos[j] >= 0) o.store(out + pos[j] * H + c, p.hidden - c);
        }
      }
    }
  }
}

// G threads a token: the sum of its routes' rows.
template <typename TY, typename T, int G>
__global__ __launch_bounds__(kThreads) void rr_combine_kernel(CombineParams p) {
  constexpr int V = kPiece<T>;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (G - 1);
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  const auto* rows = static_cast<const T*>(p.sorted);
  auto* out = static_cast<TY*>(p.out);
  const std::size_t H = p.hidden;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + tid / G; t < p.tokens;
       t += static_cast<int64_t>(gridDim.x) * (kThreads / G)) {
    for (int c = lane * V; c < p.hidden; c += G * V) {
      float sum[V] = {};
      for (int j0 = 0; j0 < p.top_k; j0 += kBatch) {
        int pos[kBatch];
        float w[kBatch];
        Piece<T, V> row[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int64_t r = t * p.top_k + j0 + j;
          pos[j] = j0 + j < p.top_k ? checked(p.route_pos[r], routes) : -1;
          w[j] = p.weights != nullptr && j0 + j < p.top_k ? p.weights[r] : 1.0F;
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (j0 + j < p.top_k) row[j].load(rows + max(pos[j], 0) * H + c, p.hidden - c);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (j0 + j < p.top_k && pos[j] >= 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = __builtin_fmaf(w[j], static_cast<float>(row[j].v[i]), sum[i]);
          }
        }
      }
      Piece<TY, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = static_cast<TY>(sum[i]);
      o.store(out + t * H + c, p.hidden - c);
    }
  }
}

// G threads a token: the gradients of its routes' rows and weights. The columns' products are
// added by lane, then over the lanes in a fixed order.
template <typename TY, typename T, int G>
__global__ __launch_bounds__(kThreads) void rr_combine_backward_kernel(CombineParams p) {
  constexpr int V = kPiece<T>;
  __shared__ float s_dot[kThreads / 64][kBatch];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (G - 1);
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  const auto* dy = static_cast<const TY*>(p.dy);
  const auto* rows = static_cast<const T*>(p.sorted);
  auto* back = static_cast<T*>(p.dy_sorted);
  const std::size_t H = p.hidden;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / G);
  // (every thread of a workgroup takes every turn: the sums of G = 256 meet at barriers)
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * (kThreads / G); t0 < p.tokens; t0 += step) {
    const int64_t t = t0 + tid / G;
    const bool here = t < p.tokens;
    for (int j0 = 0; j0 < p.top_k; j0 += kBatch) {
      int pos[kBatch];
      float w[kBatch], dot[kBatch] = {};
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int64_t r = t * p.top_k + j0 + j;
        const bool is = here && j0 + j < p.top_k;
        pos[j] = is ? checked(p.route_pos[r], routes) : -1;
        w[j] = is && p.weights != nullptr ? p.weights[r] : 1.0F;
      }
      for (int c = lane * V; here && c < p.hidden; c += G * V) {
        Piece<TY, V> g;
        g.load(dy + t * H + c, p.hidden - c);
        if (p.dweights != nullptr) {
          Piece<T, V> row[kBatch];
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            if (pos[j] >= 0) row[j].load(rows + pos[j] * H + c, p.hidden - c);
          }
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            if (pos[j] < 0) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) dot[j] = __builtin_fmaf(static_cast<float>(g.v[i]), static_cast<float>(row[j].v[i]), dot[j]);
          }
        }
        if (p.dy_sorted != nullptr) {
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            if (pos[j] < 0) continue;
            Piece<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = static_cast<T>(w[j] * static_cast<float>(g.v[i]));
            o.store(back + pos[j] * H + c, p.hidden - c);
          }
        }
      }
      if (p.dweights == nullptr) continue;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
#pragma unroll
        for (int m = 1; m < (G < 64 ? G : 64); m *= 2) dot[j] += __shfl_xor(dot[j], m, 64);
      }
      if constexpr (G > 64) {
        if ((tid & 63) == 0) {
#pragma unroll
          for (int j = 0; j < kBatch; ++j) s_dot[tid >> 6][j] = dot[j];
        }
        __syncthreads();
        if (tid == 0) {
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            dot[j] = 0.0F;
            for (int q = 0; q < kThreads / 64; ++q) dot[j] += s_dot[q][j];
          }
        }
        __syncthreads();
      }
      if (here && lane == 0) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
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

// Threads of a token: as many as its row has pieces, up to a wave.
template <typename F>
hipError_t with_group(int hidden, int piece, F f) {
  const int pieces = (hidden + piece - 1) / piece;
  if (pieces <= 8) return f(std::integral_constant<int, 8>{});
  if (pieces <= 16) return f(std::integral_constant<int, 16>{});
  if (pieces <= 32) return f(std::integral_constant<int, 32>{});
  if (pieces <= 64) return f(std::integral_constant<int, 64>{});
  return f(std::integral_constant<int, 256>{});
}

template <typename TX, typename T>
hipError_t sort_typed(const SortParams& p, hipStream_t stream) {
  const int64_t routes = static_cast<int64_t>(p.tokens) * p.top_k;
  if (routes <= kFewRoutes) {
    const int counters = (p.experts + 1 + kThreads - 1) / kThreads;
    if (p.x_sorted == nullptr) {
      rr_sort_few_kernel<TX, T, false><<<p.tokens + counters, kThreads, 0, stream>>>(p, 1);
    } else {
      const int chunks = (p.hidden + kThreads * kPiece<T> - 1) / (kThreads * kPiece<T>);
      rr_sort_few_kernel<TX, T, true><<<p.tokens * chunks + counters, kThreads, 0, stream>>>(p, chunks);
    }
    return hipGetLastError();
  }
  if (p.experts <= 256) {
    rr_sort_rank_kernel<1><<<p.experts, 64 * kRankWaves, 0, stream>>>(p);
  } else {
    rr_sort_rank_kernel<4><<<(p.experts + 3) / 4, 64 * kRankWaves, 0, stream>>>(p);
  }
  const hipError_t error = hipGetLastError();
  if (error != hipSuccess || p.x_sorted == nullptr) return error;
  return with_group(p.hidden, kPiece<T>, [&](auto g) {
    constexpr int G = decltype(g)::value;
    rr_sort_rows_kernel<TX, T, G><<<token_grid(p.tokens, kThreads / G), kThreads, 0, stream>>>(p);
    return hipGetLastError();
  });
}

template <typename TY, typename T>
hipError_t combine_typed(const CombineParams& p, hipStream_t stream) {
  return with_group(p.hidden, kPiece<T>, [&](auto g) {
    constexpr int G = decltype(g)::value;
    rr_combine_kernel<TY, T, G><<<token_grid(p.tokens, kThreads / G), kThreads, 0, stream>>>(p);
    return hipGetLastError();
  });
}

template <typename TY, typename T>
hipError_t backward_typed(const CombineParams& p, hipStream_t stream) {
  return with_group(p.hidden, kPiece<T>, [&](auto g) {
    constexpr int G = decltype(g)::value;
    rr_combine_backward_kernel<TY, T, G><<<token_grid(p.tokens, kThreads / G), kThreads, 0, stream>>>(p);
    return hipGetLastError();
  });
}

}  // namespace

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
