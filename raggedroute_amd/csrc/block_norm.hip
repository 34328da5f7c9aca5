// Norms around a block with gate and residual scale, their gradients, and the
// quantisation of rows to 8-bit integers (formulas: raggedroute_capi.h).
//
// All three are bound by memory: a row is read once into registers, its sums of
// squares and products are reduced over the G threads that share it, and its results
// are written from the same registers. Columns: thread t of a row's G holds
// V-element (16-byte) chunks t, t + G, ...; the last chunk of a row is cut element by
// element, so rows of any width and alignment take one path (a row that starts off a
// 16-byte boundary only splits its accesses over cache lines).
//
// BF16 rows of 4096, each tensor once: 16384 rows forward (x, block, h, n) 100 us = 5.4 TB/s;
// 8192 rows backward (h, block, dh, dn, dx, dblock) 87 us = 4.7 TB/s and 7 us for the
// columns' sums; a copy of that size reaches 4.75 TB/s. Quantisation, 16384 rows: 70 us = 2.9
// TB/s, with one row on its way in a workgroup. The backward pass of rows past 512 threads (BF16 8192
// values, FP32 4096) is bound by registers: 1024 threads have 128 each and keep 130 to 390
// bytes a thread in memory (4096 rows of 12288 in BF16 1080 us = 0.6 TB/s; 8192 rows of 8192
// 169 us), and rows past those (16384, 8192) are read again for every pass, an element at a
// time (4096 rows of 20480 forward 0.8 ms, backward 3.5).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "block.h"
#include "block_device.h"
#include "wave.h"

namespace rr::kern {
namespace {

using rr::dev::bf16;
using rr::dev::f16;

template <typename T>
constexpr int kChunk = 16 / sizeof(T);  // elements a thread loads at once

// V values of type T, FP32 in use.
template <typename T, int V>
struct Raw {
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec v;
  // elements [0, n) of p; 0 past them
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= V) {
      v = *reinterpret_cast<const vec*>(p);
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < n ? p[i] : static_cast<T>(0.0F);
  }
  __device__ __forceinline__ void store(T* p, int n) const {
    if (n >= V) {
      *reinterpret_cast<vec*>(p) = v;
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i < n) p[i] = v[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return static_cast<float>(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = static_cast<T>(x); }
};

// Sums of M values over the G threads of a workgroup, in a fixed order; every thread gets
// them. `slot` alternates between calls, so that one barrier a call is enough.
template <int G, int M>
__device__ __forceinline__ void reduce(float (&v)[M], float* lds, int slot) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += __shfl_xor(v[m], off, 64);
  }
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    float* at = lds + slot * W * M;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int m = 0; m < M; ++m) at[(threadIdx.x >> 6) * M + m] = v[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float s = 0.0F;
#pragma unroll
      for (int w = 0; w < W; ++w) s += at[w * M + m];
      v[m] = s;
    }
  }
}

// 1 / sqrt(v) for v > 0. v_rsq_f32 takes a subnormal v (eps may be one) for 0.
__device__ __forceinline__ float inverse_root(float v) {
  const bool small = v < 0x1p-100F;
  const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p64F : v);
  return small ? r * 0x1p32F : r;
}

template <int G, int M>
constexpr int kReduceFloats = G > 64 ? 2 * (G / 64) * M : 1;

// Calls f(c, col, left) for each of a thread's NV chunks that begins inside the row: its
// first column and the columns from there to the row's end.
template <int V, int G, int NV, typename F>
__device__ __forceinline__ void for_chunks(int D, F f) {
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int col = V * (static_cast<int>(threadIdx.x) + c * G);
    if (col < D) f(c, col, D - col);
  }
}

// The workgroup's row after `row`, `rows` where there is none (a sum of the two may pass 31 bits).
__device__ __forceinline__ int next_row(int row, int rows) {
  const int step = static_cast<int>(gridDim.x);
  return rows - row > step ? row + step : rows;
}

template <typename T, typename TB, int G, int NV>
__global__ __launch_bounds__(G) void rr_block_norm_kernel(NormParams p) {
  constexpr int V = kChunk<T>;
  __shared__ float lds[kReduceFloats<G, 1>];
  const int D = p.hidden;
  const float inv = 1.0F / static_cast<float>(D);
  const auto* x = static_cast<const T*>(p.x);
  const auto* block = static_cast<const TB*>(p.block);
  const auto* gate = static_cast<const T*>(p.gate);
  const bool post = p.post_weight != nullptr;
  Raw<T, V> wpost[NV], wpre[NV];
  for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
    if (post) wpost[c].load(static_cast<const T*>(p.post_weight) + col, left);
    if (p.n != nullptr) wpre[c].load(static_cast<const T*>(p.pre_weight) + col, left);
  });
  Raw<T, V> rx[NV], rg[NV];
  Raw<TB, V> rb[NV];
  auto fetch = [&](int t) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      rx[c].load(x + row + col, left);
      if (block != nullptr) {
        rb[c].load(block + row + col, left);
        if (gate != nullptr) rg[c].load(gate + static_cast<std::size_t>(t / p.gate_tokens) * D + col, left);
      }
    });
  };
  int t = static_cast<int>(blockIdx.x);
  if (t < p.tokens) fetch(t);
  for (; t < p.tokens; t = next_row(t, p.tokens)) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    float h[NV][V];
    float scale = p.scale;
    if (block != nullptr && post) {
      float ss[1] = {0.0F};
      for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
        for (int i = 0; i < V; ++i) ss[0] = __builtin_fmaf(rb[c][i], rb[c][i], ss[0]);
      });
      reduce<G>(ss, lds, 0);
      scale *= inverse_root(__builtin_fmaf(ss[0], inv, p.eps));
    }
    float ss[1] = {0.0F};
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      for (int i = 0; i < V; ++i) {
        float v = rx[c][i];
        if (block != nullptr) {
          float b = rb[c][i] * scale;
          if (post) b *= wpost[c][i];
          v = __builtin_fmaf(gate != nullptr ? rg[c][i] : 1.0F, b, v);
        }
        h[c][i] = v;
        ss[0] = __builtin_fmaf(v, v, ss[0]);
      }
    });
    const int next = next_row(t, p.tokens);
    if (next < p.tokens) fetch(next);
    if (p.h != nullptr) {
      for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
        Raw<T, V> out;
        for (int i = 0; i < V; ++i) out.set(i, h[c][i]);
        out.store(static_cast<T*>(p.h) + row + col, left);
      });
    }
    if (p.n != nullptr) {
      reduce<G>(ss, lds, 1);
      const float r = inverse_root(__builtin_fmaf(ss[0], inv, p.eps));
      for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
        Raw<T, V> out;
        for (int i = 0; i < V; ++i) out.set(i, h[c][i] * r * wpre[c][i]);
        out.store(static_cast<T*>(p.n) + row + col, left);
      });
    }
    if constexpr (G > 64) __syncthreads();  // the slots are free again
  }
}

// Rows wider than the registers: the row is read again for every pass.
template <typename T, typename TB>
__global__ __launch_bounds__(1024) void rr_block_norm_wide_kernel(NormParams p) {
  constexpr int G = 1024;
  __shared__ float lds[kReduceFloats<G, 1>];
  const int D = p.hidden;
  const float inv = 1.0F / static_cast<float>(D);
  const auto* block = static_cast<const TB*>(p.block);
  const auto* wpost = static_cast<const T*>(p.post_weight);
  for (int t = static_cast<int>(blockIdx.x); t < p.tokens; t = next_row(t, p.tokens)) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    const T* gate = p.gate != nullptr ? static_cast<const T*>(p.gate) + static_cast<std::size_t>(t / p.gate_tokens) * D : nullptr;
    float scale = p.scale;
    if (block != nullptr && wpost != nullptr) {
      float ss[1] = {0.0F};
      for (int col = threadIdx.x; col < D; col += G) {
        const float b = static_cast<float>(block[row + col]);
        ss[0] = __builtin_fmaf(b, b, ss[0]);
      }
      reduce<G>(ss, lds, 0);
      scale *= inverse_root(__builtin_fmaf(ss[0], inv, p.eps));
    }
    auto value = [&](int col) {
      float v = static_cast<float>(static_cast<const T*>(p.x)[row + col]);
      if (block != nullptr) {
        float b = static_cast<float>(block[row + col]) * scale;
        if (wpost != nullptr) b *= static_cast<float>(wpost[col]);
        v = __builtin_fmaf(gate != nullptr ? static_cast<float>(gate[col]) : 1.0F, b, v);
      }
      return v;
    };
    float r = 0.0F;
    if (p.n != nullptr) {
      float ss[1] = {0.0F};
      for (int col = threadIdx.x; col < D; col += G) {
        const float v = value(col);
        ss[0] = __builtin_fmaf(v, v, ss[0]);
      }
      reduce<G>(ss, lds, 1);
      r = inverse_root(__builtin_fmaf(ss[0], inv, p.eps));
    }
    for (int col = threadIdx.x; col < D; col += G) {
      const float v = value(col);  // (before h, which may be x)
      if (p.h != nullptr) static_cast<T*>(p.h)[row + col] = static_cast<T>(v);
      if (p.n != nullptr) {
        static_cast<T*>(p.n)[row + col] = static_cast<T>(v * r * static_cast<float>(static_cast<const T*>(p.pre_weight)[col]));
      }
    }
    __syncthreads();
  }
}

// How the tokens are dealt to workgroups for the column sums. A part is a run of
// tokens. Gate rows of many tokens are split into `per_group` parts each, whose gate
// gradients are added up afterwards; a part of short gate rows holds whole ones and
// writes their gradients itself. Without a gate all tokens are one group.
struct Parts {
  int count, tokens;  // parts, tokens in a part
  int group;          // tokens of a gate row
  int per_group;      // parts of a gate row (0: parts hold whole gate rows)
};

constexpr int kSumThreads = 131072;  // threads of all parts together, about eight waves a CU

// (counts of tokens go up to 2^31 - 1: sums of two of them, and a part's place in a gate row
// that ends early, pass 31 bits)
Parts make_parts(const NormParams& p, int threads) {
  Parts s{};
  if (p.tokens == 0) return s;
  auto divide = [](int64_t a, int64_t by) { return static_cast<int>((a + by - 1) / by); };
  const int want = std::max(1, divide(static_cast<int64_t>(p.tokens) * threads, kSumThreads));
  s.group = p.gate != nullptr ? std::min(p.gate_tokens, p.tokens) : p.tokens;
  if (s.group >= want) {
    s.tokens = divide(s.group, divide(s.group, want));
    s.per_group = divide(s.group, s.tokens);
    s.count = divide(p.tokens, s.group) * s.per_group;
  } else {
    s.tokens = want / s.group * s.group;
    s.count = divide(p.tokens, s.tokens);
  }
  return s;
}

// First and one past the last token of a part (a part of a short last gate row may be empty).
__device__ __forceinline__ void part_range(const Parts& s, int tokens, int part, int* first, int* end) {
  int64_t from, stop;
  if (s.per_group != 0) {
    const int g = part / s.per_group;
    from = static_cast<int64_t>(g) * s.group + static_cast<int64_t>(part - g * s.per_group) * s.tokens;
    stop = min(static_cast<int64_t>(g + 1) * s.group, from + s.tokens);
  } else {
    from = static_cast<int64_t>(part) * s.tokens;
    stop = from + s.tokens;
  }
  *end = static_cast<int>(min(stop, static_cast<int64_t>(tokens)));
  *first = static_cast<int>(min(from, static_cast<int64_t>(*end)));
}

// Column sums of part `part`: [0] pre_weight, [1] post_weight, [2] gate.
__device__ __forceinline__ float* part_sums(const NormParams& p, int part, int which) {
  return p.sums + (static_cast<std::size_t>(part) * 3 + which) * p.hidden;
}

template <typename T, typename TB, int G, int NV>
__global__ __launch_bounds__(G) void rr_block_norm_backward_kernel(NormParams p, Parts parts) {
  constexpr int V = kChunk<T>;
  __shared__ float lds[kReduceFloats<G, 3>];
  __shared__ float lds2[kReduceFloats<G, 1>];
  const int D = p.hidden;
  const float inv = 1.0F / static_cast<float>(D);
  const auto* h = static_cast<const T*>(p.x);
  const auto* block = static_cast<const TB*>(p.block);
  const auto* gate = static_cast<const T*>(p.gate);
  const auto* dh = static_cast<const T*>(p.dh);
  const auto* dn = static_cast<const T*>(p.dn);
  const bool post = p.post_weight != nullptr;
  Raw<T, V> wpost[NV], wpre[NV];
  for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
    if (post) wpost[c].load(static_cast<const T*>(p.post_weight) + col, left);
    if (dn != nullptr) wpre[c].load(static_cast<const T*>(p.pre_weight) + col, left);
  });
  float spre[NV][V] = {}, spost[NV][V] = {}, sgate[NV][V] = {};
  // The next row is on its way while one is worked on (1024 threads have no registers for
  // it, nor for all of the present one).
  constexpr bool kAhead = G < 1024;
  Raw<T, V> rh[NV], rdh[NV], rdn[NV], rg[NV], next_h[NV], next_dh[NV], next_dn[NV];
  Raw<TB, V> rb[NV], next_b[NV];
  auto fetch = [&](int t) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      next_h[c].load(h + row + col, left);
      if (dh != nullptr) next_dh[c].load(dh + row + col, left);
      if (dn != nullptr) next_dn[c].load(dn + row + col, left);
      if (block != nullptr) next_b[c].load(block + row + col, left);
    });
  };
  auto fetch_gate = [&](int t) {
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      rg[c].load(gate + static_cast<std::size_t>(t / p.gate_tokens) * D + col, left);
    });
  };
  int first, end;
  part_range(parts, p.tokens, static_cast<int>(blockIdx.x), &first, &end);
  if (first < end) {
    if (kAhead) fetch(first);
    if (gate != nullptr) fetch_gate(first);
  }
  int until_gate = parts.group;  // tokens to the next gate row, in parts of whole ones
  for (int t = first; t < end; ++t) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    if (!kAhead) fetch(t);
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      rh[c] = next_h[c];
      rdh[c] = next_dh[c];
      rdn[c] = next_dn[c];
      rb[c] = next_b[c];
    }
    if (kAhead && t + 1 < end) fetch(t + 1);
    float s[3] = {0.0F, 0.0F, 0.0F};  // h^2, dn pre_weight h, block^2
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      for (int i = 0; i < V; ++i) {
        s[0] = __builtin_fmaf(rh[c][i], rh[c][i], s[0]);
        if (dn != nullptr) s[1] = __builtin_fmaf(rdn[c][i] * wpre[c][i], rh[c][i], s[1]);
        if (post) s[2] = __builtin_fmaf(rb[c][i], rb[c][i], s[2]);
      }
    });
    reduce<G>(s, lds, 0);
    const float r = inverse_root(__builtin_fmaf(s[0], inv, p.eps));
    const float back = s[1] * inv * r * r;  // mean(dn pre_weight h) / rms^2
    const float rb_scale = post ? inverse_root(__builtin_fmaf(s[2], inv, p.eps)) : 1.0F;
    float dx[NV][V];
    float s2[1] = {0.0F};  // db post_weight block
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      Raw<T, V> out;
      for (int i = 0; i < V; ++i) {
        float v = dh != nullptr ? rdh[c][i] : 0.0F;
        if (dn != nullptr) {
          v += r * (rdn[c][i] * wpre[c][i] - rh[c][i] * back);
          spre[c][i] = __builtin_fmaf(rdn[c][i], rh[c][i] * r, spre[c][i]);
        }
        out.set(i, v);
        if (block != nullptr) {
          v *= p.scale;  // gradient of gate * N(block)
          const float unit = rb[c][i] * rb_scale;
          const float normed = post ? unit * wpost[c][i] : unit;
          sgate[c][i] = __builtin_fmaf(v, normed, sgate[c][i]);
          if (gate != nullptr) v *= rg[c][i];
          if (post) {
            spost[c][i] = __builtin_fmaf(v, unit, spost[c][i]);
            v *= wpost[c][i];
            s2[0] = __builtin_fmaf(v, unit, s2[0]);
          }
        }
        dx[c][i] = v;
      }
      out.store(static_cast<T*>(p.dx) + row + col, left);
    });
    if (block != nullptr && p.dblock != nullptr) {
      float back2 = 0.0F;
      if (post) {
        reduce<G>(s2, lds2, 0);
        back2 = s2[0] * inv;
      }
      for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
        Raw<TB, V> out;
        for (int i = 0; i < V; ++i) {
          out.set(i, post ? rb_scale * (dx[c][i] - rb[c][i] * rb_scale * back2) : dx[c][i]);
        }
        out.store(static_cast<TB*>(p.dblock) + row + col, left);
      });
    }
    if (gate != nullptr && parts.per_group == 0 && (--until_gate == 0 || t + 1 == end)) {
      until_gate = parts.group;
      if (p.dgate != nullptr) {
        for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
          Raw<T, V> out;
          for (int i = 0; i < V; ++i) {
            out.set(i, sgate[c][i]);
            sgate[c][i] = 0.0F;
          }
          out.store(static_cast<T*>(p.dgate) + static_cast<std::size_t>(t / p.gate_tokens) * D + col, left);
        });
      }
      if (t + 1 < end) fetch_gate(t + 1);
    }
    if constexpr (G > 64) __syncthreads();
  }
  auto keep = [&](const float (&v)[NV][V], int which) {
    float* out = part_sums(p, static_cast<int>(blockIdx.x), which);
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      Raw<float, V> o;
      for (int i = 0; i < V; ++i) o.v[i] = v[c][i];
      o.store(out + col, left);
    });
  };
  if (p.dpre_weight != nullptr) keep(spre, 0);
  if (p.dpost_weight != nullptr) keep(spost, 1);
  if (p.dgate != nullptr && parts.per_group != 0) keep(sgate, 2);
}

// Rows wider than the registers: read again for every pass, column sums in the workspace.
template <typename T, typename TB>
__global__ __launch_bounds__(1024) void rr_block_norm_backward_wide_kernel(NormParams p, Parts parts) {
  constexpr int G = 1024;
  __shared__ float lds[kReduceFloats<G, 3>];
  __shared__ float lds2[kReduceFloats<G, 1>];
  const int D = p.hidden;
  const float inv = 1.0F / static_cast<float>(D);
  const auto* block = static_cast<const TB*>(p.block);
  const auto* wpost = static_cast<const T*>(p.post_weight);
  const auto* wpre = static_cast<const T*>(p.pre_weight);
  const auto* dh = static_cast<const T*>(p.dh);
  const auto* dn = static_cast<const T*>(p.dn);
  const bool post = wpost != nullptr;
  float* sums[3];
  for (int w = 0; w < 3; ++w) sums[w] = part_sums(p, static_cast<int>(blockIdx.x), w);
  for (int col = threadIdx.x; col < D; col += G) {
    for (int w = 0; w < 3; ++w) sums[w][col] = 0.0F;  // (a thread adds to its own columns only)
  }
  int first, end;
  part_range(parts, p.tokens, static_cast<int>(blockIdx.x), &first, &end);
  int until_gate = parts.group;
  for (int t = first; t < end; ++t) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    const T* h = static_cast<const T*>(p.x) + row;
    const std::size_t gate_row = p.gate != nullptr ? static_cast<std::size_t>(t / p.gate_tokens) * D : 0;
    const T* gate = p.gate != nullptr ? static_cast<const T*>(p.gate) + gate_row : nullptr;
    float s[3] = {0.0F, 0.0F, 0.0F};
    for (int col = threadIdx.x; col < D; col += G) {
      const float v = static_cast<float>(h[col]);
      s[0] = __builtin_fmaf(v, v, s[0]);
      if (dn != nullptr) s[1] = __builtin_fmaf(static_cast<float>(dn[row + col]) * static_cast<float>(wpre[col]), v, s[1]);
      if (post) {
        const float b = static_cast<float>(block[row + col]);
        s[2] = __builtin_fmaf(b, b, s[2]);
      }
    }
    reduce<G>(s, lds, 0);
    const float r = inverse_root(__builtin_fmaf(s[0], inv, p.eps));
    const float back = s[1] * inv * r * r;
    const float rb_scale = post ? inverse_root(__builtin_fmaf(s[2], inv, p.eps)) : 1.0F;
    auto dx_at = [&](int col) {
      float v = dh != nullptr ? static_cast<float>(dh[row + col]) : 0.0F;
      if (dn != nullptr) {
        v += r * (static_cast<float>(dn[row + col]) * static_cast<float>(wpre[col]) - static_cast<float>(h[col]) * back);
      }
      return v;
    };
    float s2[1] = {0.0F};
    if (post) {
      for (int col = threadIdx.x; col < D; col += G) {
        const float v = dx_at(col) * p.scale * (gate != nullptr ? static_cast<float>(gate[col]) : 1.0F);
        s2[0] = __builtin_fmaf(v * static_cast<float>(wpost[col]), static_cast<float>(block[row + col]) * rb_scale, s2[0]);
      }
    }
    reduce<G>(s2, lds2, 0);
    const float back2 = s2[0] * inv;
    const bool gate_ends = gate != nullptr && parts.per_group == 0 && (--until_gate == 0 || t + 1 == end);
    for (int col = threadIdx.x; col < D; col += G) {
      float v = dx_at(col);
      if (dn != nullptr) sums[0][col] = __builtin_fmaf(static_cast<float>(dn[row + col]), static_cast<float>(h[col]) * r, sums[0][col]);
      static_cast<T*>(p.dx)[row + col] = static_cast<T>(v);
      if (block == nullptr) continue;
      v *= p.scale;
      const float b = static_cast<float>(block[row + col]);
      const float unit = b * rb_scale;
      const float g = __builtin_fmaf(v, post ? unit * static_cast<float>(wpost[col]) : unit, sums[2][col]);
      sums[2][col] = gate_ends ? 0.0F : g;
      if (gate_ends && p.dgate != nullptr) static_cast<T*>(p.dgate)[gate_row + col] = static_cast<T>(g);
      if (gate != nullptr) v *= static_cast<float>(gate[col]);
      if (post) {
        sums[1][col] = __builtin_fmaf(v, unit, sums[1][col]);
        v = rb_scale * (v * static_cast<float>(wpost[col]) - unit * back2);
      }
      if (p.dblock != nullptr) static_cast<TB*>(p.dblock)[row + col] = static_cast<TB>(v);
    }
    if (gate_ends) until_gate = parts.group;
    __syncthreads();
  }
}

// Output row blockIdx.y of the column sums: 0 pre_weight, 1 post_weight (over all parts),
// 2 + g gate row g (over its parts). 32 columns a workgroup, 32 threads a column.
template <typename T>
__global__ __launch_bounds__(1024) void rr_block_norm_sums_kernel(NormParams p, Parts parts) {
  __shared__ float lds[32][33];
  const int y = static_cast<int>(blockIdx.y);
  const int which = y < 2 ? y : 2;
  T* out = static_cast<T*>(y == 0 ? p.dpre_weight : y == 1 ? p.dpost_weight : p.dgate);
  if (out == nullptr) return;
  int first = 0, count = parts.count;
  if (y >= 2) {
    first = (y - 2) * parts.per_group;
    count = parts.per_group;
    out += static_cast<std::size_t>(y - 2) * p.hidden;
  }
  const int c = static_cast<int>(threadIdx.x) & 31, q = static_cast<int>(threadIdx.x) >> 5;
  const int col = static_cast<int>(blockIdx.x) * 32 + c;
  float s = 0.0F;
  if (col < p.hidden) {
#pragma unroll 8
    for (int i = q; i < count; i += 32) s += part_sums(p, first + i, which)[col];
  }
  lds[q][c] = s;
  __syncthreads();
  if (q == 0 && col < p.hidden) {
    float total = 0.0F;
    for (int i = 0; i < 32; ++i) total += lds[i][c];
    out[col] = static_cast<T>(total);
  }
}

// ---- quantisation ----

// |v| as ordered bits: NaN above infinity above every number.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFU; }

template <int G>
__device__ __forceinline__ uint32_t reduce_max(uint32_t v, uint32_t* lds) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), off, 64)));
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < G / 64; ++w) v = max(v, lds[w]);
  }
  return v;
}

// The scale is finite and not zero. Cut to +-127: where an FP32 row's largest value is below
// 127^2 2^-149 its scale is a subnormal of so few bits that it may be up to 1.5 times 127 of
// them (16-bit rows have no such values).
__device__ __forceinline__ int8_t quantize(float v, float scale) {
  return static_cast<int8_t>(static_cast<int>(__builtin_amdgcn_fmed3f(__builtin_rintf(__fdiv_rn(v, scale)), -127.0F, 127.0F)));
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(G) void rr_quantize_rows_kernel(const T* x, int8_t* q, float* scales, int rows, int D) {
  constexpr int V = kChunk<T>;
  __shared__ uint32_t lds[G / 64];
  for (int t = static_cast<int>(blockIdx.x); t < rows; t = next_row(t, rows)) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    Raw<T, V> v[NV];
    uint32_t top = 0;
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      v[c].load(x + row + col, left);
      for (int i = 0; i < V; ++i) top = max(top, magnitude(v[c][i]));
    });
    top = reduce_max<G>(top, lds);
    const float scale = __fdiv_rn(__uint_as_float(top), 127.0F);
    // (values so small that their scale is zero in FP32 are zeros, too)
    const bool plain = scale > 0.0F && magnitude(scale) < 0x7F800000U;
    if (threadIdx.x == 0) scales[t] = scale;
    for_chunks<V, G, NV>(D, [&](int c, int col, int left) {
      Raw<int8_t, V> out;
      for (int i = 0; i < V; ++i) {
        out.v[i] = plain ? quantize(v[c][i], scale) : static_cast<int8_t>(0);
      }
      out.store(q + row + col, left);
    });
    if constexpr (G > 64) __syncthreads();
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void rr_quantize_rows_wide_kernel(const T* x, int8_t* q, float* scales, int rows, int D) {
  constexpr int G = 1024;
  __shared__ uint32_t lds[G / 64];
  for (int t = static_cast<int>(blockIdx.x); t < rows; t = next_row(t, rows)) {
    const std::size_t row = static_cast<std::size_t>(t) * D;
    uint32_t top = 0;
    for (int col = threadIdx.x; col < D; col += G) top = max(top, magnitude(static_cast<float>(x[row + col])));
    top = reduce_max<G>(top, lds);
    const float scale = __fdiv_rn(__uint_as_float(top), 127.0F);
    const bool plain = scale > 0.0F && magnitude(scale) < 0x7F800000U;
    if (threadIdx.x == 0) scales[t] = scale;
    for (int col = threadIdx.x; col < D; col += G) {
      q[row + col] = plain ? quantize(static_cast<float>(x[row + col]), scale) : static_cast<int8_t>(0);
    }
    __syncthreads();
  }
}

// ---- launches ----

// Threads and chunks that hold a row: the fewest threads with at most two chunks each.
// Returns 0 where no shape holds it.
int row_threads(int hidden, int chunk) {
  for (int g = 64; g <= 1024; g *= 2) {
    if (hidden <= 2 * g * chunk) return g;
  }
  return 0;
}

// Calls f<G, NV>() for rows of `hidden` elements; false where the wide kernels take them.
template <typename T, typename F>
bool with_shape(int hidden, F f) {
  const int g = row_threads(hidden, kChunk<T>);
  if (g == 64 && hidden <= 64 * kChunk<T>) {
    f.template operator()<64, 1>();
  } else if (g == 64) {
    f.template operator()<64, 2>();
  } else if (g == 128) {
    f.template operator()<128, 2>();
  } else if (g == 256) {
    f.template operator()<256, 2>();
  } else if (g == 512) {
    f.template operator()<512, 2>();
  } else if (g == 1024) {
    f.template operator()<1024, 2>();
  }
  return g != 0;
}

int row_blocks(int rows, int threads) { return std::max(1, std::min(rows, 2 * kSumThreads / threads)); }

template <typename T, typename TB>
struct Forward {
  NormParams p;
  hipStream_t stream;
  template <int G, int NV>
  void operator()() const {
    rr_block_norm_kernel<T, TB, G, NV><<<row_blocks(p.tokens, G), G, 0, stream>>>(p);
  }
};

template <typename T, typename TB>
struct Backward {
  NormParams p;
  Parts parts;
  hipStream_t stream;
  template <int G, int NV>
  void operator()() const {
    rr_block_norm_backward_kernel<T, TB, G, NV><<<parts.count, G, 0, stream>>>(p, parts);
  }
};

template <typename T>
struct Quantize {
  const T* x;
  int8_t* q;
  float* scale;
  int rows, hidden;
  hipStream_t stream;
  template <int G, int NV>
  void operator()() const {
    rr_quantize_rows_kernel<T, G, NV><<<row_blocks(rows, G), G, 0, stream>>>(x, q, scale, rows, hidden);
  }
};

template <typename T, typename TB>
hipError_t forward(const NormParams& p, hipStream_t stream) {
  if (!with_shape<T>(p.hidden, Forward<T, TB>{p, stream})) {
    rr_block_norm_wide_kernel<T, TB><<<row_blocks(p.tokens, 1024), 1024, 0, stream>>>(p);
  }
  return hipGetLastError();
}

Parts parts_of(const NormParams& p) {
  const int g = row_threads(p.hidden, p.dtype == RR_DTYPE_FP32 ? 4 : 8);
  return make_parts(p, g != 0 ? g : 1024);
}

template <typename T, typename TB>
hipError_t backward(const NormParams& p, hipStream_t stream) {
  const Parts parts = parts_of(p);
  if (parts.count != 0 && !with_shape<T>(p.hidden, Backward<T, TB>{p, parts, stream})) {
    rr_block_norm_backward_wide_kernel<T, TB><<<parts.count, 1024, 0, stream>>>(p, parts);
  }
  const bool gates = p.dgate != nullptr && parts.per_group != 0;
  if (p.dpre_weight != nullptr || p.dpost_weight != nullptr || gates) {
    const dim3 grid((p.hidden + 31) / 32, 2 + (gates ? parts.count / parts.per_group : 0));
    rr_block_norm_sums_kernel<T><<<grid, 1024, 0, stream>>>(p, parts);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t quantize_typed(const void* x, int8_t* q, float* scale, int rows, int hidden, hipStream_t stream) {
  const T* in = static_cast<const T*>(x);
  if (!with_shape<T>(hidden, Quantize<T>{in, q, scale, rows, hidden, stream})) {
    rr_quantize_rows_wide_kernel<T><<<row_blocks(rows, 1024), 1024, 0, stream>>>(in, q, scale, rows, hidden);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t block_norm(const NormParams& p, hipStream_t stream) {
  if (p.dtype == RR_DTYPE_FP32) return forward<float, float>(p, stream);
  if (p.dtype == RR_DTYPE_BF16) return p.block_f32 ? forward<bf16, float>(p, stream) : forward<bf16, bf16>(p, stream);
  return p.block_f32 ? forward<f16, float>(p, stream) : forward<f16, f16>(p, stream);
}

std::size_t block_norm_backward_workspace(const NormParams& p) {
  return static_cast<std::size_t>(parts_of(p).count) * 3 * static_cast<std::size_t>(p.hidden) * sizeof(float);
}

hipError_t block_norm_backward(const NormParams& p, hipStream_t stream) {
  if (p.dtype == RR_DTYPE_FP32) return backward<float, float>(p, stream);
  if (p.dtype == RR_DTYPE_BF16) return p.block_f32 ? backward<bf16, float>(p, stream) : backward<bf16, bf16>(p, stream);
  return p.block_f32 ? backward<f16, float>(p, stream) : backward<f16, f16>(p, stream);
}

hipError_t quantize_rows(const void* x, int8_t* q, float* scale, int rows, int hidden, int dtype, hipStream_t stream) {
  if (dtype == RR_DTYPE_FP32) return quantize_typed<float>(x, q, scale, rows, hidden, stream);
  if (dtype == RR_DTYPE_BF16) return quantize_typed<bf16>(x, q, scale, rows, hidden, stream);
  return quantize_typed<f16>(x, q, scale, rows, hidden, stream);
}

}  // namespace rr::kern
