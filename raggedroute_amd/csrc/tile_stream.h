// The stream of slices of the tile kernels on the matrix cores: loads straight into LDS with
// their waits, LDS reads of 16 bytes, the order of an expert's tiles, segment bounds.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "wave.h"

namespace rr::kern {

#define RR_LDS __attribute__((address_space(3)))
typedef int i4 __attribute__((ext_vector_type(4)));

constexpr int kBufferFlags = 0x00027000;  // raw 32-bit buffer
constexpr uint32_t kPast = 0x80000000U;   // an offset past every record count
constexpr int kTileCols = 256;
constexpr int kSliceBytes = 128;               // of every row
constexpr int kHalfBytes = 128 * kSliceBytes;  // half an operand's slice

// Barriers and waits of the pipeline. The loads into LDS are written in assembly: they
// have no register results, and the compiler, which would wait for all of them before
// any LDS read, does not see them; every wait for them is one of these.
__device__ __forceinline__ void wave_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
template <int LOADS>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A raw buffer from `at` to `left` bytes further (uniform).
__device__ __forceinline__ i4 make_buffer(const char* at, int64_t left) {
  const int64_t p = reinterpret_cast<int64_t>(at);
  const int records = static_cast<int>(left <= 0 ? 0 : left < 0x7FFFFFFF ? left : 0x7FFFFFFF);
  return i4{__builtin_amdgcn_readfirstlane(static_cast<int>(p)), __builtin_amdgcn_readfirstlane(static_cast<int>(p >> 32) & 0xFFFF),
            __builtin_amdgcn_readfirstlane(records), kBufferFlags};
}
// 64 lanes x 16 bytes from `buffer` (a byte offset per lane) to LDS at `to` (uniform). The
// compiler may have written a word of the descriptor with a vector instruction (a lane read)
// just before, which has to be five wait states ahead of a load that reads it, and it does
// not look into assembly: the move and s_nop 3 are five.
__device__ __forceinline__ void load_to_lds(i4 buffer, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                   __builtin_amdgcn_readfirstlane(static_cast<int>(to))),
               "v"(offset), "s"(buffer)
               : "memory", "m0");
}

// The same past the caches.
__device__ __forceinline__ void stream_to_lds(i4 buffer, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(
                   __builtin_amdgcn_readfirstlane(static_cast<int>(to))),
               "v"(offset), "s"(buffer)
               : "memory", "m0");
}
// The same of 64 lanes x 4 bytes.
__device__ __forceinline__ void load_words_to_lds(i4 buffer, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(
                   __builtin_amdgcn_readfirstlane(static_cast<int>(to))),
               "v"(offset), "s"(buffer)
               : "memory", "m0");
}

__device__ __forceinline__ i4 read16(uint32_t at) { return *reinterpret_cast<RR_LDS const i4*>(at); }

// Tile t of an expert's: four row tiles at a time, so that the 32 that an XCD runs side by
// side span four rows of tiles and eight columns (with eight rows at a time the weight
// gradients of E = 8, K = 4096, F = 14336 took 2.19 ms instead of 2.04).
__device__ __forceinline__ void place_tile(int t, int row_tiles, int col_tiles, int* rt, int* ct) {
  constexpr int kRows = 4;
  const int group = t / (kRows * col_tiles);
  const int rows = min(row_tiles - group * kRows, kRows);
  const int within = t - group * kRows * col_tiles;
  *rt = group * kRows + within % rows;
  *ct = within / rows;
}

// The offsets in s_off[0 .. experts] to the segments' bounds: the largest of each and those
// before it. By one whole wave, whose own reads afterwards see them.
__device__ __forceinline__ void raise_offsets(int32_t* s_off, int experts, int lane) {
  const int per = experts / 64 + 1;  // entries of a lane
  int32_t most = 0;
  for (int j = 0; j < per; ++j) {
    const int e = lane * per + j;
    if (e <= experts) most = max(most, s_off[e]);
  }
  const int32_t before = __shfl_up(rr::dev::wave_inclusive_max(most), 1, 64);
  most = lane > 0 ? before : 0;
  for (int j = 0; j < per; ++j) {
    const int e = lane * per + j;
    if (e <= experts) s_off[e] = most = max(most, s_off[e]);
  }
  rr::dev::wave_lds_sync();
}

}  // namespace rr::kern
