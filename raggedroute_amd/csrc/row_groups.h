// Groups of 16 rows of an expert, for the kernels that take few rows an expert.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "block_device.h"
#include "expert_gemm.h"
#include "wave.h"

namespace rr::kern {

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

// The most groups that `rows` rows of `experts` experts make: of n rows an expert has (n - 1) /
// kGroup + 1 at most.
inline std::size_t most_groups(int rows, int experts) {
  const int busy = experts < rows ? experts : rows;
  return static_cast<std::size_t>((rows - busy) / kGroup + busy);
}

}  // namespace rr::kern
