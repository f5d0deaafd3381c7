// Where the experts' rows lie in a dispatched buffer, and the tiles a grouped product cuts them
// into, derived from the loads on the device.
#pragma once

#include "common.cuh"

namespace brt_b200 {

constexpr int kMaxExperts = 1024;

struct ExpertTable {
  int first_tile[kMaxExperts + 1];  // exclusive sums of the experts' tiles
  int row_base[kMaxExperts];
  int load[kMaxExperts];
};

// By one whole warp.  `tiles_of(load)`: how many tiles an expert with that many rows has.  Loads
// are cut at the slot of a padded buffer and at the end of the buffer.
template <typename F>
__device__ __forceinline__ void fill_expert_table(ExpertTable& t, const int* loads, int experts,
                                                  int max_path_load, long long total_rows,
                                                  F tiles_of) {
  const int lane = threadIdx.x & 31;
  int tiles = 0;
  long long row = 0;
  for (int p = 0; p < experts; p += 32) {
    const int e = p + lane;
    int load = e < experts ? loads[e] : 0;
    if (load < 0) load = 0;
    if (max_path_load != 0 && load > max_path_load) load = max_path_load;
    long long rows_incl = load;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, rows_incl, d);
      if (lane >= d) rows_incl += up;
    }
    long long base = max_path_load != 0 ? (long long)e * max_path_load : row + rows_incl - load;
    row += __shfl_sync(0xffffffffu, rows_incl, 31);
    if (base > total_rows) base = total_rows;
    if (load > total_rows - base) load = (int)(total_rows - base);
    const int mine = e < experts ? tiles_of(load) : 0;
    int tiles_incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, tiles_incl, d);
      if (lane >= d) tiles_incl += up;
    }
    if (e < experts) {
      t.first_tile[e] = tiles + tiles_incl - mine;
      t.row_base[e] = (int)base;
      t.load[e] = load;
    }
    tiles += __shfl_sync(0xffffffffu, tiles_incl, 31);
  }
  if (lane == 0) t.first_tile[experts] = tiles;
}

// The expert that tile `t` belongs to: the last one whose first tile is not behind it.
__device__ __forceinline__ int expert_of_tile(const ExpertTable& t, int experts, int tile) {
  int lo = 0, hi = experts - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first_tile[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
}

}  // namespace brt_b200
