// Rows in groups, as the kernels see them.
//
// Positions 0 .. rows - 1 hold the rows by group: the row at position p is
// order[p] (p itself without an order), and group g has the positions from
// offsets[g] to offsets[g + 1]. The positions are cut into groups + 2 segments:
// those before the first group, the groups, and those behind the last; the
// first and the last segment hold the rows of no group. Offsets and rows are
// held to the range that exists, so that wrong ones give wrong results and no
// access outside.
#pragma once

#include "layers_api.hpp"

namespace gs {

// Positions are 32-bit, with room for the last tile's rows past the end.
constexpr int64_t kMostGroupedRows = 0x7ffff000;
constexpr int64_t kMostGroupsOfRows = int64_t(1) << 20;

struct Grouping {
  const int32_t* order;  // null: the rows lie in the order of their groups
  const int32_t* offsets;
  int32_t rows, groups;
};

__device__ __forceinline__ int segments_of(const Grouping& g) { return g.groups + 2; }

// First position of segment s, `rows` for the one past the last.
__device__ __forceinline__ int begin_of(const Grouping& g, int s) {
  if (s <= 0) return 0;
  if (s > g.groups + 1) return g.rows;
  return min(max(g.offsets[s - 1], 0), g.rows);
}

__device__ __forceinline__ int64_t row_at(const Grouping& g, int position) {
  if (!g.order) return position;
  return int64_t(min(uint32_t(g.order[position]), uint32_t(g.rows - 1)));
}

// The last of segments 0 .. count - 1 whose key is at most `v`, for keys that
// do not fall, the first of them at most v. A wave looks at 64 at a time: two
// rounds of loads up to 4,096 segments, where halving the range takes twelve.
template <typename F>
__device__ __forceinline__ int find_segment(int count, int64_t v, F key) {
  const int lane = threadIdx.x & 63;
  int low = 0, left = count;
  while (left > 1) {
    const int step = (left + 63) / 64, at = lane * step;
    const bool before = at < left && key(low + at) <= v;
    const int found = max(__popcll(__ballot(before)), 1) - 1;
    low += found * step;
    left = min(step, left - found * step);
  }
  return __builtin_amdgcn_readfirstlane(low);
}

inline int check_grouping(const char* name, const void* offsets, int64_t rows, int64_t groups) {
  GS_REQUIRE(rows >= 0 && rows <= kMostGroupedRows, GS_ERR_OVERFLOW,
             "%s: rows must be 0 through %lld", name, (long long)kMostGroupedRows);
  GS_REQUIRE(groups >= 1 && groups <= kMostGroupsOfRows, GS_ERR_ARGUMENT,
             "%s: groups must be 1 through %lld", name, (long long)kMostGroupsOfRows);
  GS_REQUIRE(offsets || rows == 0, GS_ERR_ARGUMENT, "null pointer passed to %s", name);
  return GS_OK;
}

}  // namespace gs
