// Sums over each group's rows, cut into shares that go by the rows and not by
// the groups.
//
// Shares are cut from the line on which each segment takes `cost` + its rows,
// so that what a group costs beside its rows counts too. A group whose part of
// the line lies in one share is written by that share; the others' parts go to
// two places that each share has, its head (the group began before it) and its
// tail, and group_join_kernel adds them in their order. No atomics: results do not
// depend on timing.
#pragma once

#include "groups.hpp"
#include "kept8.hpp"

namespace gs {

__device__ __forceinline__ int64_t line_at(const Grouping& g, int64_t cost, int s) {
  return begin_of(g, s) + cost * s;
}
__host__ __device__ __forceinline__ int64_t line_length(const Grouping& g, int64_t cost) {
  return g.rows + cost * (int64_t(g.groups) + 2);
}

// Border b of the shares on the line. One that lies in a segment of up to
// `uncut` goes to that segment's nearer end: small groups are written at once,
// where a part of each would be as much as the whole (50k rows of 128 -> 128 in
// 512 groups: 60 MB of parts beside 58 MB of inputs and results).
// `segment` becomes the one that it lies in or begins.
__device__ __forceinline__ int64_t border_at(const Grouping& g, int64_t cost, int64_t uncut,
                                             int64_t length, int64_t shares, int64_t b,
                                             int& segment) {
  const int64_t v = length * b / shares;
  segment = find_segment(segments_of(g), v, [&](int i) { return line_at(g, cost, i); });
  const int64_t low = line_at(g, cost, segment), high = line_at(g, cost, segment + 1);
  if (b == 0 || b == shares || high - low > uncut) return v;
  if (v - low < high - v) return low;
  ++segment;
  return high;
}

// Where a share stands: segment s, whose positions from `next` to `end` are its.
struct Share {
  int64_t cost;
  int64_t from, to;  // on the line
  int s, next, end;
  bool inside;  // whether segment s begins before the share's end

  __device__ __forceinline__ void open(const Grouping& g, int segment) {
    s = segment;
    next = end = 0;
    inside = s < segments_of(g) && line_at(g, cost, s) < to;
    if (!inside) return;
    // A row at position i of segment s lies at i + cost (s + 1).
    const int64_t shift = cost * (s + 1);
    const int64_t low = begin_of(g, s), high = begin_of(g, s + 1);
    const int64_t a = from - shift > low ? from - shift : low;
    const int64_t b = to - shift < high ? to - shift : high;
    const bool some = a < b && s > 0 && s <= g.groups;
    next = some ? int(a) : 0;
    end = some ? int(b) : 0;
  }
};

// --------------------------------------------------------------------------

constexpr int kJoinThreads = 256;

// Parts [shares, 2 (head, tail), weights + biases] of a group's values, dW's and
// then db's; either result may be null.
template <typename T>
struct Join {
  const float* partial;
  T* dw;
  T* db;
  int64_t cost, uncut, shares;
  int64_t weights, biases;
  __host__ __device__ bool by_border(const Grouping& g) const { return shares - 1 < g.groups; }
  __host__ __device__ int64_t each(const Grouping& g) const {
    return by_border(g) ? shares - 1 : g.groups;
  }
};

template <typename T>
struct Joins {
  Join<T> of[2];
};

// Adds the parts of the groups that lie in several shares. blockIdx.y: a
// group, or where there are fewer borders between shares than groups a border,
// which stands for the group that it is the first border within; blockIdx.x:
// 4 kJoinThreads / Slices values of dW and db at a time, for which each slice of
// the threads adds every Slices-th part.
template <typename T, int Slices>
__global__ __launch_bounds__(kJoinThreads) void group_join_kernel(Joins<T> joins, Grouping g) {
  constexpr int columns = kJoinThreads / Slices;
  __shared__ vec<float, 4> sums[Slices][columns];
  const Join<T> p = joins.of[blockIdx.z];
  const float* __restrict__ const partial = p.partial;
  T* __restrict__ const dw = p.dw;
  T* __restrict__ const db = p.db;
  const bool by_border = p.by_border(g);
  if (blockIdx.y >= p.each(g)) return;
  const int64_t length = line_length(g, p.cost);
  int s = blockIdx.y + 1;
  int64_t border = s;
  if (by_border)
    s = find_segment(segments_of(g), length * border / p.shares,
                     [&](int i) { return line_at(g, p.cost, i); });
  const int64_t low = line_at(g, p.cost, s), high = line_at(g, p.cost, s + 1);
  if (high - low <= p.uncut) return;
  if (!by_border) {  // the first border behind `low`
    border = ((low + 1) * p.shares + length - 1) / length;
  }
  const int64_t v = length * border / p.shares;
  if (s < 1 || s > g.groups || border >= p.shares || v <= low || v >= high ||
      length * (border - 1) / p.shares > low)
    return;
  // Shares border - 1 (its tail) .. last (their heads).
  int64_t last = (high * p.shares - 1) / length;
  if (last >= p.shares) last = p.shares - 1;
  const int count = int(last - border) + 2;
  const int64_t weights = p.weights, size = weights + p.biases;
  const int slice = threadIdx.x / columns, column = threadIdx.x % columns;
  for (int64_t first = int64_t(blockIdx.x) * 4 * columns; first < size;
       first += int64_t(gridDim.x) * 4 * columns) {
    const int64_t i = first + 4 * column;
    const int valid = int(size - i < 4 ? size - i : 4);
    // Eight loads at a time, whatever the count: one after the other they
    // would each be waited for.
    vec<float, 4> sum = 0.f;
    for (int first_part = slice; first_part < count; first_part += 8 * Slices) {
      vec<float, 4> part[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = first_part + u * Slices;
        part[u] = load_valid<float, 4>(
            partial + (j ? 2 * (border - 1 + j) : 2 * border - 1) * size + i,
            j < count ? valid : 0);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += part[u];
    }
    if constexpr (Slices > 1) {
      sums[slice][column] = sum;
      __syncthreads();
      if (slice == 0)
        for (int j = 1; j < Slices; ++j) sum += sums[j][column];
      __syncthreads();
    }
    if (slice) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= valid) continue;
      if (i + j < weights) {
        if (dw) dw[(s - 1) * weights + i + j] = T(sum[j]);
      } else if (db) {
        db[(s - 1) * p.biases + (i + j - weights)] = T(sum[j]);
      }
    }
  }
}

// Joins up to two results in one launch; those of one share have no parts.
template <typename T>
int launch_joins(const Join<T>* join, int count, const Grouping& g, hipStream_t stream) {
  Joins<T> joins{};
  int some = 0;
  int64_t each = 0, values = 0, parts = 0;
  for (int i = 0; i < count; ++i) {
    if (join[i].shares == 1) continue;
    joins.of[some++] = join[i];
    each = std::max(each, join[i].each(g));
    values = std::max(values, join[i].weights + join[i].biases);
    parts = std::max(parts, join[i].shares);
  }
  if (!some) return GS_OK;
  auto launch = [&](auto slices) {
    // Workgroups go on to further values: those of the groups that lie in one
    // share have nothing to do, and a workgroup to each 64 values and border
    // (100k x 256 -> 256 in 64 groups: 32,000) took 180 us to find that out.
    const int64_t chunks = ceil_div(values, 4 * kJoinThreads / slices.value);
    const dim3 grid{unsigned(std::min(chunks, ceil_div(4096, each))), unsigned(each),
                    unsigned(some)};
    group_join_kernel<T, slices.value><<<grid, kJoinThreads, 0, stream>>>(joins, g);
  };
  // The more slices the more parts there are to a group (many of the largest
  // one's: 512 shares of 7 groups 15 us with 16 slices, 8 with 64).
  if (parts < 8 * int64_t(g.groups))
    launch(std::integral_constant<int, 1>{});
  else if (parts < 32 * int64_t(g.groups))
    launch(std::integral_constant<int, 4>{});
  else if (parts < 64 * int64_t(g.groups))
    launch(std::integral_constant<int, 16>{});
  else
    launch(std::integral_constant<int, 64>{});
  GS_LAUNCHED("group_join_kernel");
  return GS_OK;
}

}  // namespace gs
