// The rows of each group: a stable counting sort of the rows by group.
//
//   order[offsets[g] .. offsets[g + 1])  the rows of group g, in their order
//   order[offsets[groups] ..)            the rows of no group, in their order
//
// A row of no group (an index outside 0 .. groups - 1) is sorted as group
// `groups`. Blocks of rows count their groups (count_kernel), the counts of
// each group are summed over the blocks (column_kernel, or where they are few
// each block of the next kernel for itself), and the blocks place their rows
// (place_kernel): bytes read twice and written once, 12 to 20 a row. One block's
// rows need the last kernel alone. Ranks within 64 rows come from ballots over
// the bits of the group, so nothing depends on timing. 100k rows in 64 groups
// 10.8 us a call, 1M rows in 512 groups 25: latency, of the counters in LDS and
// of the rounds that follow each other.
#include "groups.hpp"
#include "layers_api.hpp"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMostGroups = 4096;  // counters for four waves, and beginnings, in LDS

struct Sorted {
  int64_t rows;
  int groups;   // without the rows of none
  int bits;     // of a group's number, `groups` included
  int64_t blocks;
  bool direct;  // every block of place_kernel sums the counts for itself
};

template <typename I>
__device__ __forceinline__ int key_of(const I* __restrict__ index, const Sorted& s, int64_t row) {
  const I i = index[row];
  return i < I(0) || i >= I(s.groups) ? s.groups : int(i);
}

// A wave takes 64 * Rounds rows that follow each other.
template <int Rounds>
__device__ __forceinline__ int64_t first_row() {
  return (int64_t(blockIdx.x) * kWaves + (threadIdx.x >> 6)) * (64 * Rounds) + (threadIdx.x & 63);
}

template <typename I, int Rounds>
__device__ __forceinline__ void load_keys(const I* __restrict__ index, const Sorted& s,
                                          int (&key)[Rounds]) {
  const int64_t row = first_row<Rounds>();
#pragma unroll
  for (int r = 0; r < Rounds; ++r)
    key[r] = row + 64 * r < s.rows ? key_of(index, s, row + 64 * r) : -1;
}

template <typename I, int Rounds>
__global__ __launch_bounds__(kThreads) void count_kernel(const I* __restrict__ index, Sorted s,
                                                         int32_t* __restrict__ counts) {
  extern __shared__ int count[];
  for (int g = threadIdx.x; g <= s.groups; g += kThreads) count[g] = 0;
  int key[Rounds];
  load_keys<I, Rounds>(index, s, key);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < Rounds; ++r)
    if (key[r] >= 0) atomicAdd(&count[key[r]], 1);
  __syncthreads();
  int32_t* const mine = counts + blockIdx.x * int64_t(s.groups + 1);
  for (int g = threadIdx.x; g <= s.groups; g += kThreads) mine[g] = count[g];
}

// Each group's counts become what the blocks before have of it, and its
// total. 16 groups to a workgroup, 64 shares of the blocks.
constexpr int kColumnThreads = 1024;
constexpr int kShares = kColumnThreads / 16;

__global__ __launch_bounds__(kColumnThreads) void column_kernel(Sorted s,
                                                                int32_t* __restrict__ counts,
                                                                int32_t* __restrict__ totals) {
  __shared__ int sums[kShares][16];
  const int column = threadIdx.x & 15, share = threadIdx.x >> 4;
  const int g = blockIdx.x * 16 + column;
  const int64_t each = (s.blocks + kShares - 1) / kShares;
  const int64_t from = share * each, to = from + each < s.blocks ? from + each : s.blocks;
  int sum = 0;
  if (g <= s.groups) {
#pragma unroll 4
    for (int64_t b = from; b < to; ++b) sum += counts[b * (s.groups + 1) + g];
  }
  sums[share][column] = sum;
  __syncthreads();
  if (g > s.groups) return;
  int before = 0;
#pragma unroll 16
  for (int i = 0; i < kShares; ++i) before += i < share ? sums[i][column] : 0;
  if (share == kShares - 1) totals[g] = before + sum;
#pragma unroll 4
  for (int64_t b = from; b < to; ++b) {
    int32_t* const at = counts + b * (s.groups + 1) + g;
    const int here = *at;
    *at = before;
    before += here;
  }
}

// Exclusive sums of 0 .. groups of `value`, in LDS: begin[g].
template <typename F>
__device__ __forceinline__ void begin_of_groups(const Sorted& s, int* begin, F value) {
  __shared__ int wave_sums[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int before = 0;
  for (int g0 = 0; g0 <= s.groups; g0 += kThreads) {
    const int g = g0 + threadIdx.x;
    const int v = g <= s.groups ? value(g) : 0;
    int up = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = __shfl_up(up, d, 64);
      if (lane >= d) up += other;
    }
    if (lane == 63) wave_sums[wave] = up;
    __syncthreads();
    int sum = before;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) sum += wave_sums[w];
      before += wave_sums[w];
    }
    if (g <= s.groups) begin[g] = sum + up - v;
    __syncthreads();
  }
}

// counts: each block's groups (null: there is one block), or but for `direct`
// what the blocks before have of them.
template <typename I, int Rounds>
__global__ __launch_bounds__(kThreads) void place_kernel(const I* __restrict__ index, Sorted s,
                                                         const int32_t* __restrict__ counts,
                                                         const int32_t* __restrict__ totals,
                                                         int32_t* __restrict__ order,
                                                         int32_t* __restrict__ offsets) {
  extern __shared__ int shared[];
  const int size = s.groups + 1;
  int* const at = shared;                   // [kWaves][size]: next place
  int* const begin = shared + kWaves * size;
  int* const all = begin + size;            // direct: each group's rows,
  int* const earlier = all + size;          // and those of the blocks before
  for (int i = threadIdx.x; i < kWaves * size; i += kThreads) at[i] = 0;
  if (s.direct)
    for (int i = threadIdx.x; i < 2 * size; i += kThreads) all[i] = 0;
  int key[Rounds];
  load_keys<I, Rounds>(index, s, key);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* const mine = at + wave * size;
#pragma unroll
  for (int r = 0; r < Rounds; ++r)
    if (key[r] >= 0) atomicAdd(&mine[key[r]], 1);
  __syncthreads();
  if (s.direct) {
    // 16 counts of a thread at a time; whole numbers have the same sum in any
    // order.
    const int entries = int(s.blocks) * size, mine_from = int(blockIdx.x) * size;
    for (int first = threadIdx.x; first < entries; first += 16 * kThreads) {
      int count[16];
#pragma unroll
      for (int u = 0; u < 16; ++u)
        count[u] = first + u * kThreads < entries ? counts[first + u * kThreads] : 0;
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const int entry = first + u * kThreads, g = entry % size;
        if (!count[u]) continue;
        atomicAdd(&all[g], count[u]);
        if (entry < mine_from) atomicAdd(&earlier[g], count[u]);
      }
    }
    __syncthreads();
  }
  begin_of_groups(s, begin, [&](int g) {
    if (s.direct) return all[g];
    if (counts) return totals[g];
    int sum = 0;
    for (int w = 0; w < kWaves; ++w) sum += at[w * size + g];
    return sum;
  });
  const int32_t* const before = counts ? counts + blockIdx.x * int64_t(size) : nullptr;
  for (int g = threadIdx.x; g <= s.groups; g += kThreads) {
    if (blockIdx.x == 0) offsets[g] = begin[g];
    int place = begin[g] + (s.direct ? earlier[g] : before ? before[g] : 0);
    for (int w = 0; w < kWaves; ++w) {
      const int here = at[w * size + g];
      at[w * size + g] = place;
      place += here;
    }
  }
  __syncthreads();
  const int64_t row = first_row<Rounds>();
#pragma unroll
  for (int r = 0; r < Rounds; ++r) {
    const int k = key[r];
    // The lanes that have this row's group.
    uint64_t same = __ballot(k >= 0);
    for (int b = 0; b < s.bits; ++b) {
      const uint64_t set = __ballot((k >> b) & 1);
      same &= (k >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((uint64_t(1) << lane) - 1));
    const int first = k >= 0 ? mine[k] : 0;
    wave_order();
    if (k >= 0) {
      order[int64_t(first) + rank] = int32_t(row + 64 * r);
      if (rank == 0) mine[k] = first + __popcll(same);
    }
    wave_order();
  }
}

// Counts up to which every block sums them for itself, which saves a launch:
// 100k rows in 64 groups (6,370 counts) 12.7 us to 10.8, 1M in 8 (4,401) 16.1 to
// 14.1; 100k in 150 (14,798) 13.0 and 14.9, 1M in 32 (16,137) 17.5 and 18.9.
constexpr int64_t kDirect = 8192;

// Rounds of 64 rows of a wave: 8 where there are rows enough for a workgroup to
// each compute unit, 4 below.
int rounds_of(int64_t rows) { return rows > (int64_t(1) << 18) ? 8 : 4; }

}  // namespace
}  // namespace gs

extern "C" {

size_t gs_row_groups_workspace_size(int64_t rows, int64_t groups) {
  using namespace gs;
  if (rows <= 0 || groups <= 0) return 0;
  const int64_t blocks = ceil_div(rows, kThreads * rounds_of(rows));
  return blocks == 1 ? 0 : size_t(blocks + 1) * size_t(groups + 1) * sizeof(int32_t);
}

int gs_row_groups(int32_t wide, const void* index, int64_t rows, int64_t groups, int32_t* order,
                  int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gs;
  clear_error();
  GS_REQUIRE(rows >= 0 && rows <= kMostGroupedRows, GS_ERR_OVERFLOW,
             "gs_row_groups: rows must be 0 through %lld", (long long)kMostGroupedRows);
  GS_REQUIRE(groups >= 1 && groups <= kMostGroups, GS_ERR_ARGUMENT,
             "gs_row_groups: groups must be 1 through %lld", (long long)kMostGroups);
  GS_REQUIRE(offsets && (rows == 0 || (index && order)), GS_ERR_ARGUMENT,
             "null pointer passed to gs_row_groups");
  const size_t need = gs_row_groups_workspace_size(rows, groups);
  GS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), GS_ERR_WORKSPACE,
             "workspace too small for gs_row_groups");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rounds = rounds_of(rows);
  Sorted sorted{rows, int(groups), 0, std::max<int64_t>(1, ceil_div(rows, kThreads * rounds)),
                false};
  sorted.direct = sorted.blocks > 1 && sorted.blocks * (groups + 1) <= kDirect;
  while (groups >> sorted.bits) ++sorted.bits;
  const bool single = sorted.blocks == 1;
  int32_t* const counts = single ? nullptr : static_cast<int32_t*>(workspace);
  int32_t* const totals = single ? nullptr : counts + sorted.blocks * (groups + 1);
  const size_t lds = size_t(groups + 1) * sizeof(int);
  const dim3 grid{unsigned(sorted.blocks)};
  auto launch = [&](auto zero, auto count) {
    using I = decltype(zero);
    const I* const from = static_cast<const I*>(index);
    if (!single) {
      count_kernel<I, count.value><<<grid, kThreads, lds, s>>>(from, sorted, counts);
      GS_LAUNCHED("row groups count");
    }
    if (!single && !sorted.direct) {
      column_kernel<<<dim3{unsigned(ceil_div(groups + 1, 16))}, kColumnThreads, 0, s>>>(
          sorted, counts, totals);
      GS_LAUNCHED("row groups columns");
    }
    auto* const kernel = &place_kernel<I, count.value>;
    const size_t all_lds = (kWaves + (sorted.direct ? 3 : 1)) * lds;
    GS_CHECK(allow_lds(reinterpret_cast<const void*>(kernel), all_lds));
    kernel<<<grid, kThreads, all_lds, s>>>(from, sorted, counts, totals, order, offsets);
    GS_LAUNCHED("row groups place");
    return int(GS_OK);
  };
  using four = std::integral_constant<int, 4>;
  using all = std::integral_constant<int, 8>;
  if (wide)
    return rounds == 4 ? launch(int64_t(0), four{}) : launch(int64_t(0), all{});
  return rounds == 4 ? launch(int32_t(0), four{}) : launch(int32_t(0), all{});
}

}  // extern "C"
