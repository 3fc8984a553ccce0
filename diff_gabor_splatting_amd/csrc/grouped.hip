// Linear layers whose matrix and bias are those of the row's group:
// y_i = W_g x_i + b_g for the rows i of group g, and the gradients dx_i = W_g^T dy_i,
// dW_g = sum dy_i x_i^T, db_g = sum dy_i. Rows of no group have y = dx = 0.
//
// Rows are read and written where they lie, through the groups' order: no
// pass sorts them. Group sizes are on the device alone, so the host launches
// grids that hold any sizes and the workgroups find their group in the offsets.
//
//   group_few_kernel   y of a few rows: a wave to a row's output
//   group_rows_kernel  y and dx: a group's matrix in LDS, its rows streamed past
//   group_tile_kernel  y and dx where a matrix has a side too long for that, or
//                      there are many groups of few rows
//   group_sum_kernel   dW and db: tiles of dW over shares of all rows, whose
//                      partial sums group_join_kernel adds in their order
//
// No atomics: results do not depend on timing.
#include "group_rows.hpp"
#include "group_sums.hpp"
#include "group_tile.hpp"

namespace gs {
namespace {

// --------------------------------------------------------------------------
// y and dx, a tile of 128 x 128 to a workgroup

template <typename T, bool NContiguous>
int launch_tiles(const char* name, const void* x, int64_t stride, const void* w, const void* bias,
                 const Grouping& g, int64_t k, int64_t n, void* out, hipStream_t stream) {
  const GroupProduct p{n, k, ceil_div(n, kEdge), stride};
  const int64_t blocks = tile_numbers(g) * p.tiles_n;
  GS_REQUIRE(blocks < (int64_t(1) << 32) / kThreads, GS_ERR_OVERFLOW, "%s: too many rows", name);
  group_tile_kernel<T, NContiguous, kByGroup><<<dim3{unsigned(blocks)}, kThreads, 0, stream>>>(
      static_cast<const T*>(x), static_cast<const T*>(w), static_cast<const T*>(bias), g, p, {},
      static_cast<T*>(out));
  GS_LAUNCHED(name);
  return GS_OK;
}

// --------------------------------------------------------------------------
// y and dx, a group's matrix in LDS and its rows streamed past it

// `taken` is false where the matrix is too large to stay in LDS, or k less
// than a lane's part of a fragment.
template <typename T, bool Transposed>
int launch_rows(const char* name, const void* x, int64_t stride, const void* w, const void* bias,
                const Grouping& g, int64_t k, int64_t n, void* out, hipStream_t stream,
                bool& taken) {
  // Groups of up to about a tile of 128 rows go by tiles, where there are
  // enough of them: a matrix to each group costs the waves a barrier and a
  // wait. 48 and 96 rows to each of 512 groups of 128 -> 128 float16: 18.1 and
  // 18.8 us so, 11.1 and 13.2 by tiles; 192 rows: 22.2 and 22.7; 8 groups of 48
  // rows of 1024 -> 1024 bfloat16: 15.1 and 24.7.
  if (g.rows <= kEdge * int64_t(g.groups) && g.groups * ceil_div(n, kEdge) >= 128) {
    taken = false;
    return GS_OK;
  }
  const int64_t rows = g.rows + int64_t(kRowTile) * std::min(g.groups, g.rows);
  const int fragments = panel_fragments(sizeof(T), rows, k, n);
  const int64_t panels = fragments ? ceil_div(n, 16 * fragments) : 0;
  taken = fragments && panels <= 32 && k >= kPart<T>;
  if (!taken) return GS_OK;
  using std::integral_constant;
  auto launch = [&](auto tn, auto ahead, auto tail) {
    const int steps = int(steps_of(sizeof(T), k));
    GroupRows p{stride, int(k), int(n), int(panels), 0, steps, steps};
    p.workers = int(std::min<int64_t>(32 / panels * 8, ceil_div(rows, kRowTile)));
    const dim3 grid{unsigned(ceil_div(p.workers, 8) * panels * 8)};
    const size_t lds = size_t(p.steps) * 2 * tn.value * 1024;
    auto* const kernel =
        &group_rows_kernel<T, tn.value, ahead.value, Transposed, tail.value, kByGroup>;
    GS_CHECK(allow_lds(reinterpret_cast<const void*>(kernel), lds));
    kernel<<<grid, kRowThreads, lds, stream>>>(static_cast<const T*>(x), static_cast<const T*>(w),
                                               static_cast<const T*>(bias), g, p, {},
                                               static_cast<T*>(out));
    GS_LAUNCHED(name);
    return int(GS_OK);
  };
  using one = integral_constant<int, 1>;
  using two = integral_constant<int, 2>;
  using four = integral_constant<int, 4>;
  auto by_tail = [&](auto tn, auto ahead) {
    return k != steps_of(sizeof(T), k) * kStep<T> ? launch(tn, ahead, std::true_type{})
                                                  : launch(tn, ahead, std::false_type{});
  };
  auto by_ahead = [&](auto tn) {
    switch (ahead_of(steps_of(sizeof(T), k))) {
      case 1: return by_tail(tn, one{});
      case 2: return by_tail(tn, two{});
      default: return by_tail(tn, four{});
    }
  };
  switch (fragments) {
    case 8: return by_ahead(integral_constant<int, 8>{});
    case 4: return by_ahead(four{});
    default:
      if constexpr (sizeof(T) == 4)
        return by_ahead(two{});
      else
        return int(GS_OK);  // not reached: panel_fragments gives no such panel
  }
}

// --------------------------------------------------------------------------
// y of a few rows: a wave to a row's output, its lanes along the features. 4 rows
// of 1024 -> 1024 bfloat16: 3.9 us, launch and loads that wait for each other.
// More than 16 rows have a matrix put in LDS (32 to 380 rows of 1024 -> 1024 in
// 8 groups: 13 to 15 us).

constexpr int kFewRows = 16;

template <typename T>
__global__ __launch_bounds__(kThreads) void group_few_kernel(
    const T* __restrict__ x, int64_t stride, const T* __restrict__ w, const T* __restrict__ bias,
    Grouping g, int k, int n, T* __restrict__ y) {
  const int lane = threadIdx.x & 63, position = blockIdx.y;
  const int output = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (output >= n) return;
  const int s = find_segment(segments_of(g), position,
                             [&](int i) { return int64_t(begin_of(g, i)); });
  const int64_t row = row_at(g, position), group = s - 1;
  float sum = 0.f;
  if (s > 0 && s <= g.groups) {
    const T* const matrix = w + (group * n + output) * k;
    const T* const from = x + row * stride;
#pragma unroll 4
    for (int c = lane * kChunk; c < k; c += 64 * kChunk) {
      const int valid = min(k - c, kChunk);
      float a[kChunk], b[kChunk];
      load8<T>(matrix + c, valid, a);
      load8<T>(from + c, valid, b);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) sum = __builtin_fmaf(a[j], b[j], sum);
    }
#pragma unroll
    for (int step = 32; step; step >>= 1) sum += __shfl_xor(sum, step);
    if (bias) sum += float(bias[group * n + output]);
  }
  if (lane == 0) y[row * n + output] = T(sum);
}

// --------------------------------------------------------------------------
// dW and db: the sums over each group's rows of dy^T x.
//
// A workgroup of eight waves (two along the outputs, four along the features)
// adds up a tile of dW over its share of the positions, `Rows` of them at a
// time, whatever groups they are in: where a group ends it writes what it
// has and begins anew, and the loads, which are two steps ahead in registers
// and one in LDS, run on across that. A share is cut from the line on which
// each segment takes kGroupCost + its rows, so that writing a group's
// tile counts too. A group whose part of the line lies in one share is
// written at once; the others' parts are joined after.
//
// 1M x 512 -> 512 bfloat16 in 32 groups: 794 us (660 TFLOP/s), matrix cores 30%
// busy, LDS 21%: the waves wait at a step's barrier and for what lies between
// LDS and its first product. 100k x 256 -> 256 in 64 groups: 48 us, and 14 for the
// joining. One loop for both halves of a pair of steps: groups that end in
// either half cost 80 registers more.

constexpr int kSumThreads = 512;
constexpr int64_t kGroupCost = 128;   // of a group's tile, in rows
constexpr int64_t kGroupUncut = 512;  // on the line: groups of up to 384 rows

struct GroupSum {
  int64_t dy_stride, x_stride;
  int outputs, features;
  int tiles_m, tiles_n;  // of dW
  int shares;
};

// Rows of dy and x that are multiplied: the positions of one step.
struct StepOf {
  int first, count;
};

// 16 rows by 16 columns of LDS as a fragment, k along the rows, `k` the first
// of Mma's step.
template <typename T>
__device__ __forceinline__ typename Mma<T>::Fragment row_fragment(const T* lds, int pitch,
                                                                  int first) {
  if constexpr (sizeof(T) == 2) {
    return turned_fragment<T>(lds, pitch, first);
  } else {
    // Value j of lane group q is row 4 j + q: with a pitch of 16 past a
    // multiple of 64, the four lane groups read different banks.
    const int lane = threadIdx.x & 63;
    const T* const p = lds + (lane >> 4) * pitch + first + (lane & 15);
    return vec<T, 4>{p[0], p[4 * pitch], p[8 * pitch], p[12 * pitch]};
  }
}

// A wave's tile: 16 A outputs x 16 B features.
template <typename T, int A, int B, int Rows, bool Narrow>
__global__ __launch_bounds__(kSumThreads) void group_sum_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, Grouping g, GroupSum p,
    float* __restrict__ partial, T* __restrict__ dw, T* __restrict__ db) {
  constexpr int tile_m = 32 * A, tile_n = 64 * B;
  // 16 values past a multiple of 64: the rows that the lanes of a fragment's
  // load read lie in different banks.
  constexpr int pitch_m = tile_m + 16, pitch_n = tile_n + 16;
  constexpr int buffer = Rows * (pitch_m + pitch_n);
  constexpr int across_m = tile_m / 8, across_n = tile_n / 8;
  constexpr int apart_m = kSumThreads / across_m, apart_n = kSumThreads / across_n;
  constexpr int loads_m = (Rows + apart_m - 1) / apart_m, loads_n = (Rows + apart_n - 1) / apart_n;
  extern __shared__ __align__(16) char shared[];
  T* const lds = reinterpret_cast<T*>(shared);

  // Workgroups go to the eight XCDs in turn: the tiles of one share have one
  // XCD, and its L2. With fewer shares than XCDs the tiles go round.
  const int tiles = p.tiles_m * p.tiles_n;
  const int in_xcd = blockIdx.x >> 3;
  const bool shared_xcd = p.shares >= 8;
  const int share = shared_xcd ? in_xcd / tiles * 8 + int(blockIdx.x & 7)
                               : int(blockIdx.x % unsigned(p.shares));
  if (share >= p.shares) return;
  const int tile = shared_xcd ? in_xcd % tiles : int(blockIdx.x / unsigned(p.shares));
  const int m0 = tile / p.tiles_n * tile_m, n0 = tile % p.tiles_n * tile_n;
  const int64_t length = line_length(g, kGroupCost);
  Share at{kGroupCost};
  int from_segment, to_segment;
  at.from = border_at(g, kGroupCost, kGroupUncut, length, p.shares, share, from_segment);
  at.to = border_at(g, kGroupCost, kGroupUncut, length, p.shares, share + 1, to_segment);
  at.open(g, from_segment);
  // Steps come in pairs, for the two buffers: a group's last may be empty.
  auto pairs_of = [](const Share& of) { return (of.end - of.next + 2 * Rows - 1) / (2 * Rows); };
  Share ahead_at = at;
  int ahead_steps = 2 * pairs_of(at);
  // The positions of the step after the last that this was called for.
  auto next_step = [&]() {
    while (ahead_steps <= 0 && ahead_at.inside) {
      ahead_at.open(g, ahead_at.s + 1);
      ahead_steps = 2 * pairs_of(ahead_at);
    }
    const int left = ahead_at.end - ahead_at.next;
    const StepOf step{ahead_at.next, left < Rows ? left : Rows};
    ahead_at.next += step.count;
    --ahead_steps;
    return step;
  };

  // Each thread's places: eight outputs of loads_m rows, eight features of
  // loads_n.
  const int row_m = threadIdx.x / across_m, column_m = threadIdx.x % across_m * 8;
  const int row_n = threadIdx.x / across_n, column_n = threadIdx.x % across_n * 8;
  const int valid_m = min(p.outputs - m0 - column_m, 8);
  const int valid_n = min(p.features - n0 - column_n, 8);
  const bool ragged = p.outputs % 8 || p.features % 8;
  const T* const from_m = dy + m0 + column_m;
  const T* const from_n = x + n0 + column_n;

  struct Load {
    vec<T, 8> m[loads_m], n[loads_n];
  };
  Load ahead[2];
  // The rows of a step, one to a lane, -1 where there is none. They are asked
  // for two steps before the rows themselves: loads come back in their order,
  // and one step is less than a load takes (1M x 512 -> 512: 1,020 us against
  // 670 without an order; one load to a lane, not one to each place).
  int ids[2];
  auto find = [&](int& id) {
    const StepOf step = next_step();
    const int r = (threadIdx.x & 63) % Rows;
    id = r < step.count ? int(row_at(g, step.first + r)) : -1;
  };
  auto send = [&](Load& to, int& id) {
    int m[loads_m], n[loads_n];
#pragma unroll
    for (int i = 0; i < loads_m; ++i) m[i] = __shfl(id, row_m + i * apart_m);
#pragma unroll
    for (int i = 0; i < loads_n; ++i) n[i] = __shfl(id, row_n + i * apart_n);
    find(id);
#pragma unroll
    for (int i = 0; i < loads_m; ++i)
      to.m[i] = load_edge<T, 8, Narrow>(
          from_m + m[i] * p.dy_stride,
          m[i] >= 0 && row_m + i * apart_m < Rows ? valid_m : 0);
#pragma unroll
    for (int i = 0; i < loads_n; ++i)
      to.n[i] = load_edge<T, 8, Narrow>(
          from_n + n[i] * p.x_stride, n[i] >= 0 && row_n + i * apart_n < Rows ? valid_n : 0);
  };
  auto settle_all = [&](Load& from) {
#pragma unroll
    for (int i = 0; i < loads_m; ++i) from.m[i] = settle<T, 8, Narrow>(from.m[i], valid_m);
#pragma unroll
    for (int i = 0; i < loads_n; ++i) from.n[i] = settle<T, 8, Narrow>(from.n[i], valid_n);
  };
  auto put = [&](Load& from, T* to) {
    if (ragged) settle_all(from);
#pragma unroll
    for (int i = 0; i < loads_m; ++i)
      if (apart_m * loads_m == Rows || row_m + i * apart_m < Rows)
        *reinterpret_cast<vec<T, 8>*>(to + (row_m + i * apart_m) * pitch_m + column_m) = from.m[i];
#pragma unroll
    for (int i = 0; i < loads_n; ++i)
      if (apart_n * loads_n == Rows || row_n + i * apart_n < Rows)
        *reinterpret_cast<vec<T, 8>*>(to + Rows * pitch_m + (row_n + i * apart_n) * pitch_n +
                                      column_n) = from.n[i];
  };

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wave_m = (wave >> 2) * 16 * A, wave_n = (wave & 3) * 16 * B;
  const bool sums = db && n0 == 0;
  // float32 sums go over to others every kFold pairs of steps: a sum of n
  // values in one go is off by about sqrt(n / 8) half units, which shows in
  // float32 alone (1M rows of 512 -> 512: 62,000 to a share).
  constexpr bool folds = sizeof(T) == 4;
  constexpr int kFold = 16;
  f32x4 c[A][B], far[A][B];
  float sum[(A + 3) / 4];  // of the outputs of fragments wave % 4, + 4, ..
  float far_sum[(A + 3) / 4];
  auto clear = [&](auto& values, auto& sums) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) values[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < (A + 3) / 4; ++i) sums[i] = 0.f;
  };
  auto add_far = [&](auto& values, auto& sums, const auto& from, const auto& from_sums)
      __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) values[i][j] += from[i][j];
#pragma unroll
    for (int i = 0; i < (A + 3) / 4; ++i) sums[i] += from_sums[i];
  };
  auto multiply_step = [&](const T* from) {
    constexpr int deep = Mma<T>::step;
#pragma unroll
    for (int k = 0; k < Rows; k += deep) {
      typename Mma<T>::Fragment b[B];
#pragma unroll
      for (int j = 0; j < B; ++j)
        b[j] = row_fragment<T>(from + Rows * pitch_m + k * pitch_n, pitch_n, wave_n + 16 * j);
#pragma unroll
      for (int i = 0; i < A; ++i) {
        const typename Mma<T>::Fragment a =
            row_fragment<T>(from + k * pitch_m, pitch_m, wave_m + 16 * i);
#pragma unroll
        for (int j = 0; j < B; ++j) c[i][j] = Mma<T>::of(b[j], a, c[i][j]);
        if (sums && (wave & 3) == (i & 3)) {
#pragma unroll
          for (int j = 0; j < int(sizeof(a) / sizeof(T)); ++j) sum[i / 4] += float(a[j]);
        }
      }
    }
  };

  const int q = lane >> 4, i16 = lane & 15;
  // Writes the tile of segment at.s.
  auto finish = [&]() __attribute__((always_inline)) {
    const int64_t low = line_at(g, kGroupCost, at.s), high = line_at(g, kGroupCost, at.s + 1);
    const bool whole = low >= at.from && high <= at.to;
    const int64_t weights = int64_t(p.outputs) * p.features;
    const bool group = at.s > 0 && at.s <= g.groups;
    float* const part =
        partial + (2 * int64_t(share) + (low < at.from ? 0 : 1)) * (weights + p.outputs);
    // The tile's corner; a lane's place from there on.
    const int64_t corner = (m0 + wave_m) * int64_t(p.features) + n0 + wave_n;
    float* const to_part = part + corner;
    T* const to_dw = dw + ((at.s - 1) * weights + corner);
    const uint32_t place = uint32_t(i16) * p.features + 4 * q;
    const int rows_left = group ? p.outputs - m0 - wave_m - i16 : 0;
    const int columns_left = p.features - n0 - wave_n - 4 * q;
    // Fragment i of the outputs.
    auto put_fragment = [&](int i, const f32x4 (&f)[B], float total)
        __attribute__((always_inline)) {
      // Lane 16 q + i holds features 4 q .. 4 q + 3 of output i of a fragment.
      if (rows_left > 16 * i && (!whole || dw)) {
#pragma unroll
        for (int j = 0; j < B; ++j) {
          const uint32_t to = place + uint32_t(16 * i) * p.features + 16 * j;
          const vec<T, 4> v = {T(f[j][0]), T(f[j][1]), T(f[j][2]), T(f[j][3])};
          if (columns_left >= 16 * j + 4) {
            if (whole)
              store_packed<T, 4>(to_dw + to, v);
            else
              store_packed<float, 4>(to_part + to, f[j]);
          } else {
#pragma unroll
            for (int h = 0; h < 3; ++h)
              if (columns_left > 16 * j + h) {
                if (whole)
                  to_dw[to + h] = v[h];
                else
                  to_part[to + h] = f[j][h];
              }
          }
        }
      }
      if (sums && (wave & 3) == (i & 3)) {
        total += __shfl_xor(total, 16);
        total += __shfl_xor(total, 32);
        const int m = m0 + wave_m + 16 * i + i16;
        if (rows_left > 16 * i && q == 0) {
          if (whole)
            db[(at.s - 1) * int64_t(p.outputs) + m] = T(total);
          else
            part[weights + m] = total;
        }
      }
    };
    if constexpr (A * B < 32) {
#pragma unroll
      for (int i = 0; i < A; ++i) {
        put_fragment(i, c[i], sum[i / 4]);
        __builtin_amdgcn_sched_barrier(0);  // or all places are held at once
      }
    } else {
      // From c[0], the others moved up: all of it in succession is 25 KB of code
      // that a workgroup runs once a group and fetches each time (100k x 512 ->
      // 512 in 64 groups: 181 us, 157 so; tiles a quarter as large: 61, 64).
#pragma unroll 1
      for (int i = 0; i < A; ++i) {
        put_fragment(i, c[0], i < 4 ? sum[0] : sum[(A + 3) / 4 - 1]);
#pragma unroll
        for (int k = 0; k + 1 < A; ++k)
#pragma unroll
          for (int j = 0; j < B; ++j) c[k][j] = c[k + 1][j];
      }
    }
  };
  find(ids[0]);
  find(ids[1]);
  send(ahead[0], ids[0]);
  send(ahead[1], ids[1]);
  put(ahead[0], lds);
  send(ahead[0], ids[0]);
  __syncthreads();
  for (; at.inside; at.open(g, at.s + 1)) {
    clear(c, sum);
    if constexpr (folds) clear(far, far_sum);
    for (int pair = pairs_of(at); pair; --pair) {
      put(ahead[1], lds + buffer);
      send(ahead[1], ids[1]);
      multiply_step(lds);
      __syncthreads();
      put(ahead[0], lds);
      send(ahead[0], ids[0]);
      multiply_step(lds + buffer);
      __syncthreads();
      if (folds && pair % kFold == 0) {
        add_far(far, far_sum, c, sum);
        clear(c, sum);
      }
    }
    if constexpr (folds) add_far(c, sum, far, far_sum);
    finish();
  }
}

// How dW's sums are cut: fragments of a wave's tile along the outputs and the
// features, and shares of the line. As for one group:
// the widest tiles where they leave little empty and there are rows enough. The
// bias's gradient alone goes by one feature's plan and reads none: the grid
// has one column of tiles, which multiplies zeros (a pass of 1M x 512 -> 512 in
// 32 groups bfloat16 305 us, 741 with the matrix's gradient; 130k rows 48 and 139).
struct GroupSumPlan {
  int a, b;
  int64_t tiles_m, tiles_n, shares;
};

GroupSumPlan sum_plan(size_t size, const Grouping& g, int64_t features, int64_t outputs) {
  GroupSumPlan p{};
  const int64_t wide = 4 * ceil_div(outputs, 256) * ceil_div(features, 256);
  const int64_t narrow = ceil_div(outputs, 128) * ceil_div(features, 128);
  const bool large = size == 2 && outputs > 128 && features > 128 && 10 * wide <= 13 * narrow &&
                     double(g.rows) * double(outputs) * double(features) >= 2e10;
  p.a = large ? 8 : outputs <= 64 ? 2 : 4;
  p.b = large ? 4 : features <= 64 ? 1 : 2;
  p.tiles_m = ceil_div(outputs, 32 * p.a);
  p.tiles_n = ceil_div(features, 64 * p.b);
  const int64_t tiles = p.tiles_m * p.tiles_n;
  // A workgroup to a compute unit: its parts cost as much as more of them gain
  // (100k, 256 -> 256 in 64 groups: 73 us with 512 workgroups, 59 with 256).
  p.shares = std::max<int64_t>(1, 256 / tiles);
  p.shares = std::min(p.shares, ceil_div(line_length(g, kGroupCost), 2 * kGroupCost));
  return p;
}

int check_grouped(const char* name, int32_t dtype, const void* offsets, int64_t rows,
                  int64_t groups, int64_t features, int64_t outputs) {
  GS_CHECK(check_grouping(name, offsets, rows, groups));
  GS_CHECK(check_rows(name, dtype, rows, features, features));
  GS_CHECK(check_rows(name, dtype, rows, outputs, outputs));
  GS_REQUIRE(outputs <= kMostFeatures / 64 && features <= kMostFeatures / 64, GS_ERR_ARGUMENT,
             "%s: at most %lld features and outputs", name, (long long)(kMostFeatures / 64));
  return GS_OK;
}

Grouping grouping(const int32_t* order, const int32_t* offsets, int64_t rows, int64_t groups) {
  return {order, offsets, int32_t(rows), int32_t(groups)};
}

}  // namespace
}  // namespace gs

extern "C" {

int gs_grouped_linear_forward(int32_t dtype, const void* x, int64_t row_stride, const void* weight,
                              const void* bias, const int32_t* order, const int32_t* offsets,
                              int64_t rows, int64_t groups, int64_t features, int64_t outputs,
                              void* y, void* stream) {
  using namespace gs;
  clear_error();
  const char* const name = "gs_grouped_linear_forward";
  GS_CHECK(check_grouped(name, dtype, offsets, rows, groups, features, outputs));
  GS_CHECK(check_rows(name, dtype, rows, features, row_stride));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && weight && y, GS_ERR_ARGUMENT, "null pointer passed to %s", name);
  const Grouping g = grouping(order, offsets, rows, groups);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (rows <= kFewRows) {
      const dim3 grid{unsigned(ceil_div(outputs, kThreads / 64)), unsigned(rows)};
      group_few_kernel<T><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
          static_cast<const T*>(x), row_stride, static_cast<const T*>(weight),
          static_cast<const T*>(bias), g, int(features), int(outputs), static_cast<T*>(y));
      GS_LAUNCHED(name);
      return int(GS_OK);
    }
    bool taken = false;
    GS_CHECK((launch_rows<T, false>(name, x, row_stride, weight, bias, g, features, outputs, y,
                                    static_cast<hipStream_t>(stream), taken)));
    if (taken) return int(GS_OK);
    return launch_tiles<T, true>(name, x, row_stride, weight, bias, g, features, outputs, y,
                                 static_cast<hipStream_t>(stream));
  });
}

int gs_grouped_linear_backward_input(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                     const void* weight, const int32_t* order,
                                     const int32_t* offsets, int64_t rows, int64_t groups,
                                     int64_t features, int64_t outputs, void* grad_x,
                                     void* stream) {
  using namespace gs;
  clear_error();
  const char* const name = "gs_grouped_linear_backward_input";
  GS_CHECK(check_grouped(name, dtype, offsets, rows, groups, features, outputs));
  GS_CHECK(check_rows(name, dtype, rows, outputs, grad_stride));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(grad_y && weight && grad_x, GS_ERR_ARGUMENT, "null pointer passed to %s", name);
  const Grouping g = grouping(order, offsets, rows, groups);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    bool taken = false;
    GS_CHECK((launch_rows<T, true>(name, grad_y, grad_stride, weight, nullptr, g, outputs,
                                   features, grad_x, static_cast<hipStream_t>(stream), taken)));
    if (taken) return int(GS_OK);
    return launch_tiles<T, false>(name, grad_y, grad_stride, weight, nullptr, g, outputs,
                                  features, grad_x, static_cast<hipStream_t>(stream));
  });
}

size_t gs_grouped_linear_backward_weight_workspace_size(int32_t dtype, int64_t rows,
                                                        int64_t groups, int64_t features,
                                                        int64_t outputs) {
  using namespace gs;
  if (rows < 0 || rows > kMostGroupedRows || groups <= 0 || groups > kMostGroupsOfRows ||
      features <= 0 || outputs <= 0)
    return 0;
  const size_t size = dtype == GS_FLOAT32 ? 4 : 2;
  const Grouping g = grouping(nullptr, nullptr, rows, groups);
  auto bytes = [&](int64_t planned, int64_t values) {
    const int64_t shares = sum_plan(size, g, planned, outputs).shares;
    return shares == 1 ? 0 : size_t(2 * shares) * size_t(outputs * values) * sizeof(float);
  };
  return std::max(bytes(features, features + 1), bytes(1, 1));
}

int gs_grouped_linear_backward_weight(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                      const void* x, int64_t row_stride, const int32_t* order,
                                      const int32_t* offsets, int64_t rows, int64_t groups,
                                      int64_t features, int64_t outputs, void* grad_weight,
                                      void* grad_bias, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  using namespace gs;
  clear_error();
  const char* const name = "gs_grouped_linear_backward_weight";
  GS_CHECK(check_grouped(name, dtype, offsets, rows, groups, features, outputs));
  GS_CHECK(check_rows(name, dtype, rows, outputs, grad_stride));
  if (grad_weight) GS_CHECK(check_rows(name, dtype, rows, features, row_stride));
  if (!grad_weight && !grad_bias) return GS_OK;
  GS_REQUIRE(offsets && (rows == 0 || (grad_y && (x || !grad_weight))), GS_ERR_ARGUMENT,
             "null pointer passed to %s", name);
  const size_t need = gs_grouped_linear_backward_weight_workspace_size(dtype, rows, groups,
                                                                       features, outputs);
  GS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), GS_ERR_WORKSPACE,
             "workspace too small for %s", name);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Grouping g = grouping(order, offsets, rows, groups);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const GroupSumPlan plan = sum_plan(sizeof(T), g, grad_weight ? features : 1, outputs);
    const int64_t across = grad_weight ? features : 0;
    const GroupSum p{grad_stride,       row_stride,        int(outputs),    int(across),
                     int(plan.tiles_m), int(plan.tiles_n), int(plan.shares)};
    const int64_t blocks = (plan.shares >= 8 ? ceil_div(plan.shares, 8) * 8 : plan.shares) *
                           plan.tiles_m * plan.tiles_n;
    GS_REQUIRE(blocks < (int64_t(1) << 32) / kSumThreads, GS_ERR_OVERFLOW,
               "%s: too many values", name);
    T* const dw = static_cast<T*>(grad_weight);
    T* const db = static_cast<T*>(grad_bias);
    float* const partial = static_cast<float*>(workspace);
    auto launch = [&](auto a, auto b, auto narrow) {
      constexpr int step = a.value == 2 || (a.value == 4 && sizeof(T) == 2) ? 64 : 32;
      constexpr size_t lds = 2 * step * (32 * a.value + 16 + 64 * b.value + 16) * sizeof(T);
      auto* const kernel = &group_sum_kernel<T, a.value, b.value, step, narrow.value>;
      GS_CHECK(allow_lds(reinterpret_cast<const void*>(kernel), lds));
      kernel<<<dim3{unsigned(blocks)}, kSumThreads, lds, s>>>(
          static_cast<const T*>(grad_y), static_cast<const T*>(x), g, p, partial, dw, db);
      GS_LAUNCHED(name);
      return int(GS_OK);
    };
    using std::integral_constant;
    using one = integral_constant<int, 1>;
    using two = integral_constant<int, 2>;
    using four = integral_constant<int, 4>;
    const int shape = plan.a * 10 + plan.b;
    // Rows of fewer than eight values have no place to load eight from.
    const bool few = outputs < 8 || features < 8;
    using wide = std::false_type;
    using narrow = std::true_type;
    if (shape == 21) GS_CHECK(few ? launch(two{}, one{}, narrow{}) : launch(two{}, one{}, wide{}));
    if (shape == 22) GS_CHECK(few ? launch(two{}, two{}, narrow{}) : launch(two{}, two{}, wide{}));
    if (shape == 41)
      GS_CHECK(few ? launch(four{}, one{}, narrow{}) : launch(four{}, one{}, wide{}));
    if (shape == 42) GS_CHECK(launch(four{}, two{}, wide{}));
    if constexpr (sizeof(T) == 2)
      if (shape == 84) GS_CHECK(launch(integral_constant<int, 8>{}, four{}, wide{}));
    if (plan.shares == 1) return int(GS_OK);
    const Join<T> join{partial,     dw,          db,      kGroupCost,
                       kGroupUncut, plan.shares, outputs * across, outputs};
    return launch_joins(&join, 1, g, s);
  });
}

}  // extern "C"
