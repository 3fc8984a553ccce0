// Linear layers that all rows share, with a low-rank adapter of the row's
// group beside them: y_i = W x_i + b + s B_g A_g x_i for the rows i of group g, and
// the gradients dx_i = W^T dy_i + s A_g^T B_g^T dy_i, dA_g = s sum (B_g^T dy_i) x_i^T,
// dB_g = s sum dy_i (A_g x_i)^T. Rows of no group have the shared layer alone.
//
// The inner rows, s A_g x_i and s B_g^T dy_i, are the sums that the other products
// share: each is computed once, kept (see Inner) and met again by the product
// with the other narrow matrix, in the accumulators of the wide one, and by
// the narrow matrices' gradients.
//
//   few_inner_kernel, few_adapted_kernel  the forward pass of a few rows
//   group_rows_kernel  inner rows; y and dx
//   group_tile_kernel  the same where a matrix has a side too long for that
//   narrow_sum_kernel  dA and dB, a wave to 128 columns of a share of the rows
#include "group_rows.hpp"
#include "group_sums.hpp"
#include "group_tile.hpp"

namespace gs {
namespace {

// --------------------------------------------------------------------------
// y of a few rows: a workgroup to an inner row, then a wave to an output. 8 rows
// of 1024 -> 1024 bfloat16, rank 16: 4.1 and 5.3 us, of which most is loads that
// wait for each other (the group, its row, the values).

constexpr int kFewRows = 16;

// A lane's part of the sum over k of a[k] b[k], and the whole of such parts.
template <typename T>
__device__ __forceinline__ float dot_part(const T* a, const T* b, int k) {
  const int lane = threadIdx.x & 63;
  float sum = 0.f;
#pragma unroll 4
  for (int c = lane * kChunk; c < k; c += 64 * kChunk) {
    const int valid = min(k - c, kChunk);
    float u[kChunk], v[kChunk];
    load8<T>(a + c, valid, u);
    load8<T>(b + c, valid, v);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) sum = __builtin_fmaf(u[j], v[j], sum);
  }
  return sum;
}
__device__ __forceinline__ float all_lanes(float sum) {
#pragma unroll
  for (int step = 32; step; step >>= 1) sum += __shfl_xor(sum, step);
  return sum;
}

// A wave to one of the rank, or to several of more than 16.
constexpr int kInnerThreads = 1024;

template <typename T>
__global__ __launch_bounds__(kInnerThreads) void few_inner_kernel(const T* __restrict__ x,
                                                             int64_t stride,
                                                             const T* __restrict__ down,
                                                             float scale, Grouping g, int k,
                                                             Inner<T> inner) {
  __shared__ float values[kMostRank];
  const int position = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int s = find_segment(segments_of(g), position,
                             [&](int i) { return int64_t(begin_of(g, i)); });
  const bool member = s > 0 && s <= g.groups;
  if (threadIdx.x < kMostRank) values[threadIdx.x] = 0.f;
  __syncthreads();
  if (member) {
    const T* const row = x + row_at(g, position) * stride;
    const T* const matrix = down + int64_t(s - 1) * inner.rank * k;
    for (int r = wave; r < inner.rank; r += kInnerThreads / 64) {
      const float sum = all_lanes(dot_part<T>(row, matrix + int64_t(r) * k, k));
      if (lane == 0) values[r] = scale * sum;
    }
  }
  __syncthreads();
  if (wave) return;
  float most = finite_size(values[lane]);
#pragma unroll
  for (int step = 32; step; step >>= 1) most = fmaxf(most, __shfl_xor(most, step));
  const float up = inner.begin_row(position, most, lane == 0);
  if (4 * lane >= 32 * inner.chunks()) return;
  const float four[4] = {values[4 * lane], values[4 * lane + 1], values[4 * lane + 2],
                         values[4 * lane + 3]};
  inner.template put<4>(position, 4 * lane, four, up);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void few_adapted_kernel(
    const T* __restrict__ x, int64_t stride, const T* __restrict__ w, const T* __restrict__ bias,
    const T* __restrict__ up, Grouping g, int k, int n, Inner<T> inner, T* __restrict__ y) {
  const int lane = threadIdx.x & 63, position = blockIdx.y;
  const int output = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (output >= n) return;
  const int64_t row = row_at(g, position);
  const int s = find_segment(segments_of(g), position,
                             [&](int i) { return int64_t(begin_of(g, i)); });
  // The shared sum, and the narrow one, a value of the rank to a lane.
  float sum = dot_part<T>(x + row * stride, w + int64_t(output) * k, k);
  if (s > 0 && s <= g.groups && lane < inner.rank)
    sum = __builtin_fmaf(inner.get(position, lane),
                         float(up[(int64_t(s - 1) * n + output) * inner.rank + lane]), sum);
  sum = all_lanes(sum);
  if (bias) sum += float(bias[output]);
  if (lane == 0) y[row * n + output] = T(sum);
}

// --------------------------------------------------------------------------
// Inner rows, y and dx by tiles

template <typename T, bool NContiguous, int Mode>
int launch_tiles(const char* name, const void* x, int64_t stride, const void* w, const void* bias,
                 const Grouping& g, int64_t k, int64_t n, const Adapters<T>& adapters, void* out,
                 hipStream_t stream) {
  const GroupProduct p{n, k, ceil_div(n, kEdge), stride};
  const int64_t blocks = tile_numbers(g) * p.tiles_n;
  GS_REQUIRE(blocks < (int64_t(1) << 32) / kThreads, GS_ERR_OVERFLOW, "%s: too many rows", name);
  group_tile_kernel<T, NContiguous, Mode><<<dim3{unsigned(blocks)}, kThreads, 0, stream>>>(
      static_cast<const T*>(x), static_cast<const T*>(w), static_cast<const T*>(bias), g, p,
      adapters, static_cast<T*>(out));
  GS_LAUNCHED(name);
  return GS_OK;
}

// --------------------------------------------------------------------------
// Inner rows, y and dx with the matrix in LDS and the rows streamed past it

// `taken` is false where the matrix is too large to stay in LDS, or k less
// than a lane's part of a fragment.
template <typename T, bool Transposed, int Mode>
int launch_rows(const char* name, const void* x, int64_t stride, const void* w, const void* bias,
                const Grouping& g, int64_t k, int64_t n, const Adapters<T>& adapters, void* out,
                hipStream_t stream, bool& taken) {
  // kAdapted's steps need no even number: the adapters' chunks are among them.
  const int64_t steps = Mode == kInner ? steps_of(sizeof(T), k) : ceil_div(k, kStep<T>);
  const int64_t chunks = Mode == kInner ? 0 : adapters.inner.chunks();
  int fragments;
  if constexpr (Mode == kInner) {
    fragments = n <= 32 ? 2 : 4;  // all of the rank, at most 64
    if (steps * 2048 * fragments > int64_t(kRowLds)) fragments = 0;
  } else {
    // The adapter's matrix and what the waves turn their rows in lie beside.
    fragments = panel_fragments(sizeof(T), g.rows, k, n);
    auto bytes = [&](int64_t of) {
      return of * 1024 * (2 * steps + chunks * (sizeof(T) == 4 ? 2 : 1)) +
             kRowWaves * 2048 + of * 64;
    };
    while (fragments && bytes(fragments) > 160 * 1024) fragments /= 2;
    if (fragments < (sizeof(T) == 4 ? 2 : 4)) fragments = 0;
  }
  // Steps under way: those that leave the fewest to be filled up.
  int64_t ahead = Mode == kInner ? ahead_of(steps) : 4;
  if constexpr (Mode == kAdapted)
    for (int64_t of = 3; of >= 2; --of)
      if (ceil_div(steps + chunks, of) * of < ceil_div(steps + chunks, ahead) * ahead) ahead = of;
  const int64_t all = ceil_div(steps + chunks, ahead) * ahead;
  const int64_t panels = fragments ? ceil_div(n, 16 * fragments) : 0;
  taken = fragments && panels <= 32 && k >= kPart<T>;
  if (!taken) return GS_OK;
  using std::integral_constant;
  auto launch = [&](auto tn, auto under_way, auto tail) {
    GroupRows p{stride, int(k), int(n), int(panels), 0, int(steps), int(all)};
    // Inner rows are bound by reading: as many workgroups as LDS lets run.
    const int64_t most = Mode == kInner ? (steps * 2048 * fragments > 48 * 1024 ? 256 : 512)
                                        : 32 / panels * 8;
    // A worker to each tile, or to each group where those are fewer rows.
    p.workers = int(std::min<int64_t>(
        most, ceil_div(g.rows, kRowTile) + std::min(g.groups, g.rows)));
    const dim3 grid{unsigned(ceil_div(p.workers, 8) * panels * 8)};
    const size_t lds =
        size_t(2 * steps + chunks * (sizeof(T) == 4 ? 2 : 1)) * tn.value * 1024;
    auto* const kernel =
        &group_rows_kernel<T, tn.value, under_way.value, Transposed, tail.value, Mode>;
    GS_CHECK(allow_lds(reinterpret_cast<const void*>(kernel), lds));
    kernel<<<grid, kRowThreads, lds, stream>>>(static_cast<const T*>(x), static_cast<const T*>(w),
                                               static_cast<const T*>(bias), g, p, adapters,
                                               static_cast<T*>(out));
    GS_LAUNCHED(name);
    return int(GS_OK);
  };
  using one = integral_constant<int, 1>;
  using two = integral_constant<int, 2>;
  using three = integral_constant<int, 3>;
  using four = integral_constant<int, 4>;
  auto by_tail = [&](auto tn, auto under_way) {
    return k != steps * kStep<T> ? launch(tn, under_way, std::true_type{})
                                 : launch(tn, under_way, std::false_type{});
  };
  auto by_ahead = [&](auto tn) {
    if constexpr (Mode == kInner) {
      if (ahead == 1) return by_tail(tn, one{});
    } else {
      if (ahead == 3) return by_tail(tn, three{});
    }
    return ahead == 2 ? by_tail(tn, two{}) : by_tail(tn, four{});
  };
  switch (fragments) {
    case 8:
      if constexpr (Mode == kAdapted) return by_ahead(integral_constant<int, 8>{});
    case 4: return by_ahead(four{});
    default:
      if constexpr (sizeof(T) == 4 || Mode == kInner) return by_ahead(two{});
      return int(GS_OK);  // not reached: panel_fragments gives no such panel
  }
}

// --------------------------------------------------------------------------
// dA and dB: the sums over each group's rows of inner^T rows, [rank, width].
//
// A wave takes 128 columns (eight to each of 16 lanes) and 16 rows at a time
// (four to each lane group), which is how memory holds them and how the matrix
// instructions take them: no LDS, and no turning but of four values of a lane.
// Waves share nothing; each has its own share of the rows. float32 and float16
// go through the float32 instruction, four rows at a time, whose rate is the
// reading's at a rank of 16 and a third of it at 64; bfloat16, whose inner
// parts need no scale, through its own, 16 rows at a time and once for each
// part, four times as fast (dB at rank 64 of 1M x 512: 790 us and 419). At rank
// 16 dA and dB of 1M x 512 -> 512 bfloat16 take 475 us together: 2.3 GB at 4.8
// TB/s, the address unit busy for 70% (a lane loads 2 bytes of an inner row).

constexpr int64_t kNarrowCost = 32;   // of a group's sums, in rows
constexpr int64_t kNarrowUncut = 96;  // on the line: groups of up to 64 rows
constexpr int kNarrowColumns = 128;
constexpr int kNarrowRows = 16;  // of a step

template <typename T>
struct NarrowSum {
  Inner<T> inner;
  const T* rows;
  int64_t stride;
  float* partial;
  T* out;
  int width, blocks, shares;
  bool turned;  // the result is [width, rank] (dB), not [rank, width] (dA)
};

template <typename T>
struct NarrowSums {
  NarrowSum<T> of[2];
};

// blockIdx.y: which of two sums. R: 16s of the rank.
template <typename T, int R, bool Narrow>
__global__ __launch_bounds__(kThreads) void narrow_sum_kernel(NarrowSums<T> sums, Grouping g) {
  const NarrowSum<T> p = sums.of[blockIdx.y];
  const Inner<T> inner = p.inner;
  const T* __restrict__ const rows = p.rows;
  float* __restrict__ const partial = p.partial;
  T* __restrict__ const out = p.out;
  constexpr int fours = kNarrowRows / 4;
  constexpr bool parts = std::is_same_v<T, bf16>;
  const int64_t number = int64_t(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  const int block = __builtin_amdgcn_readfirstlane(int(number % p.blocks));
  const int share = __builtin_amdgcn_readfirstlane(int(number / p.blocks));
  if (share >= p.shares) return;
  const int lane = threadIdx.x & 63, q = lane >> 4, i16 = lane & 15;
  const int column = block * kNarrowColumns + 8 * i16;
  const int valid = max(0, min(p.width - column, 8));
  const int64_t length = line_length(g, kNarrowCost);
  Share at{kNarrowCost};
  int from_segment, to_segment;
  at.from = border_at(g, kNarrowCost, kNarrowUncut, length, p.shares, share, from_segment);
  at.to = border_at(g, kNarrowCost, kNarrowUncut, length, p.shares, share + 1, to_segment);
  at.open(g, from_segment);
  const int64_t size = int64_t(inner.rank) * p.width;
  for (; at.inside; at.open(g, at.s + 1)) {
    f32x4 c[R][8];
    // Rows and inner rows of a step are on their way while the step before is
    // multiplied; the rows' places, 64 at a time, a whole 64 before.
    struct Step {
      vec<T, 8> rows[fours];
      typename Inner<T>::Raw inner[fours][R];
      float scales[fours];
    };
    const int first = at.next, count = at.end - at.next;
    auto find = [&](int of) {
      return count > 0 ? int(row_at(g, first + min(64 * of + lane, count - 1))) : 0;
    };
    int id, next_id;
    auto load = [&](Step& to, int step) {
      if (step % 4 == 0) {
        id = next_id;
        next_id = find(step / 4 + 1);
      }
#pragma unroll
      for (int i = 0; i < fours; ++i) {
        const int place = step * kNarrowRows + 4 * q + i;
        const int64_t row = __shfl(id, place % 64);
        const bool live = place < count;
        to.rows[i] = load_edge<T, 8, Narrow>(rows + row * p.stride + column, live ? valid : 0);
#pragma unroll
        for (int t = 0; t < R; ++t)
          to.inner[i][t] = inner.raw(first + min(place, count - 1), 16 * t + i16);
        if constexpr (Inner<T>::scaled)
          to.scales[i] = inner.scales[first + min(place, count - 1)];
      }
    };
    auto multiply_step = [&](const Step& of, int step, auto infinite) {
      vec<T, 8> v[fours];
      bool live[fours];
#pragma unroll
      for (int i = 0; i < fours; ++i) {
        live[i] = step * kNarrowRows + 4 * q + i < count;
        v[i] = settle<T, 8, Narrow>(of.rows[i], live[i] ? valid : 8);
      }
      if constexpr (parts) {
        typedef vec<short, 4> raw;
        raw b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          b[j] = __builtin_bit_cast(raw, vec<T, 4>{v[0][j], v[1][j], v[2][j], v[3][j]});
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (infinite.value && h) {
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = (b[j] & 0x7f80) == 0x7f80 ? raw(0) : b[j];
          }
#pragma unroll
          for (int t = 0; t < R; ++t) {
            vec<T, 4> a;
#pragma unroll
            for (int i = 0; i < fours; ++i)
              a[i] = live[i] ? of.inner[i][t].parts[h % (4 / sizeof(T))] : T(0.f);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              c[t][j] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(raw, a), b[j],
                                                                  c[t][j], 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < fours; ++i) {
          float a[R];
#pragma unroll
          for (int t = 0; t < R; ++t) {
            a[t] = live[i] ? of.inner[i][t].sum() : 0.f;
            if constexpr (Inner<T>::scaled) a[t] *= of.scales[i];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int t = 0; t < R; ++t)
              c[t][j] =
                  __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], float(v[i][j]), c[t][j], 0, 0, 0);
        }
      }
    };
    auto sum = [&](auto infinite) {
#pragma unroll
      for (int t = 0; t < R; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) c[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      id = 0;
      next_id = find(0);
      Step ahead[2];
      if (count > 0) load(ahead[0], 0);
      for (int step = 0; step * kNarrowRows < count; step += 2) {
        load(ahead[1], step + 1);
        multiply_step(ahead[0], step, infinite);
        load(ahead[0], step + 2);
        multiply_step(ahead[1], step + 1, infinite);
      }
    };
    sum(std::false_type{});
    if constexpr (parts) {
      // An infinity of a row times a second part, which may be zero or of the
      // other sign, is a NaN that the formula has not: sums that came out bad are
      // taken again, and infinities of the rows meet the first parts alone.
      float bad = 0.f;
#pragma unroll
      for (int t = 0; t < R; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) bad = __builtin_fmaf(c[t][j][r], 0.f, bad);
      if (__ballot(bad != bad)) sum(std::true_type{});
    }
    // Lane 16 q + i holds ranks 16 t + 4 q .. + 3 of columns 8 i .. 8 i + 7.
    if (at.s < 1 || at.s > g.groups) continue;
    const int64_t low = line_at(g, kNarrowCost, at.s), high = line_at(g, kNarrowCost, at.s + 1);
    const bool whole = low >= at.from && high <= at.to;
    float* const part = partial + (2 * int64_t(share) + (low < at.from ? 0 : 1)) * size;
    T* const to = out + (at.s - 1) * size;
#pragma unroll
    for (int t = 0; t < R; ++t) {
      const int r0 = 16 * t + 4 * q;
      if (p.turned) {
        const int left = max(0, min(inner.rank - r0, 4));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= valid) continue;
          const int64_t place = int64_t(column + j) * inner.rank + r0;
          if (whole)
            store_valid<T, 4>(to + place, left, vec<T, 4>{T(c[t][j][0]), T(c[t][j][1]),
                                                          T(c[t][j][2]), T(c[t][j][3])});
          else
            store_valid<float, 4>(part + place, left, c[t][j]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r0 + r >= inner.rank) continue;
          const int64_t place = int64_t(r0 + r) * p.width + column;
          const float v[8] = {c[t][0][r], c[t][1][r], c[t][2][r], c[t][3][r],
                              c[t][4][r], c[t][5][r], c[t][6][r], c[t][7][r]};
          if (whole)
            store8<T>(to + place, valid, v);
          else
            store8<float>(part + place, valid, v);
        }
      }
    }
  }
}

// Up to 4,096 waves, of 256 rows each, or of 64 for up to 512 shares: with fewer
// rows a wave's time counts, with more its parts (100k rows of 256 at rank 16, dA,
// dB and what they take: 82 us at 64 rows, 56 at 256; 33k of 187 and 57 at
// rank 5: 35 and 44).
int64_t narrow_shares(const Grouping& g, int64_t width) {
  const int64_t most = std::max<int64_t>(1, 4096 / ceil_div(width, kNarrowColumns));
  const int64_t length = line_length(g, kNarrowCost);
  return std::min(most, std::max(ceil_div(length, 256),
                                 std::min<int64_t>(512, ceil_div(length, 64))));
}

// dA and dB in one launch, and their joins in another: with few rows a launch
// is most of the time.
template <typename T>
int launch_narrow(const char* name, NarrowSum<T>* sums, int count, const Grouping& g,
                  hipStream_t stream) {
  NarrowSums<T> both{};
  Join<T> joins[2];
  int64_t waves = 0;
  bool narrow = false;
  for (int i = 0; i < count; ++i) {
    NarrowSum<T>& p = sums[i];
    p.blocks = int(ceil_div(p.width, kNarrowColumns));
    p.shares = int(narrow_shares(g, p.width));
    waves = std::max(waves, int64_t(p.blocks) * p.shares);
    narrow = narrow || p.width < 8;
    both.of[i] = p;
    joins[i] = {p.partial, p.out,    nullptr, kNarrowCost,
                kNarrowUncut, p.shares, int64_t(p.inner.rank) * p.width, 0};
  }
  const dim3 grid{unsigned(ceil_div(waves, kThreads / 64)), unsigned(count)};
  auto launch = [&](auto r, auto narrow) {
    narrow_sum_kernel<T, r.value, narrow.value><<<grid, kThreads, 0, stream>>>(both, g);
  };
  auto by_width = [&](auto r) {
    narrow ? launch(r, std::true_type{}) : launch(r, std::false_type{});
  };
  const int rank = sums[0].inner.rank;
  if (rank <= 16)
    by_width(std::integral_constant<int, 1>{});
  else if (rank <= 32)
    by_width(std::integral_constant<int, 2>{});
  else
    by_width(std::integral_constant<int, 4>{});
  GS_LAUNCHED(name);
  return launch_joins(joins, count, g, stream);
}

int check_adapted(const char* name, int32_t dtype, const void* offsets, int64_t rows,
                  int64_t groups, int64_t features, int64_t outputs, int64_t rank) {
  GS_CHECK(check_grouping(name, offsets, rows, groups));
  GS_CHECK(check_rows(name, dtype, rows, features, features));
  GS_CHECK(check_rows(name, dtype, rows, outputs, outputs));
  GS_REQUIRE(outputs <= kMostFeatures / 64 && features <= kMostFeatures / 64, GS_ERR_ARGUMENT,
             "%s: at most %lld features and outputs", name, (long long)(kMostFeatures / 64));
  GS_REQUIRE(rank >= 1 && rank <= kMostRank, GS_ERR_ARGUMENT, "%s: rank must be 1 through %d",
             name, kMostRank);
  return GS_OK;
}

int check_inner(const char* name, const void* inner, size_t bytes, int64_t rows, int64_t rank) {
  GS_REQUIRE(inner && bytes >= Inner<float>::bytes(rows, rank), GS_ERR_WORKSPACE,
             "inner rows too small for %s", name);
  GS_REQUIRE(reinterpret_cast<uintptr_t>(inner) % 16 == 0, GS_ERR_ARGUMENT,
             "inner rows are not 16-byte aligned in %s", name);
  return GS_OK;
}

Grouping grouping(const int32_t* order, const int32_t* offsets, int64_t rows, int64_t groups) {
  return {order, offsets, int32_t(rows), int32_t(groups)};
}

}  // namespace
}  // namespace gs

extern "C" {

size_t gs_adapted_linear_inner_size(int64_t rows, int64_t rank) {
  using namespace gs;
  if (rows <= 0 || rank <= 0 || rank > kMostRank) return 0;
  return Inner<float>::bytes(rows, rank);
}

int gs_adapted_linear_forward(int32_t dtype, const void* x, int64_t row_stride, const void* weight,
                              const void* bias, const void* down, const void* up, float scale,
                              const int32_t* order, const int32_t* offsets, int64_t rows,
                              int64_t groups, int64_t features, int64_t outputs, int64_t rank,
                              void* inner, size_t inner_bytes, void* y, void* stream) {
  using namespace gs;
  clear_error();
  const char* const name = "gs_adapted_linear_forward";
  GS_CHECK(check_adapted(name, dtype, offsets, rows, groups, features, outputs, rank));
  GS_CHECK(check_rows(name, dtype, rows, features, row_stride));
  GS_REQUIRE(std::isfinite(scale), GS_ERR_ARGUMENT, "%s: scale must be finite", name);
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && weight && down && up && y, GS_ERR_ARGUMENT, "null pointer passed to %s", name);
  GS_CHECK(check_inner(name, inner, inner_bytes, rows, rank));
  const Grouping g = grouping(order, offsets, rows, groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const Inner<T> held = Inner<T>::at(inner, rows, rank);
    if (rows <= kFewRows) {
      few_inner_kernel<T><<<dim3{unsigned(rows)}, kInnerThreads, 0, s>>>(
          static_cast<const T*>(x), row_stride, static_cast<const T*>(down), scale, g,
          int(features), held);
      GS_LAUNCHED(name);
      const dim3 grid{unsigned(ceil_div(outputs, kThreads / 64)), unsigned(rows)};
      few_adapted_kernel<T><<<grid, kThreads, 0, s>>>(
          static_cast<const T*>(x), row_stride, static_cast<const T*>(weight),
          static_cast<const T*>(bias), static_cast<const T*>(up), g, int(features), int(outputs),
          held, static_cast<T*>(y));
      GS_LAUNCHED(name);
      return int(GS_OK);
    }
    const Adapters<T> first{held, nullptr, scale};
    const Adapters<T> second{held, static_cast<const T*>(up), 0.f};
    bool taken = false;
    GS_CHECK((launch_rows<T, false, kInner>(name, x, row_stride, down, nullptr, g, features, rank,
                                            first, nullptr, s, taken)));
    if (!taken)
      GS_CHECK((launch_tiles<T, true, kInner>(name, x, row_stride, down, nullptr, g, features,
                                              rank, first, nullptr, s)));
    GS_CHECK((launch_rows<T, false, kAdapted>(name, x, row_stride, weight, bias, g, features,
                                              outputs, second, y, s, taken)));
    if (taken) return int(GS_OK);
    return launch_tiles<T, true, kAdapted>(name, x, row_stride, weight, bias, g, features,
                                           outputs, second, y, s);
  });
}

int gs_adapted_linear_backward_input(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                     const void* weight, const void* down, const void* up,
                                     float scale, const int32_t* order, const int32_t* offsets,
                                     int64_t rows, int64_t groups, int64_t features,
                                     int64_t outputs, int64_t rank, void* inner_grad,
                                     size_t inner_bytes, void* grad_x, void* stream) {
  using namespace gs;
  clear_error();
  const char* const name = "gs_adapted_linear_backward_input";
  GS_CHECK(check_adapted(name, dtype, offsets, rows, groups, features, outputs, rank));
  GS_CHECK(check_rows(name, dtype, rows, outputs, grad_stride));
  GS_REQUIRE(std::isfinite(scale), GS_ERR_ARGUMENT, "%s: scale must be finite", name);
  if (rows == 0) return GS_OK;
  GS_REQUIRE(grad_y && up && (!grad_x || (weight && down)), GS_ERR_ARGUMENT,
             "null pointer passed to %s", name);
  GS_CHECK(check_inner(name, inner_grad, inner_bytes, rows, rank));
  const Grouping g = grouping(order, offsets, rows, groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const Inner<T> held = Inner<T>::at(inner_grad, rows, rank);
    const Adapters<T> first{held, nullptr, scale};
    const Adapters<T> second{held, static_cast<const T*>(down), 0.f};
    bool taken = false;
    GS_CHECK((launch_rows<T, true, kInner>(name, grad_y, grad_stride, up, nullptr, g, outputs,
                                           rank, first, nullptr, s, taken)));
    if (!taken)
      GS_CHECK((launch_tiles<T, false, kInner>(name, grad_y, grad_stride, up, nullptr, g, outputs,
                                               rank, first, nullptr, s)));
    if (!grad_x) return int(GS_OK);
    GS_CHECK((launch_rows<T, true, kAdapted>(name, grad_y, grad_stride, weight, nullptr, g,
                                             outputs, features, second, grad_x, s, taken)));
    if (taken) return int(GS_OK);
    return launch_tiles<T, false, kAdapted>(name, grad_y, grad_stride, weight, nullptr, g,
                                            outputs, features, second, grad_x, s);
  });
}

size_t gs_adapted_linear_backward_adapters_workspace_size(int64_t rows, int64_t groups,
                                                          int64_t features, int64_t outputs,
                                                          int64_t rank) {
  using namespace gs;
  if (rows < 0 || rows > kMostGroupedRows || groups <= 0 || groups > kMostGroupsOfRows ||
      features <= 0 || outputs <= 0 || rank <= 0 || rank > kMostRank)
    return 0;
  const Grouping g = grouping(nullptr, nullptr, rows, groups);
  auto bytes = [&](int64_t width) {
    const int64_t shares = narrow_shares(g, width);
    return shares == 1 ? 0 : size_t(2 * shares) * size_t(rank * width) * sizeof(float);
  };
  return bytes(features) + bytes(outputs);
}

int gs_adapted_linear_backward_adapters(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                        const void* x, int64_t row_stride, const void* inner,
                                        const void* inner_grad, const int32_t* order,
                                        const int32_t* offsets, int64_t rows, int64_t groups,
                                        int64_t features, int64_t outputs, int64_t rank,
                                        void* grad_down, void* grad_up, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  using namespace gs;
  clear_error();
  const char* const name = "gs_adapted_linear_backward_adapters";
  GS_CHECK(check_adapted(name, dtype, offsets, rows, groups, features, outputs, rank));
  if (!grad_down && !grad_up) return GS_OK;
  GS_REQUIRE(offsets, GS_ERR_ARGUMENT, "null pointer passed to %s", name);
  if (grad_down) {
    GS_CHECK(check_rows(name, dtype, rows, features, row_stride));
    GS_REQUIRE(rows == 0 || (x && inner_grad), GS_ERR_ARGUMENT, "null pointer passed to %s", name);
  }
  if (grad_up) {
    GS_CHECK(check_rows(name, dtype, rows, outputs, grad_stride));
    GS_REQUIRE(rows == 0 || (grad_y && inner), GS_ERR_ARGUMENT, "null pointer passed to %s", name);
  }
  const size_t need =
      gs_adapted_linear_backward_adapters_workspace_size(rows, groups, features, outputs, rank);
  GS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), GS_ERR_WORKSPACE,
             "workspace too small for %s", name);
  const Grouping g = grouping(order, offsets, rows, groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* const partial = static_cast<float*>(workspace);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    NarrowSum<T> sums[2];
    int count = 0;
    if (grad_down)
      sums[count++] = {Inner<T>::at(const_cast<void*>(inner_grad), rows, rank),
                       static_cast<const T*>(x), row_stride, partial,
                       static_cast<T*>(grad_down), int(features), 0, 0, false};
    if (grad_up) {
      const int64_t shares = narrow_shares(g, features);
      sums[count++] = {Inner<T>::at(const_cast<void*>(inner), rows, rank),
                       static_cast<const T*>(grad_y), grad_stride,
                       partial + (shares == 1 ? 0 : 2 * shares * rank * features),
                       static_cast<T*>(grad_up), int(outputs), 0, 0, true};
    }
    return launch_narrow(name, sums, count, g, s);
  });
}

}  // extern "C"
