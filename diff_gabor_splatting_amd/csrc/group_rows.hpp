// Products of rows with the matrix of their group, the matrix in LDS and the
// rows streamed past it; and the products with the adapters' inner rows.
#pragma once

#include "group_tile.hpp"

namespace gs {

// A workgroup takes a panel of the columns and a share of the rows, whatever
// groups they are in, and puts another matrix in place where another group
// begins; a wave takes 32 rows at a time and, but for that, needs no other
// wave. Shares are cut from the line on which each segment takes kStageCost +
// its rows, so that putting a matrix in place counts too.
constexpr int64_t kStageCost = 64;  // of a matrix, in rows

__device__ __forceinline__ int64_t stage_line(const Grouping& g, int s) {
  return begin_of(g, s) + kStageCost * s;
}

struct GroupRows {
  int64_t stride;
  int k, n;          // length of the sum and columns of C
  int panels;        // workgroups side by side, each with its columns of C
  int workers;       // workgroups to a panel
  int steps;         // of the sum, see steps_of
};

// Where the line's place v lies in segment s, as a position: from the
// segment's begin on a whole number of tiles, so that the shares on both sides
// of it agree and few tiles are partly filled.
__device__ __forceinline__ int cut_at(int64_t v, int s, int low, int high) {
  const int64_t into = v - kStageCost * (s + 1) - low;
  if (into <= 0) return low;
  const int64_t up = (into + kRowTile - 1) / kRowTile * kRowTile;
  return up < high - low ? low + int(up) : high;
}

// Column of a panel that row i of fragment t is, and the first of the four that
// lane group q receives of it: place_in_panel the other way round.
template <typename T>
__device__ __forceinline__ int panel_column(int t, int i) {
  if constexpr (sizeof(T) == 4)
    return 16 * t + i;
  else
    return 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
}

// Sixteen rows' columns as inner rows: lane 16 q + i has row i.
template <typename T, int TN>
__device__ __forceinline__ void put_inner(const Adapters<T>& adapters, int position, int end,
                                          int group, f32x4 (&c)[TN]) {
  const int q = (threadIdx.x & 63) >> 4;
  const Inner<T>& inner = adapters.inner;
  float most = 0.f;
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[t][j] *= adapters.scale;
      most = fmaxf(most, finite_size(c[t][j]));
    }
  if constexpr (Inner<T>::scaled) {
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
  }
  if (position >= end) return;
  const float up = inner.begin_row(position, most, group, q == 0);
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    const int n = panel_column<T>(t, 4 * q);
    if (n >= 32 * inner.chunks()) continue;
    const float four[4] = {c[t][0], c[t][1], c[t][2], c[t][3]};
    inner.template put<4>(position, n, four, up);
  }
}

// Adds inner B_g to a wave's tile, whose first row is at `first`. The tile's
// rows may be of several groups: each group's product is taken with the
// others' inner rows as zeros, which costs 4 matrix instructions to a
// fragment of columns where the tile's own product has `steps` times that.
template <typename T, int TN>
__device__ __forceinline__ void add_adapters(const Adapters<T>& adapters, const Grouping& g,
                                             const GroupRows& p, int first, int end, int n0,
                                             f32x4 (&c)[kRowTile / 16][TN]) {
  constexpr int TM = kRowTile / 16, part = kPart<T>;
  typedef vec<T, part> Part;
  const Inner<T>& inner = adapters.inner;
  const int lane = threadIdx.x & 63, q = lane >> 4, i16 = lane & 15;
  int position[TM], group[TM];
  float scale[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int at = first + 16 * i + i16;
    position[i] = min(at, end - 1);
    group[i] = at < end ? inner.groups[position[i]] : -1;
    if constexpr (Inner<T>::scaled) scale[i] = inner.scales[position[i]];
  }
  if constexpr (Inner<T>::scaled) {
    // Powers of two, and far enough inside float32.
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int t = 0; t < TN; ++t) c[i][t] *= 1.f / scale[i];
  }
  for (int chunk = 0; chunk < inner.chunks(); ++chunk) {
    Part b[TM][2];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b[i][h] = *reinterpret_cast<const Part*>(
            inner.rows + position[i] * inner.stride() +
            (chunk * kInnerBytes + h * 64 + q * 16) / int(sizeof(T)));
    bool left[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) left[i] = group[i] >= 0;
    for (;;) {
      // The next group of the tile's rows.
      int of = -1;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const uint64_t lanes = __ballot(left[i]);
        if (of < 0 && lanes)
          of = __builtin_amdgcn_readlane(group[i], int(__builtin_ctzll(lanes)));
      }
      if (of < 0) break;
      Part mine[TM][2];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const bool here = group[i] == of;
        left[i] = left[i] && !here;
#pragma unroll
        for (int h = 0; h < 2; ++h) mine[i][h] = here ? b[i][h] : Part(T(0));
      }
      const T* const matrix = adapters.matrix + int64_t(of) * p.n * inner.rank;
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        const int n = n0 + panel_column<T>(t, i16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // The two parts of the 2-byte types meet the same values.
          const int k = 32 * chunk + part * q + (sizeof(T) == 4 ? 16 * h : 0);
          Part a;
          if (sizeof(T) == 4 || h == 0)
            a = load_valid<T, part>(matrix + int64_t(n) * inner.rank + k,
                                    n < p.n ? inner.rank - k : 0);
#pragma unroll
          for (int i = 0; i < TM; ++i) c[i][t] = multiply<T>(a, mine[i][h], c[i][t]);
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < TM; ++i) c[i][t] = multiply<T>(a, mine[i][1], c[i][t]);
            break;
          }
        }
      }
    }
  }
  if constexpr (Inner<T>::scaled) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int t = 0; t < TN; ++t) c[i][t] *= scale[i];
  }
}

// Ahead: steps on their way. Tail: k is no whole number of steps.
template <typename T, int TN, int Ahead, bool Transposed, bool Tail, int Mode>
__global__ __launch_bounds__(kRowThreads) void group_rows_kernel(
    const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ bias, Grouping g,
    GroupRows p, Adapters<T> adapters, T* __restrict__ out) {
  constexpr int TM = kRowTile / 16;
  constexpr int part = kPart<T>, step = kStep<T>, columns = 16 * TN;
  constexpr int loads = 2 * TM;  // of eight rows each
  typedef vec<T, part> Part;
  extern __shared__ __align__(16) char shared[];
  Part* const panel = reinterpret_cast<Part*>(shared);
  __shared__ Part turns[kRowWaves][128];
  __shared__ float offset[columns];
  // Workgroups go to the eight XCDs in turn: those that take the same rows
  // share one, and its L2.
  const int xcd = blockIdx.x & 7, in_xcd = blockIdx.x >> 3;
  const int at = in_xcd % p.panels;
  const int worker = in_xcd / p.panels * 8 + xcd;
  if (worker >= p.workers) return;
  const int n0 = at * columns;
  const int64_t length = g.rows + kStageCost * segments_of(g);
  const int64_t from_line = length * worker / p.workers;
  const int64_t to_line = length * (worker + 1) / p.workers;

  const int lane = threadIdx.x & 63, q = lane >> 4, i16 = lane & 15;
  const int row8 = lane >> 3, piece = lane & 7;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Part* const turn = turns[wave];

  int s = Mode == kAdapted
              ? 1
              : find_segment(segments_of(g), from_line, [&](int i) { return stage_line(g, i); });
  for (; Mode == kAdapted ? s == 1 : s < segments_of(g) && stage_line(g, s) < to_line; ++s) {
    int first, end;
    if constexpr (Mode == kAdapted) {  // one matrix for all rows
      first = cut_at(int64_t(g.rows) * worker / p.workers, -1, 0, g.rows);
      end = cut_at(int64_t(g.rows) * (worker + 1) / p.workers, -1, 0, g.rows);
    } else {
      const int low = begin_of(g, s), high = max(begin_of(g, s + 1), low);
      first = cut_at(from_line, s, low, high);
      end = cut_at(to_line, s, low, high);
    }
    if (first >= end) continue;
    if (Mode == kInner && (s == 0 || s > g.groups)) {
      for (int64_t id = threadIdx.x; id < end - first; id += kRowThreads)
        adapters.inner.begin_row(first + id, 0.f, -1, true);
      continue;  // nothing reads the rest
    }
    if (Mode == kByGroup && (s == 0 || s > g.groups)) {  // rows of no group
      constexpr int pieces = columns / part;
      for (int64_t id = threadIdx.x; id < int64_t(end - first) * pieces; id += kRowThreads) {
        const int n = n0 + int(id % pieces) * part;
        store_valid<T, part>(out + row_at(g, first + int(id / pieces)) * p.n + n,
                             min(p.n - n, part), Part(T(0)));
      }
      continue;
    }
    const int tiles = (end - first + kRowTile - 1) / kRowTile;

    // What is on its way: the loop below takes ring[u] and sends for the step
    // `Ahead` later in its place. Past the wave's last tile it sends for that
    // one again, so that the number of loads under way is always the same.
    // The rows' places are asked for a tile before they are needed.
    int now[loads], sent_rows[loads], after[loads];
    auto places = [&](int tile, int (&to)[loads]) {
#pragma unroll
      for (int j = 0; j < loads; ++j)  // positions past the end repeat the last one
        to[j] = int(row_at(g, min(first + tile * kRowTile + 8 * j + row8, end - 1)));
    };
    const T* from[loads];
    auto turn_to = [&]() {
#pragma unroll
      for (int j = 0; j < loads; ++j) from[j] = x + sent_rows[j] * p.stride + piece * part;
    };
    int sent = min(wave, tiles - 1), sent_step = 0;
    auto send = [&](Part (&to)[loads]) {
      if (sent_step == p.steps) {
        sent_step = 0;
        if (sent + kRowWaves < tiles) {
          sent += kRowWaves;
#pragma unroll
          for (int j = 0; j < loads; ++j) sent_rows[j] = after[j];
        }
        turn_to();
        places(min(sent + kRowWaves, tiles - 1), after);
      }
      if (!Tail || (sent_step + 1) * step <= p.k) {
#pragma unroll
        for (int j = 0; j < loads; ++j)
          to[j] = load_packed<T, part>(from[j] + sent_step * step);
      } else {
        const int left = min(p.k - sent_step * step - piece * part, part);
#pragma unroll
        for (int j = 0; j < loads; ++j)
          to[j] = load_edge<T, part, false>(from[j] + sent_step * step, left);
      }
      ++sent_step;
    };
    Part ring[Ahead][loads];
    places(sent, sent_rows);
    places(min(sent + kRowWaves, tiles - 1), after);
#pragma unroll
    for (int j = 0; j < loads; ++j) now[j] = sent_rows[j];
    turn_to();

    // The matrix, once no wave reads the one before.
    __syncthreads();
    stage_panel<T, TN, Transposed>(w + int64_t(s - 1) * p.n * p.k, p.k, p.n, p.steps, n0, panel);
    if (threadIdx.x < columns)
      offset[threadIdx.x] = bias && n0 + int(threadIdx.x) < p.n
                                ? float(bias[int64_t(s - 1) * p.n + n0 + threadIdx.x])
                                : 0.f;
#pragma unroll
    for (int u = 0; u < Ahead; ++u) send(ring[u]);
    __syncthreads();

    for (int tile = wave; tile < tiles; tile += kRowWaves) {
      f32x4 c[TM][TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) c[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int s0 = 0; s0 < p.steps; s0 += Ahead) {
#pragma unroll
        for (int u = 0; u < Ahead; ++u) {
          const int st = s0 + u;
          if (Tail && (st + 1) * step > p.k) {
            const int left = min(p.k - st * step - piece * part, part);
#pragma unroll
            for (int j = 0; j < loads; ++j) ring[u][j] = settle<T, part, false>(ring[u][j], left);
          }
          Part b[TM][2];
#pragma unroll
          for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              turn[turn_place(8 * j + row8, piece >> 2, piece & 3)] = ring[u][2 * i + j];
            wave_order();
#pragma unroll
            for (int h = 0; h < 2; ++h) b[i][h] = turn[turn_place(i16, h, q)];
            wave_order();
          }
          send(ring[u]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < TN; ++t) {
              const Part a = panel[((2 * st + h) * TN + t) * 64 + lane];
#pragma unroll
              for (int i = 0; i < TM; ++i) c[i][t] = multiply<T>(a, b[i][h], c[i][t]);
            }
        }
      }
      if constexpr (Mode == kAdapted)
        add_adapters<T, TN>(adapters, g, p, first + tile * kRowTile, end, n0, c);
      if constexpr (Mode == kInner) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
          put_inner<T, TN>(adapters, first + tile * kRowTile + 16 * i + i16, end, s - 1, c[i]);
      }
      if constexpr (Mode != kInner) {
      // Lane group q has, of every 64 bytes of the columns, the q-th 16.
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int v = 0; v < 4 * TN; v += 2 * part) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            Part r;
#pragma unroll
            for (int j = 0; j < part; ++j) {
              const int from_fragment = v + h * part + j;
              r[j] = T(c[i][from_fragment >> 2][j & 3] +
                       offset[4 * (v + h * part) + q * part + j]);
            }
            turn[turn_place(i16, h, q)] = r;
          }
          wave_order();
          const int n = n0 + 4 * v + piece * part;
          const int inside = min(p.n - n, part);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const bool row = first + tile * kRowTile + 16 * i + 8 * j + row8 < end;
            const Part r = turn[turn_place(8 * j + row8, piece >> 2, piece & 3)];
            store_valid<T, part>(out + int64_t(now[2 * i + j]) * p.n + n, row ? inside : 0, r);
          }
          wave_order();
        }
      }
#pragma unroll
      for (int j = 0; j < loads; ++j) now[j] = sent_rows[j];
      }
    }
  }
}

}  // namespace gs
