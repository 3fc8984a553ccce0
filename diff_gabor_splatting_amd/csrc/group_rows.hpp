// Products of rows with the matrix of their group, the matrix in LDS and the
// rows streamed past it; and the products with the adapters' inner rows.
#pragma once

#include "group_tile.hpp"

namespace gs {

// A workgroup takes a panel of the columns and a share of the rows, whatever
// groups they are in, and puts another matrix in place where another group
// begins; a wave takes 32 rows at a time and, but for that, needs no other
// wave. Shares are cut from the line on which each segment takes kStageCost +
// its rows, so that putting a matrix in place counts too (64 to 1,024 rows give
// the same times).
//
// 1M x 512 -> 512 bfloat16 in 32 groups: y 613 us, dx 591 (850 to 890 TFLOP/s),
// as long as with one matrix for all rows: matrix cores 40% busy, LDS 46%, the
// address unit 64%. With the adapters' steps (rank 16) 665 and 654; inner rows
// 242 and 254, bound by the address unit (80%).
constexpr int64_t kStageCost = 64;  // of a matrix, in rows

__device__ __forceinline__ int64_t stage_line(const Grouping& g, int s) {
  return begin_of(g, s) + kStageCost * s;
}

struct GroupRows {
  int64_t stride;
  int k, n;          // length of the sum and columns of C
  int panels;        // workgroups side by side, each with its columns of C
  int workers;       // workgroups to a panel, 32 / panels to an XCD at most: with
                     // 17 panels 15 of its compute units have none
  int steps;         // of the sum, of 128 bytes of a row
  int all;           // those, the adapters' chunks, and as many as make the
                     // whole a multiple of those under way
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
                                          f32x4 (&c)[TN]) {
  const int q = (threadIdx.x & 63) >> 4;
  const Inner<T>& inner = adapters.inner;
  float most = 0.f;
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[t][j] = inner.value(panel_column<T>(t, 4 * q) + j, c[t][j], adapters.scale);
      most = fmaxf(most, finite_size(c[t][j]));
    }
  if constexpr (Inner<T>::scaled) {
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
  }
  if (position >= end) return;
  const float up = inner.begin_row(position, most, q == 0);
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    const int n = panel_column<T>(t, 4 * q);
    if (n >= 32 * inner.chunks()) continue;
    const float four[4] = {c[t][0], c[t][1], c[t][2], c[t][3]};
    inner.template put<4>(position, n, four, up);
  }
}

// The adapter's matrix of a group, [n][rank] or (Transposed) [rank][n], as
// fragments beside those of the panel: one to 16 columns and chunk for the
// 2-byte types, whose two parts of an inner row meet the same values, two for
// float32. Without `some` it is zeros.
template <typename T, int TN, bool Transposed>
__device__ __forceinline__ void stage_adapter(const T* __restrict__ matrix, bool some, int n,
                                              int rank, int chunks, int n0,
                                              vec<T, kPart<T>>* lds) {
  constexpr int part = kPart<T>, columns = 16 * TN;
  const int parts = chunks * (32 / part);
  auto place = [&](int column, int c) {
    const FragmentPlace to = place_in_panel<T>(column);
    return ((c >> 2) * TN + to.t) * 64 + (c & 3) * 16 + to.i;
  };
  if constexpr (!Transposed) {
    for (int id = threadIdx.x; id < columns * parts; id += kRowThreads) {
      const int column = id / parts, c = id - column * parts;
      lds[place(column, c)] =
          load_valid<T, part>(matrix + int64_t(n0 + column) * rank + c * part,
                              some && n0 + column < n ? rank - c * part : 0);
    }
  } else {
    // Four columns of `part` ranks at a time, turned in registers.
    for (int id = threadIdx.x; id < columns / 4 * parts; id += kRowThreads) {
      const int c = id / (columns / 4), column = 4 * (id - c * (columns / 4));
      vec<T, 4> v[part];
#pragma unroll
      for (int j = 0; j < part; ++j) {
        const int k = c * part + j;
        v[j] = load_valid<T, 4>(matrix + int64_t(k) * n + n0 + column,
                                some && k < rank ? n - n0 - column : 0);
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        vec<T, part> turned;
#pragma unroll
        for (int j = 0; j < part; ++j) turned[j] = v[j][b];
        lds[place(column, c) + b] = turned;
      }
    }
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

  bool staged = false;
  int s = find_segment(segments_of(g), from_line, [&](int i) { return stage_line(g, i); });
  for (; s < segments_of(g) && stage_line(g, s) < to_line; ++s) {
    const int low = begin_of(g, s), high = max(begin_of(g, s + 1), low);
    const int first = cut_at(from_line, s, low, high), end = cut_at(to_line, s, low, high);
    if (first >= end) continue;
    const bool member = s > 0 && s <= g.groups;
    if (Mode == kInner && !member) {
      const Inner<T>& inner = adapters.inner;
      const int fours = 8 * inner.chunks();
      const float none[4] = {};
      for (int64_t id = threadIdx.x; id < int64_t(end - first) * fours; id += kRowThreads) {
        const int64_t position = first + id / fours;
        const int n = int(id % fours) * 4;
        inner.template put<4>(position, n, none, inner.begin_row(position, 0.f, n == 0));
      }
      continue;
    }
    if (Mode == kByGroup && !member) {
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
    // The rows' places are asked for a tile before they are needed; lane i
    // has that of the tile's row i % 32.
    auto places = [&](int tile) {  // positions past the end repeat the last one
      return int(row_at(g, min(first + tile * kRowTile + (lane & 31), end - 1)));
    };
    int sent = min(wave, tiles - 1), sent_step = 0;
    int sent_rows = places(sent), now = sent_rows;
    int after = places(min(sent + kRowWaves, tiles - 1));
    const T* from[loads];
    auto turn_to = [&]() {
#pragma unroll
      for (int j = 0; j < loads; ++j)
        from[j] = x + __shfl(sent_rows, 8 * j + row8) * p.stride + piece * part;
    };
    auto send = [&](Part (&to)[loads]) {
      if (sent_step == p.all) {
        sent_step = 0;
        if (sent + kRowWaves < tiles) {
          sent += kRowWaves;
          sent_rows = after;
        }
        turn_to();
        after = places(min(sent + kRowWaves, tiles - 1));
      }
      if (Mode == kAdapted && sent_step >= p.steps) {
        const int chunk = min(sent_step - p.steps, adapters.inner.chunks() - 1);
        const int in_tile = first + sent * kRowTile;
        const T* const rows = adapters.inner.rows + in_tile * adapters.inner.stride() +
                              (chunk * kInnerBytes) / int(sizeof(T));
        const int last = min(end - in_tile, kRowTile) - 1;
#pragma unroll
        for (int j = 0; j < loads; ++j)
          to[j] = load_packed<T, part>(
              rows + uint32_t(min(8 * j + row8, last) * int(adapters.inner.stride()) +
                              piece * part));
      } else if (!Tail || (sent_step + 1) * step <= p.k) {
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
    turn_to();

    // The matrix, once no wave reads the one before; the shared one of
    // kAdapted once.
    __syncthreads();
    if (Mode != kAdapted || !staged) {
      const int64_t of = Mode == kAdapted ? 0 : s - 1;
      stage_panel<T, TN, Transposed>(w + of * p.n * p.k, p.k, p.n, p.steps, n0, panel);
      if (Mode != kInner && threadIdx.x < columns)
        offset[threadIdx.x] = bias && n0 + int(threadIdx.x) < p.n
                                  ? float(bias[of * p.n + n0 + threadIdx.x])
                                  : 0.f;
      staged = true;
    }
    Part* const narrow = panel + p.steps * 2 * TN * 64;
    if constexpr (Mode == kAdapted) {
      const int rank = adapters.inner.rank;
      // Rows of no group meet zeros.
      stage_adapter<T, TN, Transposed>(
          adapters.matrix + int64_t(member ? s - 1 : 0) * p.n * rank, member, p.n, rank,
          adapters.inner.chunks(), n0, narrow);
    }
#pragma unroll
    for (int u = 0; u < Ahead; ++u) send(ring[u]);
    __syncthreads();

    for (int tile = wave; tile < tiles; tile += kRowWaves) {
      f32x4 c[TM][TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) c[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      float scale[TM];
      if constexpr (Mode == kAdapted && Inner<T>::scaled) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
          scale[i] = adapters.inner.scales[min(first + tile * kRowTile + 16 * i + i16, end - 1)];
      }
      for (int s0 = 0; s0 < p.all; s0 += Ahead) {
#pragma unroll
        for (int u = 0; u < Ahead; ++u) {
          const int st = s0 + u;
          if (Tail && (st + 1) * step > p.k && (Mode != kAdapted || st < p.steps)) {
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
          // Where the step's fragments lie, and those of its second half.
          const Part* fragments = panel + 2 * st * TN * 64 + lane;
          int second = TN * 64;
          if constexpr (Mode == kAdapted) {
            const int chunk = st - p.steps;
            if (chunk >= adapters.inner.chunks()) continue;
            if (chunk >= 0) {
              if constexpr (sizeof(T) == 2) {
                fragments = narrow + chunk * TN * 64 + lane;
                second = 0;
              }
              if (Inner<T>::scaled && chunk == 0) {
                // Powers of two: what is lost of the sum is below 2^-149 of a
                // scale of at most 2^113, far below float16's own steps.
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                  for (int t = 0; t < TN; ++t) c[i][t] *= 1.f / scale[i];
              }
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < TN; ++t) {
              const Part a = fragments[h * second + t * 64];
#pragma unroll
              for (int i = 0; i < TM; ++i) c[i][t] = multiply<T>(a, b[i][h], c[i][t]);
            }
        }
      }
      if constexpr (Mode == kAdapted && Inner<T>::scaled) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int t = 0; t < TN; ++t) c[i][t] *= scale[i];
      }
      if constexpr (Mode == kInner) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
          put_inner<T, TN>(adapters, first + tile * kRowTile + 16 * i + i16, end, c[i]);
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
            store_valid<T, part>(out + int64_t(__shfl(now, 16 * i + 8 * j + row8)) * p.n + n,
                                 row ? inside : 0, r);
          }
          wave_order();
        }
      }
        now = sent_rows;
      }
    }
  }
}

}  // namespace gs
