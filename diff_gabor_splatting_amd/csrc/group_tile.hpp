// Products of rows with the matrix of their group, a tile of 128 x 128 to a
// workgroup (50k x 128 -> 128 float16 in 512 groups: 18 us each way, bound by
// latency; 1M x 512 -> 512 bfloat16 in 32 groups: y 1,045, dx 1,171); and the
// adapters' inner rows, which such a product gives and another takes.
#pragma once

#include "groups.hpp"
#include "matrix.hpp"

namespace gs {

// --------------------------------------------------------------------------
// The adapters' inner rows: scale times x A_g^T (or dy B_g), at their positions.
//
// They are float32 sums that go into another product. For float32 they are
// kept as they are, 32 of the rank to a chunk of 128 bytes. For the 2-byte
// types a chunk has two parts of 32, each rounded to the nearest, whose sum stands
// for the value to 17 bits or (float16) 22: the matrix instructions take both, so
// the inner rounding, 2^-18 or 2^-23 of the largest, stays far below that of the
// output (one part would be a rounding as large as it). The
// rank's rest of the last chunk is zero. float16 could not hold large values, nor a
// second part of small ones: its rows are divided by a power of two
// that brings the largest value to 1/2 .. 1, and `scales` has it.
constexpr int kMostRank = 64;

// A finite value's magnitude, 0 of an infinity or a NaN.
__device__ __forceinline__ float finite_size(float v) {
  const float size = __builtin_fabsf(v);
  return size < __builtin_inff() ? size : 0.f;
}

constexpr int kInnerBytes = 128;  // of a chunk

template <typename T>
struct Inner {
  static constexpr bool scaled = std::is_same_v<T, f16>;
  T* rows;          // [positions, chunks, kInnerBytes]
  float* scales;    // [positions], float16 alone
  int rank;

  __host__ __device__ __forceinline__ int chunks() const { return (rank + 31) / 32; }
  __host__ __device__ __forceinline__ int64_t stride() const {
    return int64_t(chunks()) * (kInnerBytes / sizeof(T));
  }
  static size_t bytes(int64_t count, int64_t rank) {
    return size_t(count) * (size_t(ceil_div(rank, 32)) * kInnerBytes + sizeof(float));
  }
  static Inner at(void* memory, int64_t count, int64_t rank) {
    Inner i{static_cast<T*>(memory), nullptr, int(rank)};
    i.scales = reinterpret_cast<float*>(static_cast<char*>(memory) +
                                        size_t(count) * size_t(i.chunks()) * kInnerBytes);
    return i;
  }

  // Value n of a row, of its sum. Past the rank it is zero, and not the sum:
  // that is of products with zeros, which an infinity of the row makes NaN.
  __device__ __forceinline__ float value(int n, float sum, float scale) const {
    return n < rank ? scale * sum : 0.f;
  }
  // Writes the scale of a row (`writes`: one lane does) whose largest finite
  // magnitude is `most`; returns what its values are multiplied by.
  __device__ __forceinline__ float begin_row(int64_t position, float most, bool writes) const {
    if constexpr (scaled) {
      // most = m 2^e with 1/2 <= m < 1. Up to 2^113, so that the largest of
      // float32 comes to below 2^15; from 2^-60 on, so that the shared sum over
      // the scale stays inside float32 (2^50 at most). Both powers are normal
      // numbers.
      const int e = min(max(__builtin_amdgcn_frexp_expf(most), -60), 113);
      if (writes) scales[position] = __uint_as_float(uint32_t(127 + e) << 23);
      return __uint_as_float(uint32_t(127 - e) << 23);
    }
    return 1.f;
  }
  // Values n .. n + Count - 1 of a row, which lie in one chunk, times `up`.
  template <int Count>
  __device__ __forceinline__ void put(int64_t position, int n, const float (&v)[Count],
                                      float up) const {
    T* const to = rows + position * stride() + n / 32 * (kInnerBytes / int(sizeof(T))) + n % 32;
#pragma unroll
    for (int h = 0; h < Count; h += 4) {
      vec<T, 4> high, low;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = scaled ? v[h + j] * up : v[h + j];
        if constexpr (sizeof(T) == 4) {
          high[j] = f;
        } else {
          high[j] = T(f);
          // Cut off where bfloat16's rounding would pass its largest.
          if constexpr (!scaled)
            if (finite_size(f) > 0.f && __builtin_fabsf(float(high[j])) == __builtin_inff())
              high[j] = T(__uint_as_float(__float_as_uint(f) & 0xffff0000u));
          low[j] = finite_size(f) == __builtin_fabsf(f) ? T(f - float(high[j])) : T(0.f);
        }
      }
      *reinterpret_cast<vec<T, 4>*>(to + h) = high;
      if constexpr (sizeof(T) == 2) *reinterpret_cast<vec<T, 4>*>(to + 32 + h) = low;
    }
  }
  // Value n of a row as it is kept, but for its row's scale.
  struct Raw {
    T parts[4 / sizeof(T)];
    __device__ __forceinline__ float sum() const {
      if constexpr (sizeof(T) == 4)
        return parts[0];
      else
        return float(parts[0]) + float(parts[1]);
    }
  };
  __device__ __forceinline__ Raw raw(int64_t position, int n) const {
    const T* const from =
        rows + position * stride() + n / 32 * (kInnerBytes / int(sizeof(T))) + n % 32;
    if constexpr (sizeof(T) == 4)
      return {{from[0]}};
    else
      return {{from[0], from[32]}};
  }
  __device__ __forceinline__ float get(int64_t position, int n) const {
    const float sum = raw(position, n).sum();
    return scaled ? sum * scales[position] : sum;
  }
};

// What a product with adapters takes beside its own.
template <typename T>
struct Adapters {
  Inner<T> inner;
  const T* matrix;  // kAdapted: B_g
  float scale;      // kInner
};

// --------------------------------------------------------------------------
// The tiles

// Tiles are numbered without the groups' counts being added up: segment s
// begins at tile B / 128 + s, B its first position, which leaves it room
// enough (some numbers have no rows).
__device__ __forceinline__ int64_t tile_key(const Grouping& g, int s) {
  return begin_of(g, s) / kEdge + s;
}
inline int64_t tile_numbers(const Grouping& g) { return g.rows / kEdge + g.groups + 2; }

// A tile of rows on its way from memory to LDS, eight columns to a chunk.
template <typename T, int Columns>
struct StagedRows {
  static constexpr int across = Columns / kChunk;
  static constexpr int count = kEdge * across / kThreads;
  const T* row[count];  // null past the segment's end
  vec<T, 8> v[count];

  __device__ __forceinline__ void place(const Grouping& g, const T* data, int64_t stride,
                                        int first, int end) {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int position = first + (i * kThreads + int(threadIdx.x)) / across;
      row[i] = position < end ? data + row_at(g, position) * stride : nullptr;
    }
  }
  __device__ __forceinline__ void load(int64_t column, int64_t columns) {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int64_t c = column + (i * kThreads + threadIdx.x) % across * kChunk;
      const int64_t left = columns - c;
      v[i] = load_valid<T, 8>(row[i] + c, row[i] ? int(left < kChunk ? left : kChunk) : 0);
    }
  }
  template <int Pitch>
  __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int id = i * kThreads + threadIdx.x;
      *reinterpret_cast<vec<T, 8>*>(lds + id / across * Pitch + id % across * kChunk) = v[i];
    }
  }
};

struct GroupProduct {
  int64_t n, k;      // columns of C, length of the sum
  int64_t tiles_n;
  int64_t stride;    // of the rows
};

// What group_tile_kernel computes.
enum TileMode {
  kByGroup,  // y = x W_g (+ bias[g]), 0 for rows of no group
  kInner,    // the adapters' inner rows, scale x A_g, as an Inner
  kAdapted,  // y = x W (+ bias) + inner B_g
};

// C[i][n] = sum_k x[i][k] W_g(n, k) (+ bias[g][n]); W_g is [n][k] in memory
// (NContiguous) or [k][n]. kAdapted: the same with one W and bias, and before it
// the sum over the rank of inner[i][k] B_g(n, k), B_g laid out as W is.
template <typename T, bool NContiguous, int Mode>
__global__ __launch_bounds__(kThreads) void group_tile_kernel(
    const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ bias, Grouping g,
    GroupProduct p, Adapters<T> adapters, T* __restrict__ out) {
  constexpr int depth = Mma<T>::depth;
  __shared__ __align__(16) T m_lds[kTileSize<T, true>];
  __shared__ __align__(16) T n_lds[kTileSize<T, NContiguous>];
  const int64_t number = blockIdx.x / p.tiles_n, n0 = blockIdx.x % p.tiles_n * kEdge;
  const int s = find_segment(segments_of(g), number, [&](int i) { return tile_key(g, i); });
  const int begin = begin_of(g, s), end = begin_of(g, s + 1);
  const int64_t first64 = begin + (number - tile_key(g, s)) * kEdge;
  if (first64 < begin || first64 >= end) return;  // below only where offsets fall
  const int first = int(first64);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wave_m = (wave >> 1) * kWaveEdge, wave_n = (wave & 1) * kWaveEdge;
  const int64_t n = n0 + wave_n + 16 * (lane >> 4);
  const bool member = s > 0 && s <= g.groups;
  const int64_t group = s - 1;
  f32x4 c[kTiles][kTiles];  // [m][n]
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) c[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  StagedRows<T, depth> m_next;
  Staged<T, NContiguous ? kEdge : depth, NContiguous ? depth : kEdge> n_next;
  auto store = [&]() {
    m_next.template store<kPitch<T, true>>(m_lds);
    n_next.template store<kPitch<T, NContiguous>, true, NContiguous>(n_lds);
  };
  auto multiply_all = [&]() {
#pragma unroll
    for (int step = 0; step < depth; step += Mma<T>::step) {
      typename Mma<T>::Fragment a[kTiles], b[kTiles];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        a[i] = fragment<T, true>(m_lds, wave_m + 16 * i, step);
        b[i] = fragment<T, NContiguous>(n_lds, wave_n + 16 * i, step);
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; ++j) c[i][j] = Mma<T>::of(b[j], a[i], c[i][j]);
    }
  };

  if constexpr (Mode == kAdapted) {
    if (member) {
      // An inner row's chunk is `depth` values: 32 of the rank in float32, or
      // the two parts of 32, which both meet the same 32 of B_g.
      static_assert(depth * sizeof(T) == kInnerBytes, "a chunk is a step");
      const Inner<T>& inner = adapters.inner;
      const T* const matrix = adapters.matrix + group * p.n * inner.rank;
      const Grouping here{nullptr, g.offsets, g.rows, g.groups};
      m_next.place(here, inner.rows, inner.stride(), first, end);
      for (int chunk = 0; chunk < inner.chunks(); ++chunk) {
        m_next.load(int64_t(chunk) * depth, inner.stride());
#pragma unroll
        for (int i = 0; i < n_next.count; ++i) {
          const int id = i * kThreads + threadIdx.x;
          const int row = id / n_next.across, column = id % n_next.across * kChunk;
          if constexpr (NContiguous) {
            const int k = chunk * 32 + column % 32;
            n_next.v[i] = load_valid<T, 8>(matrix + (n0 + row) * inner.rank + k,
                                           n0 + row < p.n ? inner.rank - k : 0);
          } else {
            const int k = chunk * 32 + row % 32;
            const int64_t left = p.n - n0 - column;
            n_next.v[i] = load_valid<T, 8>(matrix + k * p.n + n0 + column,
                                           k < inner.rank ? int(left < 8 ? left : 8) : 0);
          }
        }
        store();
        __syncthreads();
        multiply_all();
        __syncthreads();
      }
      if constexpr (Inner<T>::scaled) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const int position = first + wave_m + 16 * i + (lane & 15);
          const float scale = position < end ? inner.scales[position] : 0.f;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) c[i][j] *= scale;
        }
      }
    }
  }

  float offset[16] = {};
  if (member || Mode == kAdapted) {
    const int64_t of = Mode == kAdapted ? 0 : group;
    const T* const matrix = w + of * p.n * p.k;
    const Side<T> ns{matrix, NContiguous ? p.k : p.n, NContiguous ? p.n : p.k,
                     NContiguous ? p.k : p.n};
    m_next.place(g, x, p.stride, first, end);
    auto fetch = [&](int64_t k) {
      m_next.load(k, p.k);
      if constexpr (NContiguous)
        n_next.load(ns, n0, k);
      else
        n_next.load(ns, k, n0);
    };
    fetch(0);
    for (int64_t k = 0; k < p.k; k += depth) {
      store();
      __syncthreads();
      if (k + depth < p.k) fetch(k + depth);
      multiply_all();
      __syncthreads();
    }
    if (bias) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        offset[j] = n + j < p.n ? float(bias[of * p.n + n + j]) : 0.f;
    }
  }
  // Lane 16 q + i holds, of fragment row i, the 16 columns from 16 q on.
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int64_t position = int64_t(first) + wave_m + 16 * i + (lane & 15);
    float row[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) row[j] = c[i][j >> 2][j & 3] + offset[j];
    if constexpr (Mode == kInner) {
      if (wave_n) continue;  // a rank is at most 64
      const Inner<T>& inner = adapters.inner;
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        row[j] = inner.value(int(n) + j, row[j], adapters.scale);
        most = fmaxf(most, finite_size(row[j]));
      }
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      if (position >= end) continue;
      const float up = inner.begin_row(position, most, lane >> 4 == 0);
      if (n >= 32 * inner.chunks()) continue;
      inner.template put<16>(position, int(n), row, up);
    } else {
      if (position >= end) continue;
      store_row<T>(out + row_at(g, int(position)) * p.n + n, p.n - n, row);
    }
  }
}

}  // namespace gs
