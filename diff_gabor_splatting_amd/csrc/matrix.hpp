// What the kernels that multiply matrices share: the matrix instructions of the
// three types, tiles on their way from memory to LDS, and a matrix laid out in
// LDS as the instructions' fragments.
#pragma once

#include "kept8.hpp"
#include "layers_api.hpp"

namespace gs {

constexpr int kThreads = 256;
constexpr int kEdge = 128;   // a workgroup's tile of C is 128 x 128
constexpr int kWaveEdge = 64;  // a wave's is 64 x 64
constexpr int kTiles = kWaveEdge / 16;

typedef vec<float, 4> f32x4;

// Matrix instruction of a type: `step` values of k at a time. A fragment's
// values of lane group q = lane / 16 are those at k = 4 q .. 4 q + 3 (and
// 16 more for the 2-byte types' second half): any order of k does, as long
// as both sides have the same.
template <typename T>
struct Mma {
  static constexpr int step = 32, depth = 64;
  using Fragment = vec<T, 8>;
  static __device__ __forceinline__ f32x4 of(Fragment a, Fragment b, f32x4 c) {
    if constexpr (std::is_same_v<T, bf16>)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  static constexpr int step = 16, depth = 32;
  using Fragment = vec<float, 4>;
  static __device__ __forceinline__ f32x4 of(Fragment a, Fragment b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// LDS rows. Contiguous k: `depth` values and a pad that spreads the 16 rows
// of a fragment over the banks. Otherwise the tile's edge and such a pad.
template <typename T, bool KContiguous>
constexpr int kPitch = KContiguous ? Mma<T>::depth + (sizeof(T) == 2 ? 8 : 4)
                                   : kEdge + (sizeof(T) == 2 ? 16 : 4);

template <typename T, bool KContiguous>
constexpr int kTileSize = kPitch<T, KContiguous> * (KContiguous ? kEdge : Mma<T>::depth);

// Place of column n of the N side in its LDS tile: within 64 columns, the 16
// of fragment t are n = 16 c + 4 t + 0..3, so that a lane's results of the
// four fragments are 16 consecutive columns.
__device__ __forceinline__ int place_of(int n) {
  return (n & ~63) + 16 * ((n >> 2) & 3) + 4 * ((n >> 4) & 3) + (n & 3);
}

// A side in memory: rows x columns.
template <typename T>
struct Side {
  const T* data;
  int64_t stride;
  int64_t rows, columns;
};

// A tile of a side on its way from memory to LDS, eight columns to a chunk:
// Rows x Columns from (row, column) on, zero outside the side.
template <typename T, int Rows, int Columns>
struct Staged {
  static constexpr int count = Rows * Columns / kChunk / kThreads;
  static constexpr int across = Columns / kChunk;
  vec<T, 8> v[count];

  __device__ __forceinline__ void load(const Side<T>& s, int64_t row, int64_t column) {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int id = i * kThreads + threadIdx.x;
      const int64_t r = row + id / across, c = column + (id % across) * kChunk;
      const int64_t left = s.columns - c;
      v[i] = load_valid<T, 8>(s.data + r * s.stride + c,
                              r < s.rows ? int(left < kChunk ? left : kChunk) : 0);
    }
  }

  // Order: whether the columns (or, with contiguous k, the rows) are those of
  // the N side, in place_of's order.
  template <int Pitch, bool Order, bool KContiguous>
  __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int id = i * kThreads + threadIdx.x;
      const int r = id / across, c = (id % across) * kChunk;
      if constexpr (Order && !KContiguous) {
        const vec<T, 4> low = {v[i][0], v[i][1], v[i][2], v[i][3]};
        const vec<T, 4> high = {v[i][4], v[i][5], v[i][6], v[i][7]};
        *reinterpret_cast<vec<T, 4>*>(lds + r * Pitch + place_of(c)) = low;
        *reinterpret_cast<vec<T, 4>*>(lds + r * Pitch + place_of(c + 4)) = high;
      } else {
        const int at = Order ? place_of(r) : r;
        *reinterpret_cast<vec<T, 8>*>(lds + at * Pitch + c) = v[i];
      }
    }
  }
};

// Fragment of the 16 places from `first` on, k from `k` on.
template <typename T, bool KContiguous>
__device__ __forceinline__ typename Mma<T>::Fragment fragment(const T* lds, int first, int k) {
  constexpr int pitch = kPitch<T, KContiguous>;
  const int lane = threadIdx.x & 63, q = lane >> 4, i = lane & 15;
  if constexpr (KContiguous) {
    const T* p = lds + (first + i) * pitch + k + 4 * q;
    if constexpr (sizeof(T) == 2) {
      const vec<T, 4> low = *reinterpret_cast<const vec<T, 4>*>(p);
      const vec<T, 4> high = *reinterpret_cast<const vec<T, 4>*>(p + 16);
      return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *reinterpret_cast<const vec<T, 4>*>(p);
    }
  } else if constexpr (sizeof(T) == 2) {
    // The transposing load: among 16 lanes, lane 4 a + b reads four columns
    // at 4 b of row a, and lane i receives column i of the four rows.
    typedef vec<short, 4> raw;
    const T* p = lds + (k + 4 * q + (i >> 2)) * pitch + first + 4 * (i & 3);
    typedef __attribute__((address_space(3))) raw* lds_raw;
    const raw low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_raw)p);
    const raw high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_raw)(p + 16 * pitch));
    const vec<short, 8> both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Mma<T>::Fragment, both);
  } else {
    const T* p = lds + (k + 4 * q) * pitch + first + i;
    return vec<T, 4>{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
  }
}

// Columns [n, n + 16) of a row of C, `left` of them inside.
template <typename T>
__device__ __forceinline__ void store_row(T* p, int64_t left, const float (&c)[16]) {
#pragma unroll
  for (int h = 0; h < 16; h += 8) {
    vec<T, 8> raw;
#pragma unroll
    for (int j = 0; j < 8; ++j) raw[j] = T(c[h + j]);
    store_valid<T, 8>(p + h, int(left - h < 8 ? left - h : 8), raw);
  }
}

// --------------------------------------------------------------------------
// A matrix in LDS, rows streamed past it

// Contiguous values of k in a lane's fragment, and in a step.
template <typename T>
constexpr int kPart = 16 / sizeof(T);
template <typename T>
constexpr int kStep = 8 * kPart<T>;  // two fragments: 128 bytes of a row

constexpr int kRowThreads = 512;  // eight waves: what 256 registers allow
constexpr int kRowWaves = kRowThreads / 64;
constexpr size_t kRowLds = 128 * 1024;  // of the matrix

template <typename T>
__device__ __forceinline__ f32x4 multiply(vec<T, kPart<T>> a, vec<T, kPart<T>> b, f32x4 c) {
  return Mma<T>::of(a, b, c);
}

// Where column n of a panel is among its fragments: fragment t, row i. Lane
// group q receives rows 4 q .. 4 q + 3 of each fragment. float32: fragment t
// is the columns from 16 t on. 2-byte types: two fragments are 32 columns, of
// which lane group q receives eight in succession, so that a store of 16
// bytes a lane writes 64 bytes together either way.
struct FragmentPlace {
  int t, i;
};
template <typename T>
__device__ __forceinline__ FragmentPlace place_in_panel(int n) {
  if constexpr (sizeof(T) == 4)
    return {n >> 4, n & 15};
  else
    return {2 * (n >> 5) + ((n >> 2) & 1), 4 * ((n >> 3) & 3) + (n & 3)};
}

// The matrix as fragments. Transposed: `w` is [k][n] in memory, else [n][k].
template <typename T, int TN, bool Transposed>
__device__ __forceinline__ void stage_panel(const T* __restrict__ w, int wk, int wn, int steps,
                                            int n0, vec<T, kPart<T>>* lds) {
  constexpr int part = kPart<T>, columns = 16 * TN;
  const int parts = steps * 8;
  if constexpr (!Transposed) {
    for (int id = threadIdx.x; id < columns * parts; id += kRowThreads) {
      const int n = id / parts, c = id - n * parts, k = c * part;
      const int left = wk - k;
      const vec<T, part> v =
          load_valid<T, part>(w + int64_t(n0 + n) * wk + k,
                              n0 + n < wn ? (left < part ? left : part) : 0);
      const FragmentPlace to = place_in_panel<T>(n);
      lds[((c >> 2) * TN + to.t) * 64 + (c & 3) * 16 + to.i] = v;
    }
  } else {
    // Four columns of `part` rows at a time, turned in registers.
    for (int id = threadIdx.x; id < columns / 4 * parts; id += kRowThreads) {
      const int c = id / (columns / 4), g = id - c * (columns / 4);
      const int n = n0 + 4 * g, left = wn - n;
      vec<T, 4> v[part];
#pragma unroll
      for (int j = 0; j < part; ++j) {
        const int k = c * part + j;
        v[j] = load_valid<T, 4>(w + int64_t(k) * wn + n,
                                k < wk ? (left < 4 ? left : 4) : 0);
      }
      const FragmentPlace to = place_in_panel<T>(4 * g);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        vec<T, part> turned;
#pragma unroll
        for (int j = 0; j < part; ++j) turned[j] = v[j][b];
        lds[((c >> 2) * TN + to.t) * 64 + (c & 3) * 16 + to.i + b] = turned;
      }
    }
  }
}

// Place, among a wave's 128 pieces of 16 bytes, of piece c (of four) of half
// h (of two) of row r (of 16). LDS serves eight lanes of 16 bytes at a time:
// a row's eight pieces when written, and when read 4 lanes of one lane group
// with 4 of the next, rows 0..3 of eight with rows 4..7; neither meet in a
// bank.
__device__ __forceinline__ int turn_place(int r, int h, int c) {
  return h * 64 + c * 16 + (r ^ (4 * h + c));
}

// Steps that are under way at a time, and steps of the sum: a multiple of
// them (the steps past k multiply zeros).
inline int ahead_of(int64_t steps) { return steps == 1 ? 1 : steps % 4 == 0 ? 4 : 2; }
inline int64_t steps_of(size_t size, int64_t k) {
  const int64_t steps = ceil_div(k * int64_t(size), 128);
  return steps > 1 ? steps + steps % 2 : steps;
}


// Rows of a wave's tile, and fragments side by side of a panel of the matrix:
// the widest panel that its k leaves room for in LDS, no wider than the
// columns of C ask for, at least 128 bytes of a row of C; 0 where that does
// not fit. With few rows, narrower ones, while that gives more workgroups (up
// to one per compute unit) less to put in place.
constexpr int kRowTile = 32;
inline int panel_fragments(size_t size, int64_t rows, int64_t k, int64_t n) {
  const int least = size == 4 ? 2 : 4;
  int fragments = 8;
  while (fragments >= least && steps_of(size, k) * 2048 * fragments > int64_t(kRowLds))
    fragments /= 2;
  if (fragments < least) return 0;
  const int64_t tiles = ceil_div(rows, kRowTile);
  while (fragments > least &&
         (n <= 8 * fragments || tiles * ceil_div(n, 8 * fragments) <= 256))
    fragments /= 2;
  return fragments;
}

// --------------------------------------------------------------------------
// Sums over rows

// The 16 columns from `first` on of 32 rows of LDS, as a fragment.
template <typename F>
__device__ __forceinline__ vec<F, 8> turned_fragment(const F* lds, int pitch, int first) {
  typedef vec<short, 4> raw;
  typedef __attribute__((address_space(3))) raw* lds_raw;
  const int lane = threadIdx.x & 63, q = lane >> 4, i = lane & 15;
  // Among 16 lanes, lane 4 a + b reads four columns at 4 b of row a, and
  // lane i receives column i of the four rows.
  const F* const p = lds + (4 * q + (i >> 2)) * pitch + first + 4 * (i & 3);
  const raw low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_raw)p);
  const raw high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_raw)(p + 16 * pitch));
  return __builtin_bit_cast(vec<F, 8>, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
}

}  // namespace gs
