// Linear layers whose input is kept in 8 bits: y = x W^T + b and its
// gradients dx = dy W, dW = dy^T x8, db = the sum of dy's rows, x8 what the
// checkpoint stands for.
//
// All three products are one tiled kernel: C[m][n] = sum_k M(m,k) N(n,k), on
// the matrix cores with float32 accumulators (16x16x32 for the 2-byte types,
// 16x16x4 for float32). A side whose k is the contiguous dimension in memory
// is staged in LDS as it lies; one whose m or n is (W in dx, both sides of
// dW) is staged row by row too, and the 2-byte types' fragments are read
// with the transposing LDS load. What is kept in 8 bits is expanded while it
// is staged: q 2^e is exact in each type.
//
//                M side             N side               k
//   y    rows    x  [m][k]          W  [n][k]            features
//   dx   rows    dy [m][k]          W  [k][n]            outputs
//   dW   outputs dy [k][m]          x8 [k][n]            rows, split
//
// dW's k is long and its C small: the rows are split over workgroups, each
// writes a float32 partial C, and a second kernel adds the partials in their
// order (no atomics: results do not depend on timing).
#include "kept8.hpp"
#include "layers_api.hpp"

namespace gs {
namespace {

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

// A side in memory: rows x columns of T, or of the 8-bit form.
template <typename T>
struct Side {
  const T* data;
  int64_t stride;
  int64_t rows, columns;
};
struct KeptSide {
  const uint8_t* values;
  const uint8_t* exponents;
  int64_t groups;
  int64_t rows, columns;
};

// A tile of a side on its way from memory to LDS, eight columns to a chunk:
// Rows x Columns from (row, column) on, zero outside the side.
template <typename T, int Rows, int Columns, bool Whole>
struct Staged {
  static constexpr int count = Rows * Columns / kChunk / kThreads;
  static constexpr int across = Columns / kChunk;
  vec<T, 8> v[count];

  __device__ __forceinline__ void load(const Side<T>& s, int64_t row, int64_t column,
                                       int64_t end) {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int id = i * kThreads + threadIdx.x;
      const int64_t r = row + id / across, c = column + (id % across) * kChunk;
      const T* p = s.data + r * s.stride + c;
      v[i] = T(0);
      if (r < end) {
        if constexpr (Whole) {
          if (c < s.columns) v[i] = *reinterpret_cast<const vec<T, 8>*>(p);
        } else {
#pragma unroll
          for (int j = 0; j < kChunk; ++j)
            if (c + j < s.columns) v[i][j] = p[j];
        }
      }
    }
  }

  __device__ __forceinline__ void load(const KeptSide& s, int64_t row, int64_t column,
                                       int64_t end) {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int id = i * kThreads + threadIdx.x;
      const int64_t r = row + id / across, c = column + (id % across) * kChunk;
      v[i] = T(0);
      if (r < end && c < s.groups * kGroup) {
        float f[kChunk];
        read8(*reinterpret_cast<const uint2*>(s.values + r * s.groups * kGroup + c),
              s.exponents[r * s.groups + c / kGroup], f);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[i][j] = T(f[j]);
      }
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

// Columns [n, n + 16) of a row of C.
template <typename T, bool Whole>
__device__ __forceinline__ void store_row(T* p, int64_t left, const float (&c)[16]) {
  if (Whole && left >= 16) {
#pragma unroll
    for (int h = 0; h < 16; h += 8) {
      vec<T, 8> raw;
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = T(c[h + j]);
      *reinterpret_cast<vec<T, 8>*>(p + h) = raw;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) p[j] = T(c[j]);
  }
}

struct Product {
  int64_t m, n;        // C's rows and columns
  int64_t k;           // length of the sum
  int64_t split;       // k of one workgroup (a multiple of the depth)
  int64_t tiles_n;
};

// out: C in T (split == k), or partial float32 C's, one per split, each
// followed by the M side's sums over k where sums is set.
template <typename T, bool MContiguous, bool NContiguous, typename NSide, bool WholeM,
          bool WholeN, bool WholeC>
__global__ __launch_bounds__(kThreads) void product_kernel(Side<T> ms, NSide ns, Product p,
                                                           const T* __restrict__ bias,
                                                           T* __restrict__ out,
                                                           float* __restrict__ partial) {
  constexpr int depth = Mma<T>::depth;
  __shared__ __align__(16) T m_lds[kTileSize<T, MContiguous>];
  __shared__ __align__(16) T n_lds[kTileSize<T, NContiguous>];
  Staged<T, MContiguous ? kEdge : depth, MContiguous ? depth : kEdge, WholeM> m_next;
  Staged<T, NContiguous ? kEdge : depth, NContiguous ? depth : kEdge, WholeN> n_next;
  const int64_t tile_m = blockIdx.x / p.tiles_n, tile_n = blockIdx.x % p.tiles_n;
  const int64_t m0 = tile_m * kEdge, n0 = tile_n * kEdge;
  const int64_t k0 = int64_t(blockIdx.y) * p.split;
  const int64_t k1 = k0 + p.split < p.k ? k0 + p.split : p.k;
  const int wave = threadIdx.x >> 6;
  const int wave_m = (wave >> 1) * kWaveEdge, wave_n = (wave & 1) * kWaveEdge;
  f32x4 c[kTiles][kTiles];  // [m][n]
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) c[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr bool sums = !MContiguous;
  float sum[kChunk] = {};

  auto fetch = [&](int64_t k) {
    if constexpr (MContiguous)
      m_next.load(ms, m0, k, p.m);
    else
      m_next.load(ms, k, m0, k1);
    if constexpr (NContiguous)
      n_next.load(ns, n0, k, p.n);
    else
      n_next.load(ns, k, n0, k1);
  };
  fetch(k0);
  for (int64_t k = k0; k < k1; k += depth) {
    m_next.template store<kPitch<T, MContiguous>, false, MContiguous>(m_lds);
    n_next.template store<kPitch<T, NContiguous>, true, NContiguous>(n_lds);
    if constexpr (sums) {
      // A thread's chunks of dy lie in the same eight columns throughout.
      if (tile_n == 0) {
#pragma unroll
        for (int i = 0; i < m_next.count; ++i)
#pragma unroll
          for (int j = 0; j < kChunk; ++j) sum[j] += float(m_next.v[i][j]);
      }
    }
    __syncthreads();
    if (k + depth < k1) fetch(k + depth);
#pragma unroll
    for (int s = 0; s < depth; s += Mma<T>::step) {
      typename Mma<T>::Fragment a[kTiles], b[kTiles];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        a[i] = fragment<T, MContiguous>(m_lds, wave_m + 16 * i, s);
        b[i] = fragment<T, NContiguous>(n_lds, wave_n + 16 * i, s);
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; ++j) c[i][j] = Mma<T>::of(b[j], a[i], c[i][j]);
    }
    __syncthreads();
  }

  // Lane 16 q + i holds, of fragment row i, the 16 columns from 16 q on.
  const int lane = threadIdx.x & 63;
  const int64_t n = n0 + wave_n + 16 * (lane >> 4);
  float offset[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) offset[j] = bias && n + j < p.n ? float(bias[n + j]) : 0.f;
  float* mine = partial ? partial + int64_t(blockIdx.y) * (p.m * p.n + (sums ? p.m : 0))
                        : nullptr;
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int64_t m = m0 + wave_m + 16 * i + (lane & 15);
    if (m >= p.m) continue;
    float row[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) row[j] = c[i][j >> 2][j & 3] + offset[j];
    if (mine)
      store_row<float, false>(mine + m * p.n + n, p.n - n, row);
    else
      store_row<T, WholeC>(out + m * p.n + n, p.n - n, row);
  }
  if constexpr (sums) {
    if (tile_n == 0) {
      // 16 threads a row of the staged tile; the 16 rows' sums meet in LDS.
      float* all = reinterpret_cast<float*>(m_lds);
      static_assert(sizeof(m_lds) >= 16 * kEdge * sizeof(float), "sums do not fit");
      constexpr int across = kEdge / kChunk;
      const int r = threadIdx.x / across, column = threadIdx.x % across * kChunk;
#pragma unroll
      for (int j = 0; j < kChunk; ++j) all[r * kEdge + column + j] = sum[j];
      __syncthreads();
      const int64_t m = m0 + threadIdx.x;
      if (threadIdx.x < kEdge && m < p.m) {
        float total = 0.f;
        for (int i = 0; i < kThreads / across; ++i) total += all[i * kEdge + threadIdx.x];
        mine[p.m * p.n + m] = total;
      }
    }
  }
}

// Adds `count` partial results of `size` values; the first `weights` of them
// are dW, the others db.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(const float* __restrict__ partial,
                                                        int count, int64_t size, int64_t weights,
                                                        T* __restrict__ dw, T* __restrict__ db) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= size) return;
  float sum = 0.f;
#pragma unroll 8
  for (int s = 0; s < count; ++s) sum += partial[s * size + i];
  if (i < weights) {
    if (dw) dw[i] = T(sum);
  } else if (db) {
    db[i - weights] = T(sum);
  }
}

// Splits of dW's sum over the rows: two workgroups per compute unit, and at
// least 256 rows to each.
int64_t rows_of_split(int64_t rows, int64_t features, int64_t outputs) {
  const int64_t tiles = ceil_div(features, kEdge) * ceil_div(outputs, kEdge);
  const int64_t most = std::max<int64_t>(1, 512 / tiles);
  const int64_t each = std::max<int64_t>(ceil_div(rows, most), 256);
  return ceil_div(each, 64) * 64;
}

template <typename F>
int with_flags(bool a, bool b, bool c, F&& call) {
  using std::bool_constant;
  auto third = [&](auto x, auto y) {
    c ? call(x, y, bool_constant<true>{}) : call(x, y, bool_constant<false>{});
  };
  auto second = [&](auto x) {
    b ? third(x, bool_constant<true>{}) : third(x, bool_constant<false>{});
  };
  a ? second(bool_constant<true>{}) : second(bool_constant<false>{});
  return GS_OK;
}

int check_linear(const char* name, int32_t dtype, int64_t rows, int64_t features,
                 int64_t outputs) {
  GS_CHECK(check_rows(name, dtype, rows, features, features));
  GS_CHECK(check_rows(name, dtype, rows, outputs, outputs));
  GS_REQUIRE(outputs <= kMostFeatures / 64 && features <= kMostFeatures / 64, GS_ERR_ARGUMENT,
             "%s: at most %lld features and outputs", name, (long long)(kMostFeatures / 64));
  GS_REQUIRE(ceil_div(rows, kEdge) * ceil_div(std::max(features, outputs), kEdge) <=
                 0x7fffffffLL, GS_ERR_OVERFLOW, "%s: too many rows", name);
  return GS_OK;
}

}  // namespace
}  // namespace gs

extern "C" {

int gs_linear_forward(int32_t dtype, const void* x, int64_t row_stride, const void* weight,
                      const void* bias, int64_t rows, int64_t features, int64_t outputs, void* y,
                      void* values, void* exponents, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_linear("gs_linear_forward", dtype, rows, features, outputs));
  GS_CHECK(check_rows("gs_linear_forward", dtype, rows, features, row_stride));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && weight && y && !values == !exponents, GS_ERR_ARGUMENT,
             "null pointer passed to gs_linear_forward");
  if (values)
    GS_CHECK(gs_checkpoint8_write(dtype, x, row_stride, rows, features, values, exponents,
                                  stream));
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const Side<T> ms{static_cast<const T*>(x), row_stride, rows, features};
    const Side<T> ns{static_cast<const T*>(weight), features, outputs, features};
    const Product p{rows, outputs, features, ceil_div(features, 64) * 64,
                    ceil_div(outputs, kEdge)};
    const dim3 grid{unsigned(ceil_div(rows, kEdge) * p.tiles_n)};
    const bool whole = whole_rows<T>(x, features, row_stride) &&
                       whole_rows<T>(weight, features, features);
    with_flags(whole, whole_rows<T>(y, outputs, outputs), false, [&](auto w, auto wc, auto) {
      product_kernel<T, true, true, Side<T>, w.value, w.value, wc.value>
          <<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
              ms, ns, p, static_cast<const T*>(bias), static_cast<T*>(y), nullptr);
    });
    GS_LAUNCHED("linear forward");
    return GS_OK;
  });
}

int gs_linear_backward_input(int32_t dtype, const void* grad_y, int64_t grad_stride,
                             const void* weight, int64_t rows, int64_t features, int64_t outputs,
                             void* grad_x, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_linear("gs_linear_backward_input", dtype, rows, features, outputs));
  GS_CHECK(check_rows("gs_linear_backward_input", dtype, rows, outputs, grad_stride));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(grad_y && weight && grad_x, GS_ERR_ARGUMENT,
             "null pointer passed to gs_linear_backward_input");
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const Side<T> ms{static_cast<const T*>(grad_y), grad_stride, rows, outputs};
    const Side<T> ns{static_cast<const T*>(weight), features, outputs, features};
    const Product p{rows, features, outputs, ceil_div(outputs, 64) * 64,
                    ceil_div(features, kEdge)};
    const dim3 grid{unsigned(ceil_div(rows, kEdge) * p.tiles_n)};
    with_flags(whole_rows<T>(grad_y, outputs, grad_stride),
               whole_rows<T>(weight, features, features),
               whole_rows<T>(grad_x, features, features), [&](auto wm, auto wn, auto wc) {
      product_kernel<T, true, false, Side<T>, wm.value, wn.value, wc.value>
          <<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
              ms, ns, p, static_cast<const T*>(nullptr), static_cast<T*>(grad_x), nullptr);
    });
    GS_LAUNCHED("linear backward input");
    return GS_OK;
  });
}

size_t gs_linear_backward_weight_workspace_size(int32_t, int64_t rows, int64_t features,
                                                int64_t outputs) {
  using namespace gs;
  if (rows <= 0 || features <= 0 || outputs <= 0) return 0;
  return size_t(ceil_div(rows, rows_of_split(rows, features, outputs))) *
         size_t(outputs * (features + 1)) * sizeof(float);
}

int gs_linear_backward_weight(int32_t dtype, const void* grad_y, int64_t grad_stride,
                              const void* values, const void* exponents, int64_t rows,
                              int64_t features, int64_t outputs, void* grad_weight,
                              void* grad_bias, void* workspace, size_t workspace_bytes,
                              void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_linear("gs_linear_backward_weight", dtype, rows, features, outputs));
  GS_CHECK(check_rows("gs_linear_backward_weight", dtype, rows, outputs, grad_stride));
  if (!grad_weight && !grad_bias) return GS_OK;
  GS_REQUIRE(rows == 0 || (grad_y && values && exponents), GS_ERR_ARGUMENT,
             "null pointer passed to gs_linear_backward_weight");
  const size_t need =
      gs_linear_backward_weight_workspace_size(dtype, rows, features, outputs);
  GS_REQUIRE(rows == 0 || (workspace && workspace_bytes >= need), GS_ERR_WORKSPACE,
             "workspace too small for gs_linear_backward_weight");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    int64_t splits = 0;
    if (rows > 0) {
      const int64_t split = rows_of_split(rows, features, outputs);
      splits = ceil_div(rows, split);
      const Side<T> ms{static_cast<const T*>(grad_y), grad_stride, rows, outputs};
      const KeptSide ns{static_cast<const uint8_t*>(values),
                        static_cast<const uint8_t*>(exponents), kept_groups(features), rows,
                        features};
      const Product p{outputs, features, rows, split, ceil_div(features, kEdge)};
      const dim3 grid{unsigned(ceil_div(outputs, kEdge) * p.tiles_n), unsigned(splits)};
      with_flags(whole_rows<T>(grad_y, outputs, grad_stride), true, false,
                 [&](auto wm, auto, auto) {
        product_kernel<T, false, false, KeptSide, wm.value, true, false>
            <<<grid, kThreads, 0, s>>>(ms, ns, p, static_cast<const T*>(nullptr),
                                       static_cast<T*>(nullptr),
                                       static_cast<float*>(workspace));
      });
      GS_LAUNCHED("linear backward weight");
    }
    const int64_t weights = outputs * features, size = weights + outputs;
    join_kernel<T><<<dim3{unsigned(ceil_div(size, kThreads))}, kThreads, 0, s>>>(
        static_cast<const float*>(workspace), int(splits), size, weights,
        static_cast<T*>(grad_weight), static_cast<T*>(grad_bias));
    GS_LAUNCHED("join_kernel");
    return GS_OK;
  });
}

}  // extern "C"
