// Layer norm over the last dimension, forward and backward.
//
//   mu = mean x, r = (mean (x - mu)^2 + eps)^-1/2, h = (x - mu) r
//   y  = h w + b
//   dx = r (a - mean a - h mean(a h)), a = dy w
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// A row is held in the registers of the lanes that share it (eight features
// to a lane, 1 to 64 lanes or several waves to a row), so x is read once:
// the mean first, then the squares of the differences from it, which keeps
// the variance exact where the mean is large. Sums are float32.
//
// The 8-bit form keeps d = x - c in kept8.hpp's format, c = min / 2 + max / 2
// of the row: an offset that all features share costs no bits, and d depends
// on no sum's order. The statistics kept with it are (mu - c, r), those of x
// itself (mu, r), so that h is (v - s0) s1 of what was kept either way.
//
// The weight's and bias's gradients: a lane keeps its features' sums over
// the rows that its wave takes; a workgroup adds its waves' sums in LDS and
// writes one partial row, and a second kernel adds the partial rows in their
// order. No atomics: the result does not depend on timing.
#include "kept8.hpp"
#include "layers_api.hpp"

namespace gs {
namespace {

// Lanes of a row: `lanes` (a power of two up to 64) in one wave, or Waves
// whole waves. Sums, smallest and largest over them.
struct Add {
  static __device__ float of(float a, float b) { return a + b; }
};
struct Low {
  static __device__ float of(float a, float b) { return fminf(a, b); }
};
struct High {
  static __device__ float of(float a, float b) { return fmaxf(a, b); }
};

template <int Ctrl>
__device__ __forceinline__ float swap(float v) {
  return __uint_as_float(dpp<Ctrl>(__float_as_uint(v)));
}

template <typename Op>
__device__ __forceinline__ float across(float v, int lanes) {
  if (lanes >= 2) v = Op::of(v, swap<0xB1>(v));    // quad_perm [1,0,3,2]
  if (lanes >= 4) v = Op::of(v, swap<0x4E>(v));    // quad_perm [2,3,0,1]
  if (lanes >= 8) v = Op::of(v, swap<0x141>(v));   // row_half_mirror
  if (lanes >= 16) v = Op::of(v, swap<0x140>(v));  // row_mirror
  if (lanes >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                    false, false);
    v = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (lanes >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                    false, false);
    v = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// Two values at once over the row's lanes, through LDS where the row has
// several waves (`turn` alternates the buffer, so one barrier is enough).
template <typename First, typename Second, int Waves>
__device__ __forceinline__ void across2(float& a, float& b, int lanes, int& turn) {
  a = across<First>(a, lanes);
  b = across<Second>(b, lanes);
  if constexpr (Waves > 1) {
    __shared__ float2 part[2][Waves];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[turn][wave] = make_float2(a, b);
    __syncthreads();
    float2 all = part[turn][0];
#pragma unroll
    for (int i = 1; i < Waves; ++i) {
      all.x = First::of(all.x, part[turn][i].x);
      all.y = Second::of(all.y, part[turn][i].y);
    }
    a = all.x;
    b = all.y;
    turn ^= 1;
  }
}

// A workgroup of Block threads. Waves == 1: each wave takes 64 / lanes rows
// at a time. Waves > 1: the workgroup takes one row.
template <int Waves>
constexpr int kThreads = Waves == 1 ? 256 : Waves * 64;

// The features of chunk i of this lane, and how many of them the row has.
template <int Waves>
__device__ __forceinline__ int column_of(int i, int lane, int lanes) {
  return (i * (Waves == 1 ? lanes : Waves * 64) + lane) * kChunk;
}

__device__ __forceinline__ int valid_of(int column, int features) {
  const int left = features - column;
  return left < 0 ? 0 : left < kChunk ? left : kChunk;
}

template <typename T, typename W, int Chunks, int Waves>
__global__ __launch_bounds__(kThreads<Waves>) void layer_norm_forward_kernel(
    const T* __restrict__ x, int64_t stride, const W* __restrict__ weight,
    const W* __restrict__ bias, float eps, int64_t rows, int features, int lanes,
    T* __restrict__ y, float2* __restrict__ statistics, uint8_t* __restrict__ values,
    uint8_t* __restrict__ exponents) {
  const int lane = Waves == 1 ? threadIdx.x % lanes : threadIdx.x;
  const int per_block = Waves == 1 ? kThreads<1> / lanes : 1;
  const int slot = Waves == 1 ? threadIdx.x / lanes : 0;
  const int groups = (features + kGroup - 1) / kGroup;
  const float inverse_count = 1.f / float(features);
  float w[Chunks][kChunk], b[Chunks][kChunk];
  int valid[Chunks];
#pragma unroll
  for (int i = 0; i < Chunks; ++i) {
    const int column = column_of<Waves>(i, lane, lanes);
    valid[i] = valid_of(column, features);
    load8<W>(weight + column, weight ? valid[i] : 0, w[i]);
    load8<W>(bias + column, bias ? valid[i] : 0, b[i]);
    if (!weight) {
#pragma unroll
      for (int j = 0; j < kChunk; ++j) w[i][j] = 1.f;
    }
  }
  int turn = 0;
  // The next rows are on their way while these are worked on.
  vec<T, kChunk> raw[Chunks];
  auto send = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < Chunks; ++i)
      raw[i] = load_valid<T, kChunk>(x + row * stride + column_of<Waves>(i, lane, lanes),
                                     row < rows ? valid[i] : 0);
  };
  send(int64_t(blockIdx.x) * per_block + slot);
  // The trip count is the workgroup's: waves of a row meet at barriers.
  for (int64_t first = int64_t(blockIdx.x) * per_block; first < rows;
       first += int64_t(gridDim.x) * per_block) {
    const int64_t row = first + slot;
    const bool live = row < rows;
    float v[Chunks][kChunk];
    float sum = 0.f, low = __builtin_inff(), high = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < Chunks; ++i) widen<T, kChunk>(raw[i], v[i]);
    send(row + int64_t(gridDim.x) * per_block);
#pragma unroll
    for (int i = 0; i < Chunks; ++i)
#pragma unroll
      for (int j = 0; j < kChunk; ++j) sum += v[i][j];
    float unused = 0.f;
    across2<Add, Add, Waves>(sum, unused, lanes, turn);
    // sum / features, rounded once: the product with the reciprocal and one
    // correction (a constant row's mean is then its value).
    float mean = sum * inverse_count;
    mean = __builtin_fmaf(__builtin_fmaf(-mean, float(features), sum), inverse_count, mean);
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < Chunks; ++i)
      if (valid[i] == kChunk) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          const float d = v[i][j] - mean;
          squares = __builtin_fmaf(d, d, squares);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          const float d = j < valid[i] ? v[i][j] - mean : 0.f;
          squares = __builtin_fmaf(d, d, squares);
        }
      }
    across2<Add, Add, Waves>(squares, unused, lanes, turn);
    const float inverse = rsqrtf(__builtin_fmaf(squares, inverse_count, eps));
    float centre = 0.f;
    if (values) {
#pragma unroll
      for (int i = 0; i < Chunks; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          low = Low::of(low, j < valid[i] ? v[i][j] : low);
          high = High::of(high, j < valid[i] ? v[i][j] : high);
        }
      across2<Low, High, Waves>(low, high, lanes, turn);
      centre = 0.5f * low + 0.5f * high;
    }
    if (statistics && live && lane == 0) statistics[row] = make_float2(mean - centre, inverse);
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      const int column = column_of<Waves>(i, lane, lanes);
      float out[kChunk];
#pragma unroll
      for (int j = 0; j < kChunk; ++j)
        out[j] = __builtin_fmaf((v[i][j] - mean) * inverse, w[i][j], b[i][j]);
      store8<T>(y + row * features + column, live ? valid[i] : 0, out);
      if (values) {
        // The last group's lanes past the row keep zeros. (A NaN that fmaxf
        // passes over has made the row's statistics NaN.)
        float largest = 0.f;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          v[i][j] = j < valid[i] ? v[i][j] - centre : 0.f;
          largest = fmaxf(largest, fabsf(v[i][j]));
        }
        uint32_t exponent;
        const uint2 bytes = keep8<float>(v[i], __float_as_uint(largest), exponent);
        if (live && column < groups * kGroup) {
          *reinterpret_cast<uint2*>(values + row * (int64_t(groups) * kGroup) + column) = bytes;
          if (column % kGroup == 0) exponents[row * groups + column / kGroup] = uint8_t(exponent);
        }
      }
    }
  }
}

// Partial sums: [gridDim.x][2][features] float32, dw then db.
template <typename T, typename W, int Chunks, int Waves, bool Kept>
__global__ __launch_bounds__(kThreads<Waves>) void layer_norm_backward_kernel(
    const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
    const uint8_t* __restrict__ values, const uint8_t* __restrict__ exponents,
    const float2* __restrict__ statistics, const W* __restrict__ weight, int64_t rows,
    int features, int lanes, T* __restrict__ dx, float* __restrict__ partial) {
  extern __shared__ float shared[];
  const int lane = Waves == 1 ? threadIdx.x % lanes : threadIdx.x;
  const int per_block = Waves == 1 ? kThreads<1> / lanes : 1;
  const int slot = Waves == 1 ? threadIdx.x / lanes : 0;
  const int groups = (features + kGroup - 1) / kGroup;
  const float inverse_count = 1.f / float(features);
  float w[Chunks][kChunk], dw[Chunks][kChunk], db[Chunks][kChunk];
  int valid[Chunks];
#pragma unroll
  for (int i = 0; i < Chunks; ++i) {
    const int column = column_of<Waves>(i, lane, lanes);
    valid[i] = valid_of(column, features);
    load8<W>(weight + column, weight ? valid[i] : 0, w[i]);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      if (!weight) w[i][j] = 1.f;
      dw[i][j] = db[i][j] = 0.f;
    }
  }
  int turn = 0;
  // The next rows are on their way while these are worked on.
  float2 s_next;
  vec<T, kChunk> g_next[Chunks], x_next[Chunks];
  uint2 kept_next[Chunks];
  uint32_t exponent_next[Chunks];
  auto send = [&](int64_t row) {
    const bool live = row < rows;
    s_next = live ? statistics[row] : make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      const int column = column_of<Waves>(i, lane, lanes);
      g_next[i] = load_valid<T, kChunk>(dy + row * dy_stride + column, live ? valid[i] : 0);
      if (Kept) {
        kept_next[i] = make_uint2(0, 0);
        exponent_next[i] = 0;
        if (live && valid[i] > 0) {
          kept_next[i] = *reinterpret_cast<const uint2*>(
              values + row * (int64_t(groups) * kGroup) + column);
          exponent_next[i] = exponents[row * groups + column / kGroup];
        }
      } else {
        x_next[i] = load_valid<T, kChunk>(x + row * x_stride + column, live ? valid[i] : 0);
      }
    }
  };
  send(int64_t(blockIdx.x) * per_block + slot);
  for (int64_t first = int64_t(blockIdx.x) * per_block; first < rows;
       first += int64_t(gridDim.x) * per_block) {
    const int64_t row = first + slot;
    const bool live = row < rows;
    const float2 s = s_next;
    float g[Chunks][kChunk], h[Chunks][kChunk];
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      widen<T, kChunk>(g_next[i], g[i]);
      if (Kept)
        read8(kept_next[i], exponent_next[i], h[i]);
      else
        widen<T, kChunk>(x_next[i], h[i]);
    }
    send(row + int64_t(gridDim.x) * per_block);
    float sum = 0.f, product = 0.f;
#pragma unroll
    for (int i = 0; i < Chunks; ++i)
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        h[i][j] = (h[i][j] - s.x) * s.y;
        const float a = g[i][j] * w[i][j];
        sum += a;
        product = __builtin_fmaf(a, h[i][j], product);
        dw[i][j] = __builtin_fmaf(g[i][j], h[i][j], dw[i][j]);
        db[i][j] += g[i][j];
      }
    across2<Add, Add, Waves>(sum, product, lanes, turn);
    sum *= inverse_count;
    product *= inverse_count;
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      float out[kChunk];
#pragma unroll
      for (int j = 0; j < kChunk; ++j)
        out[j] = s.y * (__builtin_fmaf(g[i][j], w[i][j], -sum) - h[i][j] * product);
      store8<T>(dx + row * features + column_of<Waves>(i, lane, lanes),
                       live ? valid[i] : 0, out);
    }
  }
  if (!partial) return;
  float* mine = partial + int64_t(blockIdx.x) * 2 * features;
  if constexpr (Waves > 1) {
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      const int column = column_of<Waves>(i, lane, lanes);
#pragma unroll
      for (int j = 0; j < kChunk; ++j)
        if (j < valid[i]) {
          mine[column + j] = dw[i][j];
          mine[features + column + j] = db[i][j];
        }
    }
  } else {
    // The workgroup's slots each hold sums of every feature: slots add theirs
    // to LDS one after the other's barrier, in their order. Slots of one wave
    // are added across its lanes first.
    for (int step = lanes; step < 64; step *= 2) {
#pragma unroll
      for (int i = 0; i < Chunks; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          dw[i][j] += __shfl_xor(dw[i][j], step);
          db[i][j] += __shfl_xor(db[i][j], step);
        }
    }
    const int wave = threadIdx.x >> 6;
    const bool holds = (threadIdx.x & 63) < lanes;
    for (int turn_of = 0; turn_of < kThreads<1> / 64; ++turn_of) {
      if (wave == turn_of && holds) {
#pragma unroll
        for (int i = 0; i < Chunks; ++i) {
          const int column = column_of<Waves>(i, lane, lanes);
#pragma unroll
          for (int j = 0; j < kChunk; ++j)
            if (j < valid[i]) {
              float* at = shared + column + j;
              const float before_w = turn_of ? at[0] : 0.f;
              const float before_b = turn_of ? at[features] : 0.f;
              at[0] = before_w + dw[i][j];
              at[features] = before_b + db[i][j];
            }
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * features; i += kThreads<1>) mine[i] = shared[i];
  }
}

// Adds the partial rows: 16 columns and 16 slices of the rows to a
// workgroup; slices are added in LDS in their order.
constexpr int kColumns = 16, kSlices = 16;

template <typename W>
__global__ __launch_bounds__(kColumns* kSlices) void layer_norm_parameters_kernel(
    const float* __restrict__ partial, int count, int features, W* __restrict__ dweight,
    W* __restrict__ dbias) {
  __shared__ float sums[kSlices][kColumns];
  const int column = blockIdx.x * kColumns + threadIdx.x % kColumns;
  const int slice = threadIdx.x / kColumns;
  float sum = 0.f;
  if (column < 2 * features) {
#pragma unroll 8
    for (int i = slice; i < count; i += kSlices)
      sum += partial[int64_t(i) * 2 * features + column];
  }
  sums[slice][threadIdx.x % kColumns] = sum;
  __syncthreads();
  if (slice || column >= 2 * features) return;
  for (int i = 1; i < kSlices; ++i) sum += sums[i][threadIdx.x];
  if (column < features) {
    if (dweight) dweight[column] = W(sum);
  } else if (dbias) {
    dbias[column - features] = W(sum);
  }
}

// Rows wider than this are refused.
constexpr int64_t kMostNormFeatures = 16384;

int lanes_of(int64_t features) {
  int lanes = 1;
  while (lanes < 64 && lanes * kChunk < features) lanes *= 2;
  return lanes < 4 ? 4 : lanes;  // a group of the checkpoint takes four
}

// Workgroups: enough rows at a time to fill the chip, each taking several
// after one another, so that parameters are loaded and partial sums written
// once for all of them.
int64_t blocks_of(int64_t rows, int64_t features, bool backward) {
  const int64_t per_block = features <= 2048 ? 256 / lanes_of(features) : 1;
  const int64_t most = backward ? 1024 : 2048;
  return std::min(ceil_div(rows, per_block), most);
}

template <typename F>
void with_shape(int64_t features, F&& launch) {
  using std::integral_constant;
  using one = integral_constant<int, 1>;
  using two = integral_constant<int, 2>;
  using four = integral_constant<int, 4>;
  if (features <= 512)
    launch(one{}, one{});
  else if (features <= 1024)
    launch(two{}, one{});
  else if (features <= 2048)
    launch(four{}, one{});
  else if (features <= 8192)
    launch(four{}, four{});
  else
    launch(two{}, integral_constant<int, 16>{});
}

template <typename F>
int with_types(int32_t dtype, int32_t weight_dtype, F&& call) {
  return with_type(dtype, [&](auto zero) {
    return weight_dtype == GS_FLOAT32 ? call(zero, float(0)) : call(zero, zero);
  });
}

int check_norm(const char* name, int32_t dtype, int32_t weight_dtype, int64_t rows,
               int64_t features, int64_t stride) {
  GS_CHECK(check_rows(name, dtype, rows, features, stride));
  GS_REQUIRE(weight_dtype == dtype || weight_dtype == GS_FLOAT32, GS_ERR_ARGUMENT,
             "%s: parameters must have the rows' type or float32", name);
  GS_REQUIRE(features <= kMostNormFeatures, GS_ERR_ARGUMENT,
             "%s: at most %lld features", name, (long long)kMostNormFeatures);
  return GS_OK;
}

}  // namespace
}  // namespace gs

extern "C" {

int gs_layer_norm_forward(int32_t dtype, int32_t weight_dtype, const void* x, int64_t row_stride,
                          const void* weight, const void* bias, float eps, int64_t rows,
                          int64_t features, void* y, void* statistics, void* values,
                          void* exponents, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_norm("gs_layer_norm_forward", dtype, weight_dtype, rows, features, row_stride));
  GS_REQUIRE(std::isfinite(eps) && eps >= 0.f, GS_ERR_ARGUMENT,
             "eps must be finite and not negative");
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && y && !values == !exponents && (!values || statistics), GS_ERR_ARGUMENT,
             "null pointer passed to gs_layer_norm_forward");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_types(dtype, weight_dtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    const dim3 grid{unsigned(blocks_of(rows, features, false))};
    with_shape(features, [&](auto chunks, auto waves) {
      layer_norm_forward_kernel<T, W, chunks.value, waves.value>
          <<<grid, kThreads<waves.value>, 0, s>>>(
              static_cast<const T*>(x), row_stride, static_cast<const W*>(weight),
              static_cast<const W*>(bias), eps, rows, int(features), lanes_of(features),
              static_cast<T*>(y), static_cast<float2*>(statistics),
              static_cast<uint8_t*>(values), static_cast<uint8_t*>(exponents));
    });
    GS_LAUNCHED("layer_norm_forward_kernel");
    return GS_OK;
  });
}

size_t gs_layer_norm_backward_workspace_size(int64_t rows, int64_t features) {
  if (rows <= 0 || features <= 0) return 0;
  return size_t(gs::blocks_of(rows, features, true)) * 2 * size_t(features) * sizeof(float);
}

int gs_layer_norm_backward(int32_t dtype, int32_t weight_dtype, const void* grad_y,
                           int64_t grad_stride, const void* x, int64_t row_stride,
                           const void* values, const void* exponents, const void* statistics,
                           const void* weight, int64_t rows, int64_t features, void* grad_x,
                           void* grad_weight, void* grad_bias, void* workspace,
                           size_t workspace_bytes, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_norm("gs_layer_norm_backward", dtype, weight_dtype, rows, features,
                      grad_stride));
  GS_REQUIRE(values || rows <= 1 || row_stride >= features, GS_ERR_ARGUMENT,
             "gs_layer_norm_backward: rows overlap");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool parameters = grad_weight || grad_bias;
  if (rows > 0) {
    GS_REQUIRE(grad_y && !x != !values && !values == !exponents && statistics && grad_x,
               GS_ERR_ARGUMENT, "null pointer passed to gs_layer_norm_backward");
    GS_REQUIRE(!parameters || (workspace && workspace_bytes >=
                                                gs_layer_norm_backward_workspace_size(
                                                    rows, features)),
               GS_ERR_WORKSPACE, "workspace too small for gs_layer_norm_backward");
  }
  return with_types(dtype, weight_dtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    const int64_t blocks = rows > 0 ? blocks_of(rows, features, true) : 0;
    if (rows > 0) {
      with_shape(features, [&](auto chunks, auto waves) {
        const size_t shared = waves.value == 1 ? 2 * size_t(features) * sizeof(float) : 0;
        auto launch = [&](auto kept) {
          layer_norm_backward_kernel<T, W, chunks.value, waves.value, kept.value>
              <<<dim3{unsigned(blocks)}, kThreads<waves.value>, shared, s>>>(
                  static_cast<const T*>(grad_y), grad_stride, static_cast<const T*>(x),
                  row_stride, static_cast<const uint8_t*>(values),
                  static_cast<const uint8_t*>(exponents), static_cast<const float2*>(statistics),
                  static_cast<const W*>(weight), rows, int(features), lanes_of(features),
                  static_cast<T*>(grad_x),
                  parameters ? static_cast<float*>(workspace) : nullptr);
        };
        values ? launch(std::true_type{}) : launch(std::false_type{});
      });
      GS_LAUNCHED("layer_norm_backward_kernel");
    }
    if (parameters) {
      layer_norm_parameters_kernel<W>
          <<<dim3{unsigned(ceil_div(2 * features, kColumns))}, kColumns * kSlices, 0, s>>>(
              static_cast<const float*>(workspace), int(blocks), int(features),
              static_cast<W*>(grad_weight), static_cast<W*>(grad_bias));
      GS_LAUNCHED("layer_norm_parameters_kernel");
    }
    return GS_OK;
  });
}

}  // extern "C"
