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
//
// Memory bounds both passes. 1M x 512 bfloat16: forward 381 us (5.4 TB/s), 533
// with the 8-bit form (4.8; the vector units, with 202 instructions a row and
// wave, then issue for 73% of the time), backward 565 (5.4), 475 from the 8-bit
// form (5.4; 63%). With 1,024 x 64 float32 rows it is launches: 3.5 us, 5.6
// and 2.5 for the partial sums.
#include "kept8.hpp"
#include "layers_api.hpp"

namespace gs {
namespace {

// Lanes of a row: Lanes (a power of two from 4 to 64) of one wave, or Waves
// whole waves. The lower lane bits are crossed with DPP moves, the upper two
// with the lane swaps.
template <int Ctrl>
__device__ __forceinline__ float swap(float v) {
  return __uint_as_float(dpp<Ctrl>(__float_as_uint(v)));
}

template <int Lanes>
__device__ __forceinline__ float sum_across(float v) {
  v += swap<0xB1>(v);                            // quad_perm [1,0,3,2]
  v += swap<0x4E>(v);                            // quad_perm [2,3,0,1]
  if constexpr (Lanes >= 8) v += swap<0x141>(v);   // row_half_mirror
  if constexpr (Lanes >= 16) v += swap<0x140>(v);  // row_mirror
  if constexpr (Lanes >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                    false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (Lanes >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                    false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Smallest and largest. As instructions, since the compiler quiets every
// operand of fminf and fmaxf first (four instructions for one); a NaN is
// passed over. Each s_nop is the distance that a DPP or lane swap keeps from
// the write of what it reads.
__device__ __forceinline__ void range_of_8(const float (&v)[kChunk], float& low, float& high) {
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(low) : "v"(v[0]), "v"(v[1]), "v"(v[2]));
  asm("v_min3_f32 %0, %0, %1, %2" : "+v"(low) : "v"(v[3]), "v"(v[4]));
  asm("v_min3_f32 %0, %0, %1, %2" : "+v"(low) : "v"(v[5]), "v"(v[6]));
  asm("v_min_f32 %0, %0, %1" : "+v"(low) : "v"(v[7]));
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(high) : "v"(v[0]), "v"(v[1]), "v"(v[2]));
  asm("v_max3_f32 %0, %0, %1, %2" : "+v"(high) : "v"(v[3]), "v"(v[4]));
  asm("v_max3_f32 %0, %0, %1, %2" : "+v"(high) : "v"(v[5]), "v"(v[6]));
  asm("v_max_f32 %0, %0, %1" : "+v"(high) : "v"(v[7]));
}

__device__ __forceinline__ void widen_range(float& low, float& high, float other_low,
                                            float other_high) {
  asm("v_min_f32 %0, %0, %1" : "+v"(low) : "v"(other_low));
  asm("v_max_f32 %0, %0, %1" : "+v"(high) : "v"(other_high));
}

#define GS_RANGE_DPP(control)                                                        \
  asm("s_nop 1\n\t"                                                                  \
      "v_min_f32_dpp %0, %0, %0 " control " row_mask:0xf bank_mask:0xf\n\t"           \
      "v_max_f32_dpp %1, %1, %1 " control " row_mask:0xf bank_mask:0xf\n\t"           \
      "s_nop 1"                                                                      \
      : "+v"(low), "+v"(high))

template <int Lanes>
__device__ __forceinline__ void range_across(float& low, float& high) {
  GS_RANGE_DPP("quad_perm:[1,0,3,2]");
  GS_RANGE_DPP("quad_perm:[2,3,0,1]");
  if constexpr (Lanes >= 8) GS_RANGE_DPP("row_half_mirror");
  if constexpr (Lanes >= 16) GS_RANGE_DPP("row_mirror");
  if constexpr (Lanes >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(low), __float_as_uint(low),
                                                    false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(high), __float_as_uint(high),
                                                    false, false);
    low = __uint_as_float(a[0]);
    high = __uint_as_float(b[0]);
    widen_range(low, high, __uint_as_float(a[1]), __uint_as_float(b[1]));
    asm("s_nop 1" : "+v"(low), "+v"(high));
  }
  if constexpr (Lanes >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(low), __float_as_uint(low),
                                                    false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(high), __float_as_uint(high),
                                                    false, false);
    low = __uint_as_float(a[0]);
    high = __uint_as_float(b[0]);
    widen_range(low, high, __uint_as_float(a[1]), __uint_as_float(b[1]));
  }
}
#undef GS_RANGE_DPP

// Two values of every wave of a row's, in LDS. `turn` alternates the buffer,
// so that one barrier is enough.
template <int Waves>
struct Meet {
  float2 part[2][Waves];
};

template <int Lanes, int Waves>
__device__ __forceinline__ void sum2(float& a, float& b, Meet<Waves>& meet, int& turn) {
  a = sum_across<Lanes>(a);
  b = sum_across<Lanes>(b);
  if constexpr (Waves > 1) {
    if ((threadIdx.x & 63) == 0) meet.part[turn][threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    float2 all = meet.part[turn][0];
#pragma unroll
    for (int i = 1; i < Waves; ++i) {
      all.x += meet.part[turn][i].x;
      all.y += meet.part[turn][i].y;
    }
    a = all.x;
    b = all.y;
    turn ^= 1;
  }
}

template <int Lanes, int Waves>
__device__ __forceinline__ float sum1(float a, Meet<Waves>& meet, int& turn) {
  if constexpr (Waves > 1) {
    float unused = 0.f;
    sum2<Lanes, Waves>(a, unused, meet, turn);
    return a;
  } else {
    return sum_across<Lanes>(a);
  }
}

template <int Lanes, int Waves>
__device__ __forceinline__ void range2(float& low, float& high, Meet<Waves>& meet, int& turn) {
  range_across<Lanes>(low, high);
  if constexpr (Waves > 1) {
    if ((threadIdx.x & 63) == 0) meet.part[turn][threadIdx.x >> 6] = make_float2(low, high);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Waves; ++i)
      widen_range(low, high, meet.part[turn][i].x, meet.part[turn][i].y);
    turn ^= 1;
  }
}

// A workgroup of kThreads threads. Waves == 1: each wave takes 64 / Lanes rows
// at a time. Waves > 1: the workgroup takes one row.
template <int Waves>
constexpr int kThreads = Waves == 1 ? 256 : Waves * 64;

// Workgroups to a compute unit. The grid is that many for each of the 256,
// all of them running at once (one more would wait for the rest and then run
// by itself), and no more than memory likes: 1M x 512 bfloat16 rows, forward
// with 3, 4, 5, 6: 398, 380, 367, 412 us; keeping 8 bits: 510, 569, 546, 539
// (both before the mean's correction, which added 2% to the latter);
// backward with 2, 3, 4, 5: 564, 572, 610, 603, from 8 bits 530, 461, 502,
// 517. They are those of this size; fewer or shorter rows may want others. The
// registers of a row set the limit where it takes more lanes' worth.
enum Pass { kForward, kForwardKept, kBackward };
template <int Chunks, int Waves>
constexpr int workgroups_of(Pass pass) {
  if (Waves == 16) return 1;
  if (Chunks == 1) return pass == kForward ? 5 : 3;
  if (Chunks == 2) return pass == kBackward ? 2 : 3;
  return pass == kBackward ? 1 : 2;
}
template <int Waves>
constexpr int kSimdWaves = Waves == 16 ? 4 : 1;  // of a workgroup, on each of the four
constexpr int kUnits = 256;

// The features of chunk i of this lane, and how many of them the row has.
template <int Lanes, int Waves>
__device__ __forceinline__ int column_of(int i, int lane) {
  return (i * Lanes * Waves + lane) * kChunk;
}

__device__ __forceinline__ int valid_of(int column, int features) {
  const int left = features - column;
  return left < 0 ? 0 : left < kChunk ? left : kChunk;
}

template <typename T, typename W, int Chunks, int Waves, int Lanes, bool Narrow>
__global__ __launch_bounds__(
    kThreads<Waves>, (workgroups_of<Chunks, Waves>(kForward) * kSimdWaves<Waves>)) void layer_norm_forward_kernel(
    const T* __restrict__ x, int64_t stride, const W* __restrict__ weight,
    const W* __restrict__ bias, float eps, int64_t rows, int features,
    T* __restrict__ y, float2* __restrict__ statistics, uint8_t* __restrict__ values,
    uint8_t* __restrict__ exponents) {
  static_assert(Waves == 1 || Lanes == 64, "a row of several waves takes whole ones");
  constexpr int per_block = Waves == 1 ? kThreads<1> / Lanes : 1;
  const int lane = Waves == 1 ? threadIdx.x % Lanes : threadIdx.x;
  const int slot = Waves == 1 ? threadIdx.x / Lanes : 0;
  __shared__ Meet<Waves> meet;
  const int groups = (features + kGroup - 1) / kGroup;
  const float inverse_count = 1.f / float(features);
  const bool ragged = features % kChunk;
  float w[Chunks][kChunk], b[Chunks][kChunk];
  int valid[Chunks];
#pragma unroll
  for (int i = 0; i < Chunks; ++i) {
    const int column = column_of<Lanes, Waves>(i, lane);
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
      raw[i] = load_edge<T, kChunk, Narrow>(
          x + row * stride + column_of<Lanes, Waves>(i, lane), row < rows ? valid[i] : 0);
  };
  send(int64_t(blockIdx.x) * per_block + slot);
  // The trip count is the workgroup's: waves of a row meet at barriers.
  for (int64_t first = int64_t(blockIdx.x) * per_block; first < rows;
       first += int64_t(gridDim.x) * per_block) {
    const int64_t row = first + slot;
    const bool live = row < rows;
    float v[Chunks][kChunk];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      if (ragged) raw[i] = settle<T, kChunk, Narrow>(raw[i], valid[i]);
      widen<T, kChunk>(raw[i], v[i]);
    }
    send(row + int64_t(gridDim.x) * per_block);
#pragma unroll
    for (int i = 0; i < Chunks; ++i)
#pragma unroll
      for (int j = 0; j < kChunk; ++j) sum += v[i][j];
    sum = sum1<Lanes, Waves>(sum, meet, turn);
    // sum / features, rounded once: the product with the reciprocal and one
    // correction.
    float mean = sum * inverse_count;
    mean = __builtin_fmaf(__builtin_fmaf(-mean, float(features), sum), inverse_count, mean);
    // The differences from it, zero past the row.
    float d[Chunks][kChunk];
    auto differ = [&] {
#pragma unroll
      for (int i = 0; i < Chunks; ++i) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) d[i][j] = v[i][j] - mean;
        if (valid[i] != kChunk) {
#pragma unroll
          for (int j = 0; j < kChunk; ++j) d[i][j] = j < valid[i] ? d[i][j] : 0.f;
        }
      }
    };
    differ();
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < Chunks; ++i)
#pragma unroll
      for (int j = 0; j < kChunk; ++j) squares = __builtin_fmaf(d[i][j], d[i][j], squares);
    squares = sum1<Lanes, Waves>(squares, meet, turn);
    float inverse = rsqrtf(__builtin_fmaf(squares, inverse_count, eps));
    // The sum has lost units of its own last place. Where the mean is larger
    // than the deviation they show in h: the mean of the differences from it is
    // then added (a constant row's mean becomes its value) and its square taken
    // off the variance. 1M x 512 bfloat16 rows with the 8-bit form: 499 us without
    // the test, 509 with it, 524 where every row goes through. A row's result is
    // its own: rows that share a wave with such a one stay as they are.
    const bool far = mean * mean > squares * inverse_count;
    if (__any(far)) {
      float rest = 0.f;
#pragma unroll
      for (int i = 0; i < Chunks; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) rest += d[i][j];
      rest = sum1<Lanes, Waves>(rest, meet, turn) * inverse_count;
      const float variance = __builtin_fmaf(squares, inverse_count, -rest * rest);
      if (far) {
        mean += rest;
        inverse = rsqrtf((variance < 0.f ? 0.f : variance) + eps);
        differ();
      }
    }
    float centre = 0.f;
    if (values) {
      float low = __builtin_inff(), high = -low;
#pragma unroll
      for (int i = 0; i < Chunks; ++i) {
        float in_low = __builtin_inff(), in_high = -in_low;
        if (valid[i] == kChunk) {
          range_of_8(v[i], in_low, in_high);
        } else if (valid[i] > 0) {
          // The row's last chunk, its first value in place of what it lacks.
          float filled[kChunk];
#pragma unroll
          for (int j = 0; j < kChunk; ++j) filled[j] = j < valid[i] ? v[i][j] : v[i][0];
          range_of_8(filled, in_low, in_high);
        }
        widen_range(low, high, in_low, in_high);
      }
      range2<Lanes, Waves>(low, high, meet, turn);
      centre = 0.5f * low + 0.5f * high;
    }
    if (statistics && live && lane == 0) statistics[row] = make_float2(mean - centre, inverse);
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      const int column = column_of<Lanes, Waves>(i, lane);
      float out[kChunk];
#pragma unroll
      for (int j = 0; j < kChunk; ++j)
        out[j] = __builtin_fmaf(d[i][j] * inverse, w[i][j], b[i][j]);
      store8<T>(y + row * features + column, live ? valid[i] : 0, out);
      if (values) {
        // The last group's lanes past the row keep zeros. (A NaN that fmaxf
        // passes over has made the row's statistics NaN.)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[i][j] -= centre;
        if (valid[i] != kChunk) {
#pragma unroll
          for (int j = 0; j < kChunk; ++j) v[i][j] = j < valid[i] ? v[i][j] : 0.f;
        }
        float largest = 0.f;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) largest = fmaxf(largest, fabsf(v[i][j]));
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
template <typename T, typename W, int Chunks, int Waves, int Lanes, bool Narrow, bool Kept>
__global__ __launch_bounds__(
    kThreads<Waves>,
    (workgroups_of<Chunks, Waves>(kBackward) * kSimdWaves<Waves>)) void layer_norm_backward_kernel(
    const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
    const uint8_t* __restrict__ values, const uint8_t* __restrict__ exponents,
    const float2* __restrict__ statistics, const W* __restrict__ weight, int64_t rows,
    int features, T* __restrict__ dx, float* __restrict__ partial) {
  extern __shared__ float shared[];
  static_assert(Waves == 1 || Lanes == 64, "a row of several waves takes whole ones");
  constexpr int per_block = Waves == 1 ? kThreads<1> / Lanes : 1;
  const int lane = Waves == 1 ? threadIdx.x % Lanes : threadIdx.x;
  const int slot = Waves == 1 ? threadIdx.x / Lanes : 0;
  __shared__ Meet<Waves> meet;
  const int groups = (features + kGroup - 1) / kGroup;
  const float inverse_count = 1.f / float(features);
  const bool ragged = features % kChunk;
  float w[Chunks][kChunk], dw[Chunks][kChunk], db[Chunks][kChunk];
  int valid[Chunks];
#pragma unroll
  for (int i = 0; i < Chunks; ++i) {
    const int column = column_of<Lanes, Waves>(i, lane);
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
      const int column = column_of<Lanes, Waves>(i, lane);
      g_next[i] =
          load_edge<T, kChunk, Narrow>(dy + row * dy_stride + column, live ? valid[i] : 0);
      if (Kept) {
        kept_next[i] = make_uint2(0, 0);
        exponent_next[i] = 0;
        if (live && valid[i] > 0) {
          kept_next[i] = *reinterpret_cast<const uint2*>(
              values + row * (int64_t(groups) * kGroup) + column);
          exponent_next[i] = exponents[row * groups + column / kGroup];
        }
      } else {
        x_next[i] =
            load_edge<T, kChunk, Narrow>(x + row * x_stride + column, live ? valid[i] : 0);
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
      if (ragged) g_next[i] = settle<T, kChunk, Narrow>(g_next[i], valid[i]);
      widen<T, kChunk>(g_next[i], g[i]);
      if (Kept) {
        read8(kept_next[i], exponent_next[i], h[i]);
      } else {
        if (ragged) x_next[i] = settle<T, kChunk, Narrow>(x_next[i], valid[i]);
        widen<T, kChunk>(x_next[i], h[i]);
      }
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
    sum2<Lanes, Waves>(sum, product, meet, turn);
    sum *= inverse_count;
    product *= inverse_count;
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      float out[kChunk];
#pragma unroll
      for (int j = 0; j < kChunk; ++j)
        out[j] = s.y * (__builtin_fmaf(g[i][j], w[i][j], -sum) - h[i][j] * product);
      store8<T>(dx + row * features + column_of<Lanes, Waves>(i, lane),
                       live ? valid[i] : 0, out);
    }
  }
  if (!partial) return;
  float* mine = partial + int64_t(blockIdx.x) * 2 * features;
  if constexpr (Waves > 1) {
#pragma unroll
    for (int i = 0; i < Chunks; ++i) {
      const int column = column_of<Lanes, Waves>(i, lane);
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
    for (int step = Lanes; step < 64; step *= 2) {
#pragma unroll
      for (int i = 0; i < Chunks; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          dw[i][j] += __shfl_xor(dw[i][j], step);
          db[i][j] += __shfl_xor(db[i][j], step);
        }
    }
    const int wave = threadIdx.x >> 6;
    const bool holds = (threadIdx.x & 63) < Lanes;
    for (int turn_of = 0; turn_of < kThreads<1> / 64; ++turn_of) {
      if (wave == turn_of && holds) {
#pragma unroll
        for (int i = 0; i < Chunks; ++i) {
          const int column = column_of<Lanes, Waves>(i, lane);
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

// Chunks of a lane, waves of a row and lanes of a wave for a width, and whether
// it is less than a chunk. A group
// of the checkpoint takes four lanes, so a row takes as many at least.
template <typename F>
void with_shape(int64_t features, F&& launch) {
  using std::integral_constant;
  using one = integral_constant<int, 1>;
  using two = integral_constant<int, 2>;
  using four = integral_constant<int, 4>;
  using all = integral_constant<int, 64>;
  using wide = std::false_type;
  if (features < kChunk)
    launch(one{}, one{}, four{}, std::true_type{});
  else if (features <= 32)
    launch(one{}, one{}, four{}, wide{});
  else if (features <= 64)
    launch(one{}, one{}, integral_constant<int, 8>{}, wide{});
  else if (features <= 128)
    launch(one{}, one{}, integral_constant<int, 16>{}, wide{});
  else if (features <= 256)
    launch(one{}, one{}, integral_constant<int, 32>{}, wide{});
  else if (features <= 512)
    launch(one{}, one{}, all{}, wide{});
  else if (features <= 1024)
    launch(two{}, one{}, all{}, wide{});
  else if (features <= 2048)
    launch(four{}, one{}, all{}, wide{});
  else if (features <= 4096)
    launch(two{}, four{}, all{}, wide{});
  else if (features <= 8192)
    launch(four{}, four{}, all{}, wide{});
  else
    launch(two{}, integral_constant<int, 16>{}, all{}, wide{});
}

// Workgroups: as many as the chip holds, each taking several rows after one
// another, so that parameters are loaded and partial sums written once for
// all of them; fewer where there are not the rows.
int64_t blocks_of(int64_t rows, int64_t features, Pass pass) {
  int64_t blocks = 0;
  with_shape(features, [&](auto chunks, auto waves, auto lanes, auto) {
    const int64_t per_block = waves.value == 1 ? kThreads<1> / lanes.value : 1;
    const int64_t most = kUnits * workgroups_of<chunks.value, waves.value>(pass);
    blocks = std::min(ceil_div(rows, per_block), most);
  });
  return blocks;
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
    const dim3 grid{unsigned(blocks_of(rows, features, values ? kForwardKept : kForward))};
    with_shape(features, [&](auto chunks, auto waves, auto lanes, auto narrow) {
      layer_norm_forward_kernel<T, W, chunks.value, waves.value, lanes.value, narrow.value>
          <<<grid, kThreads<waves.value>, 0, s>>>(
              static_cast<const T*>(x), row_stride, static_cast<const W*>(weight),
              static_cast<const W*>(bias), eps, rows, int(features),
              static_cast<T*>(y), static_cast<float2*>(statistics),
              static_cast<uint8_t*>(values), static_cast<uint8_t*>(exponents));
    });
    GS_LAUNCHED("layer_norm_forward_kernel");
    return GS_OK;
  });
}

size_t gs_layer_norm_backward_workspace_size(int64_t rows, int64_t features) {
  if (rows <= 0 || features <= 0) return 0;
  return size_t(gs::blocks_of(rows, features, gs::kBackward)) * 2 * size_t(features) * sizeof(float);
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
    const int64_t blocks = rows > 0 ? blocks_of(rows, features, kBackward) : 0;
    if (rows > 0) {
      with_shape(features, [&](auto chunks, auto waves, auto lanes, auto narrow) {
        const size_t shared = waves.value == 1 ? 2 * size_t(features) * sizeof(float) : 0;
        auto launch = [&](auto kept) {
          layer_norm_backward_kernel<T, W, chunks.value, waves.value, lanes.value, narrow.value,
                                     kept.value>
              <<<dim3{unsigned(blocks)}, kThreads<waves.value>, shared, s>>>(
                  static_cast<const T*>(grad_y), grad_stride, static_cast<const T*>(x),
                  row_stride, static_cast<const uint8_t*>(values),
                  static_cast<const uint8_t*>(exponents), static_cast<const float2*>(statistics),
                  static_cast<const W*>(weight), rows, int(features),
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
