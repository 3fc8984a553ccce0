// 8-bit checkpoints written and read, and activations that keep their input
// in that form (see kept8.hpp for the format).
//
//   activation: y = f(z);  dz = dy f'(z8), z8 the kept z
//     sine  f = sin(omega z)      f' = omega cos(omega z)
//     gelu  f = z Phi(z)          f' = Phi(z) + z phi(z)
//     silu  f = z s, s = 1 / (1 + exp(-z))   f' = s (1 + z (1 - s))
//
// Each kernel reads and writes each byte once, and memory bounds it: a lane
// takes eight features (16 bytes of a 2-byte type), so four lanes hold a group
// and its largest magnitude takes two quad permutations, no LDS; a thread has
// four such chunks on their way. 1M x 512 bfloat16: written in 285 us (5.4
// TB/s), read back in 253 (6.1), gelu forward in 458 (5.6) and backward in 487
// (5.3; the vector units issue for 90% and 80% of the time, 25 and 24
// instructions a value, most of them Phi's); sine 447 and 461, silu 434 and
// 464. 500k x 512 float32: gelu and sine 422 and 435 (6.1 and 5.9 TB/s).
#include "kept8.hpp"
#include "layers_api.hpp"

namespace gs {
namespace {

constexpr int kBlock = 256;

// Where a lane's chunk lies. Flat: rows follow each other without padding
// and hold whole groups, so that the chunk's number is its place. Otherwise
// the block's first chunk is divided into row and chunk once, in 64 bits and
// for all lanes alike, and the lanes divide what remains in 32 bits.
struct Rows {
  int64_t rows, features, stride;
  uint32_t per_row;  // chunks of a row, padding included
};

struct Place {
  int64_t row;
  uint32_t chunk;
};

__device__ __forceinline__ Place place(const Rows& r, int64_t first, uint32_t local) {
  const int64_t row0 = first / r.per_row;
  const uint32_t rest = uint32_t(first - row0 * r.per_row) + local;
  const uint32_t down = rest / r.per_row;
  return {row0 + down, rest - down * r.per_row};
}

enum Kind { kSine = GS_ACTIVATION_SINE, kGelu = GS_ACTIVATION_GELU, kSilu = GS_ACTIVATION_SILU };

// Whether a type shows errors of 2^-24: float32's functions are evaluated to
// its own rounding, which costs no time beside four bytes a value (gelu of
// 500k x 512: 425 and 420 us, 423 and 426 with the shorter form). The 2-byte
// types' rounding is 2^13 and 2^16 times as large, and the longer forms take
// time there: gelu of 1M x 512 bfloat16 569 and 574 us against 461 and 450,
// the sine's slope 513 against 456.
template <typename T>
constexpr bool kFine = sizeof(T) == 4;

// The fraction f of z (high + low) revolutions, high + low = omega / 2 pi, for
// sin and cos of 2 pi f: the product's fraction is taken with fused
// multiply-adds, so the phase has no rounding error of its size. From 2^24
// revolutions on the rounded product is a whole number further than 1/2 from
// the product, so what is left is brought to |f| <= 1/2 once more (f is off by
// 2^-48 of the revolutions at most; a product past float32's range gives NaN).
__device__ __forceinline__ float turn(float z, float high, float low) {
  const float k = rintf(z * high);
  const float f = __builtin_fmaf(z, low, __builtin_fmaf(z, high, -k));
  return f - rintf(f);
}

// sin r, |r| <= pi/2: the Taylor polynomial of sin to the 13th degree, whose
// first omitted term is below 7e-10.
__device__ __forceinline__ float sine_of_angle(float r) {
  const float s = r * r;
  float p = 1.6059043836821613e-10f;
  p = __builtin_fmaf(p, s, -2.5052108385441720e-8f);
  p = __builtin_fmaf(p, s, 2.7557319223985893e-6f);
  p = __builtin_fmaf(p, s, -1.9841269841269841e-4f);
  p = __builtin_fmaf(p, s, 8.3333333333333333e-3f);
  p = __builtin_fmaf(p, s, -1.6666666666666667e-1f);
  return __builtin_fmaf(p * s, r, r);
}

// sin(2 pi f), |f| <= 1/4.
__device__ __forceinline__ float sine_of_quarter(float f) {
  return sine_of_angle(f * 6.283185307179586f);
}

// sin(2 pi f), |f| <= 1/2: reflected at 1/4.
__device__ __forceinline__ float sine_of_turn(float f) {
  const float a = fabsf(f);
  return sine_of_quarter(copysignf(fminf(a, 0.5f - a), f));
}

// float32's fraction in two parts, whose sum it is to 2^-48 of the
// revolutions: the product less the nearest whole number is exact, and so is
// its rounding error (of the rounded product: contracted, it would count
// twice). What passes 1/2 (from 2^24 revolutions on) comes off the second part.
struct Turn {
  float high, low;
};

__device__ __forceinline__ Turn fine_turn(float z, float high, float low) {
#pragma clang fp contract(off)
  const float p = z * high;
  const float rest = __builtin_fmaf(z, low, __builtin_fmaf(z, high, -p));
  return {p - rintf(p), rest - rintf(rest)};
}

// sin(2 pi (high + low)), the sum within 1/4: 2 pi too has two parts, so that
// the angle is rounded once.
__device__ __forceinline__ float sine_of_parts(float high, float low) {
  constexpr float two_pi = 6.283185307179586f;
  constexpr float rest = float(6.283185307179586 - double(two_pi));
  return sine_of_angle(
      __builtin_fmaf(high, two_pi, __builtin_fmaf(high, rest, low * two_pi)));
}

// sin(2 pi f) from the nearest half revolution n / 2 on, with n's sign.
__device__ __forceinline__ float fine_sine(Turn f) {
  constexpr float magic = 12582912.f;  // 1.5 2^23: the sum's low bit is n's
  const float n = __builtin_fmaf(2.f, f.high + f.low, magic);
  const float r = sine_of_parts(__builtin_fmaf(n - magic, -0.5f, f.high), f.low);
  return __uint_as_float(__float_as_uint(r) ^ (__float_as_uint(n) << 31));
}

// cos(2 pi f) = sin(2 pi (1/4 - |f|)), |f| = high + low once both have the
// sign that makes it so, and 1/4 - high with its rounding error.
__device__ __forceinline__ float fine_cosine(Turn f) {
  float high = f.high - rintf(f.high + f.low), low = f.low;
  const bool negative = high + low < 0.f;
  high = negative ? -high : high;
  low = negative ? -low : low;
  const float rest = 0.25f - high;
  return sine_of_parts(rest, ((0.25f - rest) - high) - low);
}

struct Parameters {
  float omega, high, low;
};

// The 2-byte types' Phi(z) and exp(-z^2/2): Phi(-|z|) = t P(t) exp(-z^2/2),
// t = 1 / (1 + 0.3 |z|), P of degree 5 fitted for |z| up to 13.5 to 2.5e-7 of
// Phi and, so that the tail keeps its digits, 1.2e-5 of Phi(-|z|), 1/40 of
// float16's half a unit.
__device__ __forceinline__ void normal_cdf(float z, float& cdf, float& bell) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, fabsf(z), 1.f));
  bell = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  float p = -0.07940997333659087f;
  p = __builtin_fmaf(p, t, 0.2223334973660695f);
  p = __builtin_fmaf(p, t, -0.023300158444618253f);
  p = __builtin_fmaf(p, t, 0.14712824046081913f);
  p = __builtin_fmaf(p, t, 0.11312709265706829f);
  p = __builtin_fmaf(p, t, 0.12012105298966325f);
  const float tail = p * t * bell;
  cdf = z < 0.f ? tail : 1.f - tail;
}

// float32's Phi(z) and exp(-z^2/2), each to a few units of 2^-24 of itself,
// tails included; the sum that torch rounds, 1 + erf, has no such tail.
//
// The bell as 2^(h + l), h + l = -z^2 log2(e) / 2 with the rounding errors of
// the square and of the product in l. |z| is cut at 15, where the bell is 0.
// Phi: |z| < 5/4: 1/2 + z Q(z^2), Q of degree 5; beyond: Phi(-|z|) = t P(t)
// bell, t = 1 / (1 + |z| / 4), P of degree 7 for |z| up to 13.5. Both fitted
// for the least relative error: 8.5e-9 of Q and 7.8e-9 of t P.
struct Normal {
  float bell, centre, cdf;  // cdf: outside of the centre, Phi = 1/2 + z centre
  bool inside;
};

__device__ __forceinline__ Normal normal(float z) {
  Normal n;
  const float x = fminf(fabsf(z), 15.f);
  const float s = x * x;
  constexpr float rate = -0.72134752044448170f;  // -log2(e) / 2 = rate + rest
  constexpr float rest = float(-0.72134752044448170 - double(rate));
  const float h = s * rate;
  float l = __builtin_fmaf(s, rest, __builtin_fmaf(s, rate, -h));
  l = __builtin_fmaf(__builtin_fmaf(x, x, -s), rate, l);
  const float bell = __builtin_amdgcn_exp2f(h);
  n.bell = __builtin_fmaf(bell, l * 0.69314718055994531f, bell);
  float q = -6.831350674474379e-06f;
  q = __builtin_fmaf(q, s, 0.00011112703941762447f);
  q = __builtin_fmaf(q, s, -0.0011839555809274316f);
  q = __builtin_fmaf(q, s, 0.009972349740564823f);
  q = __builtin_fmaf(q, s, -0.06649021804332733f);
  n.centre = __builtin_fmaf(q, s, 0.3989422917366028f);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.25f, x, 1.f));
  float p = -0.04807112365961075f;
  p = __builtin_fmaf(p, t, 0.11373986303806305f);
  p = __builtin_fmaf(p, t, -0.02872179076075554f);
  p = __builtin_fmaf(p, t, 0.09712773561477661f);
  p = __builtin_fmaf(p, t, 0.07140213251113892f);
  p = __builtin_fmaf(p, t, 0.0951610654592514f);
  p = __builtin_fmaf(p, t, 0.09957888722419739f);
  p = __builtin_fmaf(p, t, 0.09974174946546555f);
  const float tail = p * t * n.bell;
  n.cdf = z < 0.f ? tail : 1.f - tail;
  n.inside = x < 1.25f;
  return n;
}

// 1 / (1 + exp(-z)). float32: the exponent as h + l, l the rounding errors of
// -z log2(e), z cut where the result is 0 or 1.
template <typename T>
__device__ __forceinline__ float sigmoid(float z, float& denominator) {
  constexpr float rate = -1.4426950408889634f;
  float e;
  if constexpr (kFine<T>) {
    constexpr float rest = float(-1.4426950408889634 - double(rate));
    const float x = __builtin_amdgcn_fmed3f(z, -130.f, 130.f);
    const float h = x * rate;
    const float l = __builtin_fmaf(x, rest, __builtin_fmaf(x, rate, -h));
    const float whole = __builtin_amdgcn_exp2f(h);
    e = __builtin_fmaf(whole, l * 0.69314718055994531f, whole);
  } else {
    e = __builtin_amdgcn_exp2f(z * rate);
  }
  denominator = 1.f + e;
  return __builtin_amdgcn_rcpf(denominator);
}

template <typename T, int K>
__device__ __forceinline__ float value(float z, const Parameters& c) {
  if constexpr (K == kSine && kFine<T>) {
    return fine_sine(fine_turn(z, c.high, c.low));
  } else if constexpr (K == kSine) {
    return sine_of_turn(turn(z, c.high, c.low));
  } else if constexpr (K == kGelu && kFine<T>) {
    const Normal n = normal(z);
    return z * (n.inside ? __builtin_fmaf(z, n.centre, 0.5f) : n.cdf);
  } else if constexpr (K == kGelu) {
    float cdf, bell;
    normal_cdf(z, cdf, bell);
    return z * cdf;
  } else {
    float d;
    const float s = sigmoid<T>(z, d), y = z * s;
    if constexpr (!kFine<T>) return y;
    // The quotient z / d to its rounding, where d is no infinity.
    return fabsf(z) < 88.f ? __builtin_fmaf(__builtin_fmaf(-d, y, z), s, y) : y;
  }
}

template <typename T, int K>
__device__ __forceinline__ float slope(float z, const Parameters& c) {
  if constexpr (K == kSine && kFine<T>) {
    return c.omega * fine_cosine(fine_turn(z, c.high, c.low));
  } else if constexpr (K == kSine) {
    const float f = turn(z, c.high, c.low);
    // cos(2 pi f) = sin(2 pi (1/4 - |f|))
    return c.omega * sine_of_quarter(0.25f - fabsf(f));
  } else if constexpr (K == kGelu && kFine<T>) {
    const Normal n = normal(z);
    constexpr float unit = 0.39894228040143268f;  // phi(0)
    return n.inside ? __builtin_fmaf(z, __builtin_fmaf(n.bell, unit, n.centre), 0.5f)
                    : __builtin_fmaf(z * n.bell, unit, n.cdf);
  } else if constexpr (K == kGelu) {
    float cdf, bell;
    normal_cdf(z, cdf, bell);
    return __builtin_fmaf(z * bell, 0.39894228040143268f, cdf);
  } else {
    float d;
    const float s = sigmoid<T>(z, d);
    return s * __builtin_fmaf(z, 1.f - s, 1.f);
  }
}

constexpr int kNone = -1;

// Writes the checkpoint of x (where values is not null) and, with an
// activation, y.
template <typename T, int K, bool Flat, bool Narrow, int Each>
__global__ __launch_bounds__(kBlock) void keep_kernel(const T* __restrict__ x, Rows r,
                                                      T* __restrict__ y,
                                                      uint8_t* __restrict__ values,
                                                      uint8_t* __restrict__ exponents,
                                                      Parameters c) {
  const int64_t total = r.rows * r.per_row;
  const int64_t first = int64_t(blockIdx.x) * (kBlock * Each);
  vec<T, kChunk> raw[Each];
  Place at[Each];
  int valid[Each];
#pragma unroll
  for (int i = 0; i < Each; ++i) {
    const uint32_t local = i * kBlock + threadIdx.x;
    const bool live = first + local < total;
    if constexpr (Flat) {
      valid[i] = live ? kChunk : 0;
      raw[i] = load_valid<T, kChunk>(x + (first + local) * kChunk, valid[i]);
    } else {
      at[i] = place(r, first, local);
      const int64_t left = r.features - int64_t(at[i].chunk) * kChunk;
      valid[i] = live ? int(left < 0 ? 0 : left < kChunk ? left : kChunk) : 0;
      raw[i] = load_edge<T, kChunk, Narrow>(
          x + at[i].row * r.stride + int64_t(at[i].chunk) * kChunk, valid[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < Each; ++i) {
    const uint32_t local = i * kBlock + threadIdx.x;
    if (first + local >= total) break;
    const int64_t chunk = first + local;  // rows of the checkpoint follow each other
    if constexpr (!Flat) raw[i] = settle<T, kChunk, Narrow>(raw[i], valid[i]);
    float v[kChunk];
    widen<T, kChunk>(raw[i], v);
    if (values) {
      uint32_t exponent;
      const uint2 bytes = keep8<T>(v, largest_of<T, kChunk>(raw[i]), exponent);
      *reinterpret_cast<uint2*>(values + chunk * kChunk) = bytes;
      if ((threadIdx.x & 3) == 0) exponents[chunk >> 2] = uint8_t(exponent);
    }
    if constexpr (K != kNone) {
      float f[kChunk];
#pragma unroll
      for (int j = 0; j < kChunk; ++j) f[j] = value<T, K>(v[j], c);
      if constexpr (Flat)
        store8<T>(y + chunk * kChunk, kChunk, f);
      else
        store8<T>(y + at[i].row * r.features + int64_t(at[i].chunk) * kChunk, valid[i],
                         f);
    }
  }
}

// Reads a checkpoint back, or applies an activation's derivative at it to dy.
template <typename T, int K, bool Flat, bool Narrow, int Each>
__global__ __launch_bounds__(kBlock) void read_kernel(const uint8_t* __restrict__ values,
                                                      const uint8_t* __restrict__ exponents,
                                                      const T* __restrict__ dy, Rows r,
                                                      T* __restrict__ out, Parameters c) {
  const int64_t total = r.rows * r.per_row;
  const int64_t first = int64_t(blockIdx.x) * (kBlock * Each);
  vec<T, kChunk> g[Each];
  uint2 bytes[Each];
  uint32_t exponent[Each];
  Place at[Each];
  int valid[Each];
#pragma unroll
  for (int i = 0; i < Each; ++i) {
    const uint32_t local = i * kBlock + threadIdx.x;
    const int64_t chunk = first + local;
    const bool live = chunk < total;
    bytes[i] = make_uint2(0, 0);
    exponent[i] = 0;
    if (live) {
      bytes[i] = *reinterpret_cast<const uint2*>(values + chunk * kChunk);
      exponent[i] = exponents[chunk >> 2];
    }
    if constexpr (Flat) {
      valid[i] = live ? kChunk : 0;
      if constexpr (K != kNone) g[i] = load_valid<T, kChunk>(dy + chunk * kChunk, valid[i]);
    } else {
      at[i] = place(r, first, local);
      const int64_t left = r.features - int64_t(at[i].chunk) * kChunk;
      valid[i] = live ? int(left < 0 ? 0 : left < kChunk ? left : kChunk) : 0;
      if constexpr (K != kNone)
        g[i] = load_edge<T, kChunk, Narrow>(
            dy + at[i].row * r.stride + int64_t(at[i].chunk) * kChunk, valid[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < Each; ++i) {
    if (valid[i] <= 0) continue;
    float v[kChunk];
    read8(bytes[i], exponent[i], v);
    if constexpr (K != kNone) {
      if constexpr (!Flat) g[i] = settle<T, kChunk, Narrow>(g[i], valid[i]);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) v[j] = float(g[i][j]) * slope<T, K>(v[j], c);
    }
    if constexpr (Flat)
      store8<T>(out + (first + i * kBlock + threadIdx.x) * kChunk, kChunk, v);
    else
      store8<T>(out + at[i].row * r.features + int64_t(at[i].chunk) * kChunk, valid[i],
                       v);
  }
}

// Chunks from which a thread takes four of them: one a thread for 1,024
// workgroups. Below that, one each fills more of the chip.
constexpr int64_t kFour = int64_t(4) * 256 * kBlock;

// Chunks of a launch at most: a launch takes less than 2^32 threads, here a
// quarter of them, and more rows take several launches.
constexpr int64_t kMostChunks = int64_t(4) << 30;

// Calls `part(first row, rows)` for each launch's rows.
template <typename F>
int in_parts(int64_t rows, int64_t features, F&& part) {
  const int64_t most = kMostChunks / (kept_groups(features) * (kGroup / kChunk));
  for (int64_t first = 0; first < rows; first += most)
    GS_CHECK(part(first, std::min(rows - first, most)));
  return GS_OK;
}

template <typename F>
int with_layout(const char* name, const Rows& r, bool flat, F&& launch) {
  const int64_t total = r.rows * r.per_row;
  const bool four = total >= kFour;
  const int64_t blocks = ceil_div(total, four ? 4 * kBlock : kBlock);
  using std::bool_constant;
  using one = std::integral_constant<int, 1>;
  using all = std::integral_constant<int, 4>;
  const dim3 grid{unsigned(blocks)};
  auto by_count = [&](auto flat_, auto narrow) {
    four ? launch(grid, flat_, narrow, all{}) : launch(grid, flat_, narrow, one{});
  };
  if (flat)
    by_count(bool_constant<true>{}, bool_constant<false>{});
  else if (r.features >= kChunk)
    by_count(bool_constant<false>{}, bool_constant<false>{});
  else
    by_count(bool_constant<false>{}, bool_constant<true>{});
  GS_LAUNCHED(name);
  return GS_OK;
}

template <typename F>
int with_kind(int32_t kind, F&& call) {
  switch (kind) {
    case kSine: return call(std::integral_constant<int, kSine>{});
    case kGelu: return call(std::integral_constant<int, kGelu>{});
    default: return call(std::integral_constant<int, kSilu>{});
  }
}

Parameters parameters(float omega) {
  const double turns = double(omega) / 6.283185307179586476925;
  const float high = float(turns);
  return {omega, high, float(turns - double(high))};
}

Rows rows_of(int64_t rows, int64_t features, int64_t stride) {
  return {rows, features, stride, uint32_t(kept_groups(features) * (kGroup / kChunk))};
}

template <typename T, int K>
int keep_rows(const char* name, const void* x, int64_t rows, int64_t features, int64_t stride,
              void* y, void* values, void* exponents, float omega, hipStream_t s) {
  const bool flat = (stride == features || rows == 1) && features % kGroup == 0;
  return in_parts(rows, features, [&](int64_t first, int64_t count) {
    const Rows r = rows_of(count, features, stride);
    const int64_t groups = kept_groups(features);
    const T* const from = static_cast<const T*>(x) + first * stride;
    T* const to = y ? static_cast<T*>(y) + first * features : nullptr;
    uint8_t* const v = values ? static_cast<uint8_t*>(values) + first * groups * kGroup : nullptr;
    uint8_t* const e = exponents ? static_cast<uint8_t*>(exponents) + first * groups : nullptr;
    return with_layout(name, r, flat, [&](dim3 grid, auto f, auto narrow, auto each) {
      keep_kernel<T, K, f.value, narrow.value, each.value><<<grid, kBlock, 0, s>>>(
          from, r, to, v, e, parameters(omega));
    });
  });
}

template <typename T, int K>
int read_rows(const char* name, const void* values, const void* exponents, const void* dy,
              int64_t rows, int64_t features, int64_t stride, void* out, float omega,
              hipStream_t s) {
  const bool flat = features % kGroup == 0 && (K == kNone || stride == features || rows == 1);
  return in_parts(rows, features, [&](int64_t first, int64_t count) {
    const Rows r = rows_of(count, features, stride);
    const int64_t groups = kept_groups(features);
    const uint8_t* const v = static_cast<const uint8_t*>(values) + first * groups * kGroup;
    const uint8_t* const e = static_cast<const uint8_t*>(exponents) + first * groups;
    const T* const g = dy ? static_cast<const T*>(dy) + first * stride : nullptr;
    T* const to = static_cast<T*>(out) + first * features;
    return with_layout(name, r, flat, [&](dim3 grid, auto f, auto narrow, auto each) {
      read_kernel<T, K, f.value, narrow.value, each.value><<<grid, kBlock, 0, s>>>(
          v, e, g, r, to, parameters(omega));
    });
  });
}

int check_activation(int32_t kind, float omega) {
  GS_REQUIRE(kind == kSine || kind == kGelu || kind == kSilu, GS_ERR_ARGUMENT,
             "unknown activation %d", int(kind));
  GS_REQUIRE(std::isfinite(omega), GS_ERR_ARGUMENT, "omega must be finite");
  return GS_OK;
}

}  // namespace
}  // namespace gs

extern "C" {

int gs_checkpoint8_write(int32_t dtype, const void* x, int64_t row_stride, int64_t rows,
                         int64_t features, void* values, void* exponents, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_rows("gs_checkpoint8_write", dtype, rows, features, row_stride));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && values && exponents, GS_ERR_ARGUMENT,
             "null pointer passed to gs_checkpoint8_write");
  return with_type(dtype, [&](auto zero) {
    return keep_rows<decltype(zero), kNone>("checkpoint8 write", x, rows, features, row_stride,
                                            nullptr, values, exponents, 0.f,
                                            static_cast<hipStream_t>(stream));
  });
}

int gs_checkpoint8_read(int32_t dtype, const void* values, const void* exponents, int64_t rows,
                        int64_t features, void* out, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_rows("gs_checkpoint8_read", dtype, rows, features, features));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(values && exponents && out, GS_ERR_ARGUMENT,
             "null pointer passed to gs_checkpoint8_read");
  return with_type(dtype, [&](auto zero) {
    return read_rows<decltype(zero), kNone>("checkpoint8 read", values, exponents, nullptr, rows,
                                            features, features, out, 0.f,
                                            static_cast<hipStream_t>(stream));
  });
}

int gs_activation_forward(int32_t dtype, int32_t kind, float omega, const void* x,
                          int64_t row_stride, int64_t rows, int64_t features, void* y,
                          void* values, void* exponents, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_rows("gs_activation_forward", dtype, rows, features, row_stride));
  GS_CHECK(check_activation(kind, omega));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && y && !values == !exponents, GS_ERR_ARGUMENT,
             "null pointer passed to gs_activation_forward");
  return with_type(dtype, [&](auto zero) {
    return with_kind(kind, [&](auto k) {
      return keep_rows<decltype(zero), k.value>("activation forward", x, rows, features,
                                                row_stride, y, values, exponents, omega,
                                                static_cast<hipStream_t>(stream));
    });
  });
}

int gs_activation_backward(int32_t dtype, int32_t kind, float omega, const void* grad_y,
                           int64_t grad_stride, const void* values, const void* exponents,
                           int64_t rows, int64_t features, void* grad_x, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_rows("gs_activation_backward", dtype, rows, features, grad_stride));
  GS_CHECK(check_activation(kind, omega));
  if (rows == 0) return GS_OK;
  GS_REQUIRE(grad_y && values && exponents && grad_x, GS_ERR_ARGUMENT,
             "null pointer passed to gs_activation_backward");
  return with_type(dtype, [&](auto zero) {
    return with_kind(kind, [&](auto k) {
      return read_rows<decltype(zero), k.value>("activation backward", values, exponents, grad_y,
                                                rows, features, grad_stride, grad_x, omega,
                                                static_cast<hipStream_t>(stream));
    });
  });
}

}  // extern "C"
