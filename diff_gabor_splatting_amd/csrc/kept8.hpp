// 8-bit checkpoints: the form in which a row of activations is kept between
// the forward and the backward pass, and the loads and stores of the three
// float types that the layer kernels share.
//
// A row's features are cut into groups of 32 (the last may be shorter). A
// group keeps one exponent byte b and a signed byte q per feature, which
// stand for q 2^(b-127): b is the smallest with which the group's largest
// magnitude rounds to at most 127, within [least, most]. A power of two and
// not largest / 127: v 2^-e is exact, so q is a function of the inputs alone
// (no rounding of a scale comes before it), and q 2^e is exact in the type that
// the values came from (in bfloat16 and float32 whatever they came from, in
// float16 within its range), so the matrix instructions of the linear layer's
// weight gradient take it without another rounding. It costs at most one of
// the eight bits. A group that holds an infinity or a NaN keeps b = 255 and
// reads back as NaN throughout.
//
// A row of F features takes 32 ceil(F / 32) value bytes (the rest of the
// last group is zero) and ceil(F / 32) exponent bytes, so rows of values are
// 32-byte aligned whatever F is.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace gs {

constexpr int kGroup = 32;   // features per exponent
constexpr int kChunk = 8;    // features per lane: four lanes hold a group

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// Exponent limits by the type the values came from. float16's values are
// multiples of 2^-24, and 127 * 2^9 is its largest q 2^e; elsewhere 2^-126
// and 127 * 2^121 keep the scale and every q 2^e within float32's normal
// range.
template <typename T>
struct KeptRange {
  static constexpr int least = 1, most = 248;
};
template <>
struct KeptRange<f16> {
  static constexpr int least = 127 - 24, most = 127 + 9;
};

template <int Ctrl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), Ctrl, 0xf, 0xf, true));
}

// A vector in memory at any element's address: the global loads and stores
// of gfx950 take 16 bytes from any of them, so rows of odd widths are read as
// wide as others.
template <typename T, int N>
struct Packed {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <typename T, int N>
__device__ __forceinline__ vec<T, N> load_packed(const T* p) {
  return *reinterpret_cast<const typename Packed<T, N>::type*>(p);
}

template <typename T, int N>
__device__ __forceinline__ void store_packed(T* p, vec<T, N> v) {
  *reinterpret_cast<typename Packed<T, N>::type*>(p) = v;
}

// The first `valid` < N values at p, zero after them: 4, 2 and 1 at a time.
template <typename T, int N>
__device__ __forceinline__ vec<T, N> load_part(const T* p, int valid) {
  vec<T, N> v = T(0);
  int at = 0;
  if (N > 4 && (valid & 4)) {
    const vec<T, 4> four = load_packed<T, 4>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = four[j];
    at = 4;
  }
  if (valid & 2) {
    const vec<T, 2> two = load_packed<T, 2>(p + at);
    if (N > 4 && at) {
      v[N > 4 ? 4 : 0] = two[0];
      v[N > 4 ? 5 : 1] = two[1];
    } else {
      v[0] = two[0];
      v[1] = two[1];
    }
    at += 2;
  }
  if (valid & 1) {
    const T one = p[at];
#pragma unroll
    for (int j = 0; j < N; j += 2)
      if (at == j) v[j] = one;
  }
  return v;
}

// N consecutive values, `valid` of them in the row (none below 1).
template <typename T, int N>
__device__ __forceinline__ vec<T, N> load_valid(const T* p, int valid) {
  if (valid >= N) return load_packed<T, N>(p);
  if (valid > 0) return load_part<T, N>(p, valid);
  return vec<T, N>(T(0));
}

// The same without waiting for memory: the last, partly filled piece of a
// row is loaded N - valid values earlier, where it is whole and inside the
// row, and `settle` moves it down once it is there. (load_part puts its pieces
// together at once, so a load ahead of its use would not be one.) Rows of
// fewer than N values (Narrow) have no such place and take load_valid.
template <typename T, int N, bool Narrow>
__device__ __forceinline__ vec<T, N> load_edge(const T* p, int valid) {
  if constexpr (Narrow) {
    return load_valid<T, N>(p, valid);
  } else {
    vec<T, N> v = T(0);
    if (valid > 0) v = load_packed<T, N>(p - (N - valid));
    return v;
  }
}

template <typename T, int N, bool Narrow>
__device__ __forceinline__ vec<T, N> settle(vec<T, N> v, int valid) {
  if constexpr (Narrow) {
    return v;
  } else {
    if (valid >= N) return v;
    constexpr int words = N * sizeof(T) / 4;
    vec<uint32_t, words> w = __builtin_bit_cast(vec<uint32_t, words>, v);
    // Down by `words_down` words, 4, 2 and 1 at a time, then by half a word.
    const int missing = N - valid, words_down = missing * int(sizeof(T)) / 4;
#pragma unroll
    for (int step = 4; step; step >>= 1) {
      if (step >= words) continue;
      const bool move = words_down & step;
#pragma unroll
      for (int j = 0; j < words; ++j) {
        const uint32_t from = j + step < words ? w[j + step < words ? j + step : 0] : 0u;
        w[j] = move ? from : w[j];
      }
    }
    if constexpr (sizeof(T) == 2) {
      const bool move = missing & 1;
#pragma unroll
      for (int j = 0; j < words; ++j) {
        const uint32_t next = j + 1 < words ? w[j + 1 < words ? j + 1 : 0] : 0u;
        w[j] = move ? __builtin_amdgcn_alignbit(next, w[j], 16) : w[j];
      }
    }
    return __builtin_bit_cast(vec<T, N>, w);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_valid(T* p, int valid, vec<T, N> v) {
  if (valid >= N) {
    store_packed<T, N>(p, v);
  } else if (valid > 0) {
    int at = 0;
    if (N > 4 && (valid & 4)) {
      store_packed<T, 4>(p, vec<T, 4>{v[0], v[1], v[2], v[3]});
      at = 4;
    }
    if (valid & 2) {
      store_packed<T, 2>(p + at, N > 4 && at ? vec<T, 2>{v[N > 4 ? 4 : 0], v[N > 4 ? 5 : 1]}
                                             : vec<T, 2>{v[0], v[1]});
      at += 2;
    }
    if (valid & 1) {
      T one = v[0];
#pragma unroll
      for (int j = 2; j < N; j += 2)
        if (at == j) one = v[j];
      p[at] = one;
    }
  }
}

template <typename T, int N>
__device__ __forceinline__ void widen(vec<T, N> raw, float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = float(raw[j]);
}

// Eight consecutive features as float32, zero past `valid`.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[kChunk]) {
  const vec<T, 8> raw = load_valid<T, 8>(p, valid);
#pragma unroll
  for (int j = 0; j < kChunk; ++j) v[j] = float(raw[j]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int valid, const float (&v)[kChunk]) {
  vec<T, 8> raw;
#pragma unroll
  for (int j = 0; j < kChunk; ++j) raw[j] = T(v[j]);
  store_valid<T, 8>(p, valid, raw);
}

// Exponent byte of a group from its largest magnitude's bits. Adding 2^16
// carries into the exponent from a mantissa of 127.5 / 64 on, which would
// round to 128. As unsigned integers NaN > infinity > every finite value.
template <typename T>
__device__ __forceinline__ uint32_t kept_exponent(uint32_t largest) {
  const int b = int((largest + 0x10000u) >> 23) - 6;
  const int within = min(max(b, KeptRange<T>::least), KeptRange<T>::most);
  return largest >= 0x7f800000u ? 255u : uint32_t(within);
}

// The largest magnitude of N values, as float32 bits. The 2-byte types'
// magnitudes compare as 16-bit integers, two at a time.
template <typename T, int N>
__device__ __forceinline__ uint32_t largest_of(vec<T, N> v) {
  if constexpr (sizeof(T) == 4) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
    return most;
  } else {
    typedef vec<uint16_t, 2> pair;
    vec<uint32_t, N / 2> words = __builtin_bit_cast(vec<uint32_t, N / 2>, v);
    pair most = {0, 0};
#pragma unroll
    for (int j = 0; j < N / 2; ++j)
      most = __builtin_elementwise_max(most,
                                       __builtin_bit_cast(pair, words[j] & 0x7fff7fffu));
    const uint16_t one = most[0] > most[1] ? most[0] : most[1];
    if constexpr (std::is_same_v<T, bf16>)
      return uint32_t(one) << 16;
    else
      return __float_as_uint(float(__builtin_bit_cast(f16, one)));
  }
}

// N values over a group's power of two, as bytes, four to a word.
template <typename T, int N>
__device__ __forceinline__ void keep_bytes(const float (&v)[N], uint32_t exponent,
                                           uint32_t (&out)[N / 4]) {
  const float inverse = exponent == 255 ? 0.f : __uint_as_float((254u - exponent) << 23);
  // v 2^-e + 1.5 2^23 rounds v 2^-e to an integer (ties to even) whose low
  // byte is q. Only at the largest exponent of a type can q pass 127.
  constexpr float magic = 12582912.f;
  uint32_t bits[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    bits[j] = __float_as_uint(__builtin_fmaf(v[j], inverse, magic));
  if (__builtin_expect(__ballot(exponent == KeptRange<T>::most) != 0, 0)) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      bits[j] = __float_as_uint(
          __builtin_amdgcn_fmed3f(__uint_as_float(bits[j]), magic - 127.f, magic + 127.f));
  }
  const uint32_t fine = exponent == 255 ? 0u : ~0u;
#pragma unroll
  for (int j = 0; j < N; j += 4)
    out[j / 4] = fine & __builtin_amdgcn_perm(
                            __builtin_amdgcn_perm(bits[j + 3], bits[j + 2], 0x0c0c0400u),
                            __builtin_amdgcn_perm(bits[j + 1], bits[j], 0x0c0c0400u),
                            0x05040100u);
}

// The eight values of this lane, as bytes; the quad of lanes that holds the
// group calls it together. `largest`: their largest magnitude's bits. T: the
// type that sets the exponent's range.
template <typename T>
__device__ __forceinline__ uint2 keep8(const float (&v)[kChunk], uint32_t largest,
                                       uint32_t& exponent) {
  largest = max(largest, dpp<0xB1>(largest));  // quad_perm [1,0,3,2]
  largest = max(largest, dpp<0x4E>(largest));  // quad_perm [2,3,0,1]
  exponent = kept_exponent<T>(largest);
  uint32_t bytes[2];
  keep_bytes<T, kChunk>(v, exponent, bytes);
  return make_uint2(bytes[0], bytes[1]);
}

// q 2^e of four bytes, exact. b = 255 makes the scale infinite, and 0 times
// it NaN (all q of such a group are 0).
__device__ __forceinline__ void read4(uint32_t word, float scale, float* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = float(int(int8_t(word >> (8 * j)))) * scale;
}

__device__ __forceinline__ void read8(uint2 bytes, uint32_t exponent, float (&v)[kChunk]) {
  const float scale = __uint_as_float(exponent << 23);
  read4(bytes.x, scale, v);
  read4(bytes.y, scale, v + 4);
}

inline int64_t kept_groups(int64_t features) { return ceil_div(features, kGroup); }

}  // namespace gs
