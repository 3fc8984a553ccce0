// 8-bit checkpoints: the form in which a row of activations is kept between
// the forward and the backward pass, and the loads and stores of the three
// float types that the layer kernels share.
//
// A row's features are cut into groups of 32 (the last may be shorter). A
// group keeps one exponent byte b and a signed byte q per feature, which
// stand for q 2^(b-127): b is the smallest with which the group's largest
// magnitude rounds to at most 127, within [least, most]. A power of two and
// not largest / 127: v 2^-e is exact, so q is a function of the inputs alone
// (no rounding of a scale comes before it), and q 2^e is exact in bfloat16,
// float16 and float32, so the matrix instructions of the linear layer's
// weight gradient take it without another rounding. It costs at most one of
// the eight bits. A group that holds an infinity or a NaN keeps b = 255 and
// reads back as NaN throughout.
//
// A row of F features takes 32 ceil(F / 32) value bytes (the rest of the
// last group is zero) and ceil(F / 32) exponent bytes, so rows of values are
// 32-byte aligned whatever F is.
#pragma once

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

// Eight consecutive features, zero past `valid`. Whole: one or two 16-byte
// loads (the address is 16-byte aligned and valid is 8 or 0).
template <typename T, bool Whole>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[kChunk]) {
  if constexpr (Whole) {
    vec<T, 8> raw = T(0);
    if (valid > 0) raw = *reinterpret_cast<const vec<T, 8>*>(p);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] = float(raw[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] = j < valid ? float(p[j]) : 0.f;
  }
}

template <typename T, bool Whole>
__device__ __forceinline__ void store8(T* p, int valid, const float (&v)[kChunk]) {
  if constexpr (Whole) {
    if (valid <= 0) return;
    vec<T, 8> raw;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) raw[j] = T(v[j]);
    *reinterpret_cast<vec<T, 8>*>(p) = raw;
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j)
      if (j < valid) p[j] = T(v[j]);
  }
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

// The eight values of this lane, as bytes; the quad of lanes that holds the
// group calls it together. T: the type that sets the exponent's range.
template <typename T>
__device__ __forceinline__ uint2 keep8(const float (&v)[kChunk], uint32_t& exponent) {
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < kChunk; ++j)
    largest = max(largest, __float_as_uint(v[j]) & 0x7fffffffu);
  largest = max(largest, dpp<0xB1>(largest));  // quad_perm [1,0,3,2]
  largest = max(largest, dpp<0x4E>(largest));  // quad_perm [2,3,0,1]
  exponent = kept_exponent<T>(largest);
  const float inverse = exponent == 255 ? 0.f : __uint_as_float((254u - exponent) << 23);
  // v 2^-e + 1.5 2^23 rounds v 2^-e to an integer (ties to even) whose low
  // byte is q; the clamp acts only at `most`.
  constexpr float magic = 12582912.f;
  uint32_t bits[kChunk];
#pragma unroll
  for (int j = 0; j < kChunk; ++j) {
    const float t = __builtin_fmaf(v[j], inverse, magic);
    bits[j] = __float_as_uint(__builtin_amdgcn_fmed3f(t, magic - 127.f, magic + 127.f));
  }
  uint2 out;
  out.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits[3], bits[2], 0x0c0c0400u),
                                __builtin_amdgcn_perm(bits[1], bits[0], 0x0c0c0400u),
                                0x05040100u);
  out.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits[7], bits[6], 0x0c0c0400u),
                                __builtin_amdgcn_perm(bits[5], bits[4], 0x0c0c0400u),
                                0x05040100u);
  const uint32_t fine = exponent == 255 ? 0u : ~0u;
  out.x &= fine;
  out.y &= fine;
  return out;
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

// Whether rows of this type can be read and written in whole 16-byte pieces.
template <typename T>
inline bool whole_rows(const void* p, int64_t features, int64_t stride) {
  return features % kChunk == 0 && stride % kChunk == 0 &&
         reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

inline int64_t kept_groups(int64_t features) { return ceil_div(features, kGroup); }

}  // namespace gs
