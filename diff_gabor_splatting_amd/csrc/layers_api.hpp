// What the entry points of the layer kernels share: types and row checks.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gabor_layers.h"
#include "kept8.hpp"

#define GS_CHECK(call)                         \
  do {                                         \
    int gs_status_ = (call);                   \
    if (gs_status_ != GS_OK) return gs_status_; \
  } while (0)

namespace gs {

// Widest row: column indices stay in 32 bits with room to spare.
constexpr int64_t kMostFeatures = int64_t(1) << 24;

inline int check_type(const char* name, int32_t dtype) {
  GS_REQUIRE(dtype == GS_FLOAT32 || dtype == GS_BFLOAT16 || dtype == GS_FLOAT16,
             GS_ERR_ARGUMENT, "%s: unknown type %d", name, int(dtype));
  return GS_OK;
}

// rows x features values, rows `stride` apart (one row has any stride).
inline int check_rows(const char* name, int32_t dtype, int64_t rows, int64_t features,
                      int64_t stride) {
  GS_CHECK(check_type(name, dtype));
  GS_REQUIRE(rows >= 0, GS_ERR_ARGUMENT, "%s: negative row count", name);
  GS_REQUIRE(features >= 1 && features <= kMostFeatures, GS_ERR_ARGUMENT,
             "%s: features must be 1 through %lld", name, (long long)kMostFeatures);
  GS_REQUIRE(rows <= 0x7fffffffffffLL / features, GS_ERR_OVERFLOW, "%s: too many rows", name);
  GS_REQUIRE(stride >= features || rows <= 1, GS_ERR_ARGUMENT, "%s: rows overlap", name);
  return GS_OK;
}

// Orders a wave's own LDS writes before its other lanes' reads, and those
// before later writes: the hardware keeps a wave's LDS order by itself, this
// keeps the compiler's.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// LDS beyond 64 KB is asked for, each time: the kernel may be running on a
// device where it was not.
inline int allow_lds(const void* kernel, size_t bytes) {
  if (bytes <= 64 * 1024) return GS_OK;
  GS_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
  return GS_OK;
}

// Calls `call` with a zero of the type.
template <typename F>
int with_type(int32_t dtype, F&& call) {
  switch (dtype) {
    case GS_FLOAT32: return call(float(0));
    case GS_BFLOAT16: return call(bf16(0.f));
    default: return call(f16(0));
  }
}

}  // namespace gs
