// Dropout whose mask is a function of the place and a seed, so that nothing
// is kept for the backward pass: y = x k / (1 - p), dx = dy k / (1 - p).
//
// The generator is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011): the seed's two words are the
// key, (column / 8, row's low word, row's high word, 0) the counter, and the
// four words it gives are 16 bits, low half first, for each of eight columns. A
// value is kept where its bits are at least t = rint(65536 p); its scale is
// 65536 / (65536 - t), so the mean is that of x whatever p was rounded to.
// 16 bits a value and not 32: the ten rounds of two 32 x 32 products each are
// what a lane spends its time on beside its loads, and they serve eight
// values this way. 1M x 512 bfloat16: 367 us a pass, 5.6 TB/s (410 under the
// profiler); the vector units issue for 72% of it.
#include "layers_api.hpp"

namespace gs {
namespace {

constexpr int kBlock = 256;

struct Masked {
  int64_t rows, features, stride;
  uint32_t per_row;  // chunks of eight columns to a row
  uint32_t least;    // bits from which on a value is kept
  float scale;
  uint64_t seed;
  const uint64_t* seed_at;  // where not null, the seed is read here
};

__device__ __forceinline__ void philox(uint32_t (&c)[4], uint64_t seed) {
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t a = uint64_t(c[0]) * 0xD2511F53u, b = uint64_t(c[2]) * 0xCD9E8D57u;
    c[0] = uint32_t(b >> 32) ^ c[1] ^ k0;
    c[2] = uint32_t(a >> 32) ^ c[3] ^ k1;
    c[1] = uint32_t(b);
    c[3] = uint32_t(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

template <typename T, bool Narrow, int Each>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const T* __restrict__ x, Masked m,
                                                         T* __restrict__ y) {
  const uint64_t seed = m.seed_at ? *m.seed_at : m.seed;
  const int64_t total = m.rows * m.per_row;
  const int64_t first = int64_t(blockIdx.x) * (kBlock * Each);
  // The workgroup's first chunk is divided into row and chunk once, in 64
  // bits, and the lanes divide what remains in 32.
  const int64_t row0 = first / m.per_row;
  const uint32_t rest0 = uint32_t(first - row0 * m.per_row);
  vec<T, kChunk> raw[Each];
  int64_t row[Each];
  uint32_t chunk[Each];
  int valid[Each];
#pragma unroll
  for (int i = 0; i < Each; ++i) {
    const uint32_t local = i * kBlock + threadIdx.x;
    const uint32_t down = (rest0 + local) / m.per_row;
    row[i] = row0 + down;
    chunk[i] = rest0 + local - down * m.per_row;
    const int64_t left = m.features - int64_t(chunk[i]) * kChunk;
    valid[i] = first + local < total ? int(left < kChunk ? left : kChunk) : 0;
    raw[i] = load_edge<T, kChunk, Narrow>(x + row[i] * m.stride + int64_t(chunk[i]) * kChunk,
                                          valid[i]);
  }
#pragma unroll
  for (int i = 0; i < Each; ++i) {
    if (valid[i] <= 0) continue;
    uint32_t word[4] = {chunk[i], uint32_t(row[i]), uint32_t(uint64_t(row[i]) >> 32), 0};
    philox(word, seed);
    raw[i] = settle<T, kChunk, Narrow>(raw[i], valid[i]);
    float v[kChunk];
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      const uint32_t bits = j & 1 ? word[j / 2] >> 16 : word[j / 2] & 0xffffu;
      v[j] = bits >= m.least ? float(raw[i][j]) * m.scale : 0.f;
    }
    store8<T>(y + row[i] * m.features + int64_t(chunk[i]) * kChunk, valid[i], v);
  }
}

// Chunks from which a thread takes four of them, and of a launch at most (a
// launch takes less than 2^32 threads).
constexpr int64_t kFour = int64_t(4) * 256 * kBlock;
constexpr int64_t kMostChunks = int64_t(4) << 30;

}  // namespace
}  // namespace gs

extern "C" int gs_dropout(int32_t dtype, double p, int64_t seed, const void* seed_at,
                          const void* x, int64_t row_stride, int64_t rows, int64_t features,
                          void* y, void* stream) {
  using namespace gs;
  clear_error();
  GS_CHECK(check_rows("gs_dropout", dtype, rows, features, row_stride));
  GS_REQUIRE(p >= 0.0 && p <= 1.0, GS_ERR_ARGUMENT, "gs_dropout: p must be 0 through 1");
  GS_REQUIRE(rows <= kMostChunks / ceil_div(features, kChunk), GS_ERR_OVERFLOW,
             "gs_dropout: too many rows");
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && y, GS_ERR_ARGUMENT, "null pointer passed to gs_dropout");
  const uint32_t least = uint32_t(std::nearbyint(65536.0 * p));
  const Masked m{rows, features, row_stride, uint32_t(ceil_div(features, kChunk)), least,
                 least < 65536 ? float(65536.0 / (65536.0 - least)) : 0.f, uint64_t(seed),
                 static_cast<const uint64_t*>(seed_at)};
  const int64_t total = rows * m.per_row;
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    auto launch = [&](auto narrow, auto each) {
      dropout_kernel<T, narrow.value, each.value>
          <<<dim3{unsigned(ceil_div(total, kBlock * each.value))}, kBlock, 0,
             static_cast<hipStream_t>(stream)>>>(static_cast<const T*>(x), m,
                                                 static_cast<T*>(y));
    };
    using one = std::integral_constant<int, 1>;
    using four = std::integral_constant<int, 4>;
    auto by_count = [&](auto narrow) {
      total >= kFour ? launch(narrow, four{}) : launch(narrow, one{});
    };
    features >= kChunk ? by_count(std::false_type{}) : by_count(std::true_type{});
    GS_LAUNCHED("dropout");
    return int(GS_OK);
  });
}
