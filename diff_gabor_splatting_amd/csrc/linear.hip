// Linear layers whose input is kept in 8 bits: y = x W^T + b and its
// gradients dx = dy W, dW = dy^T x8, db = the sum of dy's rows, x8 what the
// checkpoint stands for.
//
// All products run on the matrix cores with float32 accumulators (16x16x32
// for the 2-byte types, 16x16x4 for float32). What bounds them is memory up to
// about 256 features and outputs, the matrix cores beyond:
//
//   few_rows_kernel  y of up to eight rows: a wave to an output
//   rows_kernel      y and dx: the matrix in LDS, rows streamed past it
//   product_kernel   y and dx where the matrix has a side too long for that
//   sum_kernel       dW and db: tiles of dW over shares of the rows, whose
//                    partial sums join_kernel adds in their order
//
// No atomics: results do not depend on timing.
#include "matrix.hpp"

namespace gs {
namespace {

struct Product {
  int64_t m, n;     // C's rows and columns
  int64_t k;        // length of the sum
  int64_t tiles_n;
};

// C[m][n] = sum_k M(m, k) N(n, k) (+ bias[n]), for matrices with a side too
// long to stay in LDS (over 1,024 values, or over 32 panels wide): one
// 128 x 128 tile to a workgroup; a step of both sides is in registers while the step before is
// multiplied out of LDS. M is the rows, k contiguous; N the matrix, [n][k] in
// memory (NContiguous) or [k][n]. 50k x 2048 -> 2048 bfloat16: y 573 us (732
// TFLOP/s), dx 611.
template <typename T, bool NContiguous>
__global__ __launch_bounds__(kThreads) void product_kernel(Side<T> ms, Side<T> ns, Product p,
                                                           const T* __restrict__ bias,
                                                           T* __restrict__ out) {
  constexpr int depth = Mma<T>::depth;
  __shared__ __align__(16) T m_lds[kTileSize<T, true>];
  __shared__ __align__(16) T n_lds[kTileSize<T, NContiguous>];
  Staged<T, kEdge, depth> m_next;
  Staged<T, NContiguous ? kEdge : depth, NContiguous ? depth : kEdge> n_next;
  const int64_t m0 = blockIdx.x / p.tiles_n * kEdge, n0 = blockIdx.x % p.tiles_n * kEdge;
  const int wave = threadIdx.x >> 6;
  const int wave_m = (wave >> 1) * kWaveEdge, wave_n = (wave & 1) * kWaveEdge;
  f32x4 c[kTiles][kTiles];  // [m][n]
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) c[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](int64_t k) {
    m_next.load(ms, m0, k);
    if constexpr (NContiguous)
      n_next.load(ns, n0, k);
    else
      n_next.load(ns, k, n0);
  };
  fetch(0);
  for (int64_t k = 0; k < p.k; k += depth) {
    m_next.template store<kPitch<T, true>, false, true>(m_lds);
    n_next.template store<kPitch<T, NContiguous>, true, NContiguous>(n_lds);
    __syncthreads();
    if (k + depth < p.k) fetch(k + depth);
#pragma unroll
    for (int s = 0; s < depth; s += Mma<T>::step) {
      typename Mma<T>::Fragment a[kTiles], b[kTiles];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        a[i] = fragment<T, true>(m_lds, wave_m + 16 * i, s);
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
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int64_t m = m0 + wave_m + 16 * i + (lane & 15);
    if (m >= p.m) continue;
    float row[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) row[j] = c[i][j >> 2][j & 3] + offset[j];
    store_row<T>(out + m * p.n + n, p.n - n, row);
  }
}

// --------------------------------------------------------------------------
// y and dx: many rows against a small matrix.
//
// The matrix (W, or W transposed for dx) stays in LDS, laid out as the
// matrix instruction's fragments, for all the rows that a workgroup takes.
// A wave takes TM * 16 rows at a time and needs no other wave: no barriers
// after the matrix is in place, and its loads are `Ahead` steps (of 128 bytes
// of each row) ahead of its products, across tiles too.
//
// A fragment's lanes lie 16 rows apart in memory, and loading it so costs the
// address unit a cycle a lane (it was busy for 83% of the kernel). Rows are
// therefore loaded and results stored with eight lanes to 128 bytes of a row,
// and turned through 2 KB of LDS that the wave has to itself.
//
// 1M x 512 -> 512 bfloat16 (524 Gflop, 2.0 GB): y 562 us, with the 8-bit form
// 683, dx 555 (945 TFLOP/s; a library product of these sizes takes 770 and
// 711). In dx the matrix cores are busy for 51% of the time, the address unit
// for 50%, LDS for 55%, in y with the 8-bit form for 42%, 62% and 45%: eight
// waves, as many as the registers allow, do not fill any of them. 100k x 256 ->
// 256: 24, 31 to 36 and 24 to 27 us (4.3 TB/s). float32 is bound by its matrix
// instructions: 1M x 256 -> 256 1006 us (130 TFLOP/s).
//
// 32 compute units of an XCD are shared by whole sets of panels: where the
// panels are no divisor of 32 some stay idle (19 panels of float32 600 -> 600
// leave 104 of 256), and rows of fewer tiles than XCDs leave XCDs idle.

struct RowsProduct {
  int64_t rows, stride;
  int k, n;          // length of the sum and columns of C
  int panels;        // workgroups side by side, each with its columns of C
  int workers;       // workgroups to a panel
  int steps;         // of the sum, see steps_of
};

// The 8-bit form of one step of a tile's rows, as they were loaded: lane l
// has piece l % 8 of row 8 j + l / 8 of x[j]. `rows_left`: of the tile's.
template <typename T, int Loads>
__device__ __forceinline__ void keep_step(const vec<T, kPart<T>> (&x)[Loads], int64_t first,
                                          int rows_left, int s, int groups,
                                          uint8_t* __restrict__ values,
                                          uint8_t* __restrict__ exponents) {
  constexpr int part = kPart<T>;
  const int lane = threadIdx.x & 63, piece = lane & 7;
  const int in_step = piece * part / kGroup;  // group of the step
  const int group = s * (kStep<T> / kGroup) + in_step;
  uint8_t* const to_values = values + first * (groups * kGroup) + s * kStep<T>;
  uint8_t* const to_exponents = exponents + first * groups + s * (kStep<T> / kGroup);
#pragma unroll
  for (int j = 0; j < Loads; ++j) {
    const int row = 8 * j + (lane >> 3);
    uint32_t largest = largest_of<T, part>(x[j]);
    largest = max(largest, dpp<0xB1>(largest));  // quad_perm [1,0,3,2]
    largest = max(largest, dpp<0x4E>(largest));  // quad_perm [2,3,0,1]
    if constexpr (part == 4) largest = max(largest, dpp<0x141>(largest));  // row_half_mirror
    const uint32_t exponent = kept_exponent<T>(largest);
    float v[part];
    widen<T, part>(x[j], v);
    uint32_t bytes[part / 4];
    keep_bytes<T, part>(v, exponent, bytes);
    if (row < rows_left && group < groups) {
      uint8_t* const to = to_values + uint32_t(row * groups * kGroup + piece * part);
      if constexpr (part == 8)
        *reinterpret_cast<uint2*>(to) = make_uint2(bytes[0], bytes[1]);
      else
        *reinterpret_cast<uint32_t*>(to) = bytes[0];
      if (piece * part % kGroup == 0)
        to_exponents[uint32_t(row * groups + in_step)] = uint8_t(exponent);
    }
  }
}

// Ahead: steps on their way. Tail: k is no whole number of steps.
template <typename T, int TM, int TN, int Ahead, bool Transposed, bool Keep, bool Tail>
__global__ __launch_bounds__(kRowThreads) void rows_kernel(
    const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ bias, RowsProduct p,
    T* __restrict__ out, uint8_t* __restrict__ values, uint8_t* __restrict__ exponents) {
  constexpr int part = kPart<T>, step = kStep<T>, columns = 16 * TN;
  constexpr int loads = 2 * TM;  // of eight rows each
  typedef vec<T, part> Part;
  extern __shared__ __align__(16) char shared[];
  Part* const panel = reinterpret_cast<Part*>(shared);
  __shared__ Part turns[kRowWaves][128];
  __shared__ float offset[columns];
  // Workgroups go to the eight XCDs in turn: those that take the same rows
  // share one, and its L2.
  const int xcd = blockIdx.x & 7, in_xcd = blockIdx.x >> 3;
  const int at = in_xcd % p.panels;
  const int worker = in_xcd / p.panels * 8 + xcd;
  if (worker >= p.workers) return;
  const int n0 = at * columns;
  stage_panel<T, TN, Transposed>(w, p.k, p.n, p.steps, n0, panel);
  if (threadIdx.x < columns)
    offset[threadIdx.x] =
        bias && n0 + int(threadIdx.x) < p.n ? float(bias[n0 + threadIdx.x]) : 0.f;
  __syncthreads();

  const int lane = threadIdx.x & 63, q = lane >> 4, i16 = lane & 15;
  const int row8 = lane >> 3, piece = lane & 7;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Part* const turn = turns[wave];
  const int groups = (p.k + kGroup - 1) / kGroup;
  // Steps that lie together in memory go to one panel, whole lines of it.
  const int keep_each = (p.steps + p.panels - 1) / p.panels;
  const int keep_from = at * keep_each, keep_to = keep_from + keep_each;
  const int64_t tiles = (p.rows + 16 * TM - 1) / (16 * TM);
  const int64_t each = int64_t(p.workers) * kRowWaves;
  // Tiles go round the workgroups first, then round their waves.
  int64_t tile = worker + int64_t(wave) * p.workers;
  if (tile >= tiles) return;

  // What is on its way: the loop below takes ring[u] and sends for the step
  // `Ahead` later in its place. Past the last tile it sends for that one
  // again, so that the number of loads under way is always the same.
  Part ring[Ahead][loads];
  const T* base;
  uint32_t from[loads];
  int64_t sent = tile;
  int sent_step = 0;
  auto turn_to = [&](int64_t of) {
    const int64_t first = of * (16 * TM);
    const int most = int(p.rows - first < 16 * TM ? p.rows - first : 16 * TM) - 1;
    base = x + first * p.stride;
#pragma unroll
    for (int j = 0; j < loads; ++j)  // rows past the end repeat the last one
      from[j] = uint32_t(min(8 * j + row8, most) * int(p.stride) + piece * part);
  };
  turn_to(tile);
  auto send = [&](Part (&to)[loads]) {
    const T* const at_step = base + sent_step * step;
    if (!Tail || (sent_step + 1) * step <= p.k) {
#pragma unroll
      for (int j = 0; j < loads; ++j) to[j] = load_packed<T, part>(at_step + from[j]);
    } else {
      const int left = min(p.k - sent_step * step - piece * part, part);
#pragma unroll
      for (int j = 0; j < loads; ++j)
        to[j] = load_edge<T, part, false>(at_step + from[j], left);
    }
    if (++sent_step == p.steps) {
      sent_step = 0;
      sent += each;
      turn_to(sent < tiles ? sent : tile);
    }
  };
#pragma unroll
  for (int u = 0; u < Ahead; ++u) send(ring[u]);

  for (; tile < tiles; tile += each) {
    f32x4 c[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int t = 0; t < TN; ++t) c[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.steps; s0 += Ahead) {
#pragma unroll
      for (int u = 0; u < Ahead; ++u) {
        const int s = s0 + u;
        if (Tail && (s + 1) * step > p.k) {
          const int left = min(p.k - s * step - piece * part, part);
#pragma unroll
          for (int j = 0; j < loads; ++j) ring[u][j] = settle<T, part, false>(ring[u][j], left);
        }
        Part b[TM][2];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            turn[turn_place(8 * j + row8, piece >> 2, piece & 3)] = ring[u][2 * i + j];
          wave_order();
#pragma unroll
          for (int h = 0; h < 2; ++h) b[i][h] = turn[turn_place(i16, h, q)];
          wave_order();
        }
        if constexpr (Keep) {
          // The panels share the rows' 8-bit form: each keeps its own steps.
          if (s >= keep_from && s < keep_to)
            keep_step<T, loads>(ring[u], tile * (16 * TM),
                                int(min(p.rows - tile * (16 * TM), int64_t(16 * TM))), s,
                                groups, values, exponents);
        }
        send(ring[u]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < TN; ++t) {
            const Part a = panel[((2 * s + h) * TN + t) * 64 + lane];
#pragma unroll
            for (int i = 0; i < TM; ++i) c[i][t] = multiply<T>(a, b[i][h], c[i][t]);
          }
      }
    }
    // Lane group q has, of every 64 bytes of the columns, the q-th 16.
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int v = 0; v < 4 * TN; v += 2 * part) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Part r;
#pragma unroll
          for (int j = 0; j < part; ++j) {
            const int from_fragment = v + h * part + j;
            r[j] = T(c[i][from_fragment >> 2][j & 3] +
                     offset[4 * (v + h * part) + q * part + j]);
          }
          turn[turn_place(i16, h, q)] = r;
        }
        wave_order();
        const int n = n0 + 4 * v + piece * part;
        const int inside = min(p.n - n, part);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t row = tile * (16 * TM) + 16 * i + 8 * j + row8;
          const Part r = turn[turn_place(8 * j + row8, piece >> 2, piece & 3)];
          store_valid<T, part>(out + row * p.n + n, row < p.rows ? inside : 0, r);
        }
        wave_order();
      }
    }
  }
}

// --------------------------------------------------------------------------
// dW and db: the sum over many rows of dy^T x8.
//
// A workgroup of eight waves (two along the outputs, four along the features)
// adds up a tile of dW over its share of the rows, 32 rows at a time: they
// are two steps ahead in registers, then in one of two LDS buffers, row by
// row as in memory, and the transposing LDS load makes fragments of them. One
// barrier a step. x8 is expanded to bfloat16 (float16) on the way. float32 dy
// is cut into three bfloat16 parts of eight bits each, whose sum it is, and
// each is multiplied by x8, which is exact in bfloat16: three products at
// the bfloat16 rate, a fifth of the time of float32's, and none of them
// rounded (an infinity or a NaN is the first part alone).
//
// 1M rows, 512 -> 512 bfloat16: 637 us (823 TFLOP/s; a library product of
// these sizes takes 2166), 100k, 256 -> 256: 30 and 6 for the partial sums.
// With the widest tiles the matrix cores are busy for 43% of the time, the
// vector units issue for 43% (a quarter of it matrix instructions, most of the
// rest the expansion of x8), LDS is busy for 32%: a step's barrier and the way
// from LDS to its first product take the rest.

// What the matrix instructions multiply.
template <typename T>
using Factor = std::conditional_t<sizeof(T) == 4, bf16, T>;

constexpr int kSumThreads = 512;

struct SumProduct {
  int64_t rows, stride;   // of dy
  int outputs, features;
  int tiles_m, tiles_n;   // of dW
  int splits;
  int64_t share;          // rows of a split, a multiple of a step's
};

template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 1;

// Eight values as their parts.
template <typename T>
__device__ __forceinline__ void parts_of(vec<T, 8> v, vec<Factor<T>, 8> (&out)[kParts<T>]) {
  if constexpr (sizeof(T) == 2) {
    out[0] = v;
  } else {
    vec<uint32_t, 4> words[3];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      uint32_t part[3][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t first = __float_as_uint(v[j + i]) & 0xffff0000u;
        const bool finite = (first & 0x7f800000u) != 0x7f800000u;
        // Whole NaN payloads keep to the first part.
        const uint32_t top =
            finite ? first : __float_as_uint(v[j + i]) | (v[j + i] != v[j + i] ? 0x10000u : 0u);
        const float rest = finite ? v[j + i] - __uint_as_float(first) : 0.f;
        const uint32_t second = __float_as_uint(rest) & 0xffff0000u;
        part[0][i] = top;
        part[1][i] = second;
        part[2][i] = __float_as_uint(rest - __uint_as_float(second));
      }
#pragma unroll
      for (int h = 0; h < 3; ++h)
        words[h][j / 2] = __builtin_amdgcn_perm(part[h][1], part[h][0], 0x07060302u);
    }
#pragma unroll
    for (int h = 0; h < 3; ++h) out[h] = __builtin_bit_cast(vec<bf16, 8>, words[h]);
  }
}

// A wave's tile: 16 A outputs x 16 B features.
template <typename T, int A, int B, int Rows, bool Narrow>
__global__ __launch_bounds__(kSumThreads) void sum_kernel(const T* __restrict__ dy,
                                                          const uint8_t* __restrict__ values,
                                                          const uint8_t* __restrict__ exponents,
                                                          SumProduct p,
                                                          float* __restrict__ partial) {
  typedef Factor<T> F;
  constexpr int parts = kParts<T>;
  constexpr int tile_m = 32 * A, tile_n = 64 * B;
  // 32 bytes past a multiple of 256: the eight rows that 32 lanes of a
  // fragment's load read lie in different banks.
  constexpr int pitch_m = tile_m + 16, pitch_n = tile_n + 16;
  constexpr int buffer = Rows * (parts * pitch_m + pitch_n);
  constexpr int across_m = tile_m / 8, across_n = tile_n / 16;
  constexpr int loads_m = Rows * across_m / kSumThreads;  // chunks of a thread
  constexpr bool all_n = Rows * across_n >= kSumThreads;
  static_assert(Rows * across_m % kSumThreads == 0 && Rows * across_n <= kSumThreads,
                "the threads do not divide the tile");
  extern __shared__ __align__(16) char shared[];
  F* const lds = reinterpret_cast<F*>(shared);

  // Workgroups go to the eight XCDs in turn: the tiles of one share of the
  // rows have one XCD, and its L2. With fewer shares than XCDs the tiles go
  // round, a workgroup each, so that their number is that of the launch.
  const int tiles = p.tiles_m * p.tiles_n;
  const int in_xcd = blockIdx.x >> 3;
  const bool shared_xcd = p.splits >= 8;
  const int split = shared_xcd ? in_xcd / tiles * 8 + int(blockIdx.x & 7)
                               : int(blockIdx.x % unsigned(p.splits));
  if (split >= p.splits) return;
  const int tile = shared_xcd ? in_xcd % tiles : int(blockIdx.x / unsigned(p.splits));
  const int m0 = tile / p.tiles_n * tile_m, n0 = tile % p.tiles_n * tile_n;
  const int64_t k0 = split * p.share;
  const int64_t k1 = k0 + p.share < p.rows ? k0 + p.share : p.rows;
  const int groups = (p.features + kGroup - 1) / kGroup;

  // Each thread's places: eight outputs of loads_m rows, 16 features of one.
  const int row_m = threadIdx.x / across_m, column_m = threadIdx.x % across_m * 8;
  const int row_n = threadIdx.x / across_n, column_n = threadIdx.x % across_n * 16;
  const int valid_m = min(p.outputs - m0 - column_m, 8);
  const bool ragged = p.outputs % 8;
  const bool has_n = (all_n || row_n < Rows) && n0 + column_n < groups * kGroup;
  const T* from_m = dy + (k0 + row_m) * p.stride + m0 + column_m;
  const uint8_t* from_n = values + (k0 + row_n) * (int64_t(groups) * kGroup) + n0 + column_n;
  const uint8_t* from_e = exponents + (k0 + row_n) * groups + (n0 + column_n) / kGroup;

  struct Load {
    vec<T, 8> m[loads_m];
    vec<uint32_t, 4> n;
    uint32_t exponent;
  };
  Load ahead[2];
  int64_t sent = k0;
  auto send = [&](Load& to) {
#pragma unroll
    for (int i = 0; i < loads_m; ++i) {
      constexpr int apart = kSumThreads / across_m;
      to.m[i] = load_edge<T, 8, Narrow>(from_m + i * apart * p.stride,
                                        sent + row_m + i * apart < k1 ? valid_m : 0);
    }
    to.n = vec<uint32_t, 4>{0, 0, 0, 0};
    to.exponent = 0;
    if (has_n && sent + row_n < k1) {
      to.n = *reinterpret_cast<const vec<uint32_t, 4>*>(from_n);
      to.exponent = *from_e;
    }
    sent += Rows;
    from_m += Rows * p.stride;
    from_n += Rows * int64_t(groups) * kGroup;
    from_e += Rows * groups;
  };
  float sum[8] = {};
  const bool sums = n0 == 0;
  auto put = [&](Load& from, F* to) {
#pragma unroll
    for (int i = 0; i < loads_m; ++i) {
      if (ragged) from.m[i] = settle<T, 8, Narrow>(from.m[i], valid_m);
      vec<F, 8> cut[parts];
      parts_of<T>(from.m[i], cut);
      if (sums) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += float(from.m[i][j]);
      }
#pragma unroll
      for (int h = 0; h < parts; ++h)
        *reinterpret_cast<vec<F, 8>*>(
            to + (h * Rows + row_m + i * (kSumThreads / across_m)) * pitch_m + column_m) =
            cut[h];
    }
    if (all_n || row_n < Rows) {
      const float scale = __uint_as_float(from.exponent << 23);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[8];
        read4(from.n[2 * h], scale, f);
        read4(from.n[2 * h + 1], scale, f + 4);
        vec<F, 8> v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = F(f[j]);
        *reinterpret_cast<vec<F, 8>*>(to + parts * Rows * pitch_m + row_n * pitch_n +
                                      column_n + 8 * h) = v;
      }
    }
  };

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wave_m = (wave >> 2) * 16 * A, wave_n = (wave & 3) * 16 * B;
  f32x4 c[A][B];
#pragma unroll
  for (int i = 0; i < A; ++i)
#pragma unroll
    for (int j = 0; j < B; ++j) c[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply_step = [&](const F* from) {
#pragma unroll
    for (int k = 0; k < Rows; k += 32) {
      vec<F, 8> b[B];
#pragma unroll
      for (int j = 0; j < B; ++j)
        b[j] = turned_fragment<F>(from + (parts * Rows) * pitch_m + k * pitch_n, pitch_n,
                                  wave_n + 16 * j);
#pragma unroll
      for (int h = 0; h < parts; ++h)
#pragma unroll
        for (int i = 0; i < A; ++i) {
          const vec<F, 8> a =
              turned_fragment<F>(from + (h * Rows + k) * pitch_m, pitch_m, wave_m + 16 * i);
#pragma unroll
          for (int j = 0; j < B; ++j) c[i][j] = Mma<F>::of(b[j], a, c[i][j]);
        }
    }
  };

  const int64_t steps = (k1 - k0 + Rows - 1) / Rows;
  send(ahead[0]);
  send(ahead[1]);
  put(ahead[0], lds);
  send(ahead[0]);
  __syncthreads();
  // Steps past the last read zeros: an odd count's last pair needs no case.
  for (int64_t s = 0; s < steps; s += 2) {
    put(ahead[1], lds + buffer);
    send(ahead[1]);
    multiply_step(lds);
    __syncthreads();
    put(ahead[0], lds);
    send(ahead[0]);
    multiply_step(lds + buffer);
    __syncthreads();
  }

  // Lane 16 q + i holds features 4 q .. 4 q + 3 of output i of a fragment.
  float* const mine = partial + int64_t(split) * p.outputs * (int64_t(p.features) + 1);
  const int q = lane >> 4, i16 = lane & 15;
#pragma unroll
  for (int i = 0; i < A; ++i) {
    const int m = m0 + wave_m + 16 * i + i16;
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int n = n0 + wave_n + 16 * j + 4 * q;
      store_valid<float, 4>(mine + int64_t(m) * p.features + n,
                            m < p.outputs ? min(p.features - n, 4) : 0, c[i][j]);
    }
  }
  if (sums) {
    // The threads of a column add up in LDS, in their order.
    float* const all = reinterpret_cast<float*>(shared);
#pragma unroll
    for (int j = 0; j < 8; ++j) all[row_m * tile_m + column_m + j] = sum[j];
    __syncthreads();
    const int m = m0 + threadIdx.x;
    if (int(threadIdx.x) < tile_m && m < p.outputs) {
      float total = 0.f;
      for (int i = 0; i < kSumThreads / across_m; ++i) total += all[i * tile_m + threadIdx.x];
      mine[int64_t(p.outputs) * p.features + m] = total;
    }
  }
}

// Adds `count` partial results of `size` values; the first `weights` of them
// are dW, the others db. A workgroup takes kThreads / Slices values; each
// slice of its threads adds every Slices-th result, and the slices meet in
// LDS, in their order. With one slice a workgroup goes on to further values:
// the grid stays at kJoinBlocks, far below the 2^32 threads of a launch.
constexpr int64_t kJoinBlocks = 1 << 20;

template <typename T, int Slices>
__global__ __launch_bounds__(kThreads) void join_kernel(const float* __restrict__ partial,
                                                        int count, int64_t size, int64_t weights,
                                                        T* __restrict__ dw, T* __restrict__ db) {
  constexpr int columns = kThreads / Slices;
  __shared__ float sums[Slices][columns];
  const int slice = threadIdx.x / columns, column = threadIdx.x % columns;
  auto add = [&](int64_t i) {
    float sum = 0.f;
#pragma unroll 8
    for (int s = slice; s < count; s += Slices) sum += partial[s * size + i];
    return sum;
  };
  auto put = [&](int64_t i, float sum) {
    if (i < weights) {
      if (dw) dw[i] = T(sum);
    } else if (db) {
      db[i - weights] = T(sum);
    }
  };
  int64_t i = int64_t(blockIdx.x) * columns + column;
  if constexpr (Slices == 1) {
    for (; i < size; i += int64_t(gridDim.x) * columns) put(i, add(i));
  } else {
    float sum = i < size ? add(i) : 0.f;
    sums[slice][column] = sum;
    __syncthreads();
    if (slice || i >= size) return;
    for (int s = 1; s < Slices; ++s) sum += sums[s][column];
    put(i, sum);
  }
}

// How dW's sum is cut: tiles of dW (fragments of a wave's tile along the
// outputs and the features), rows of a step, and shares of the rows.
//
// Tiles are as wide as dW asks for, and the widest only where there are rows
// enough: every workgroup writes a partial tile, so 256 x 256 of them cost 64
// MB whatever the rows (256 -> 256, bfloat16: 100k rows 45 us with 256-wide
// tiles, 38 with 128; 1M rows 185 and 225). Shares for two workgroups per
// compute unit of the narrower ones, which the registers allow but for float32's
// 128 x 128 tile: its 144 allow one, so that they come in two rounds. 64 rows
// at least to each, 128 from eight tiles on. Where the shares are no multiple of
// the eight XCDs some XCDs have one more of them than others (600 -> 600: 20
// shares of 25 tiles, 390 us for 200k rows where 127 would do).
//
// The bias's gradient alone goes by one feature's plan and reads none: the grid
// has one column of tiles, which multiplies zeros (a pass of 1M x 512 -> 512
// bfloat16 197 us, 589 with the matrix's gradient).
struct SumPlan {
  int a, b, step;
  int64_t tiles_m, tiles_n, splits, share;
};

SumPlan sum_plan(size_t size, int64_t rows, int64_t features, int64_t outputs) {
  SumPlan p{};
  // What of the wide tiles dW leaves empty, against the narrow ones, which
  // take 1.3 times as long for the same area (1M, 512 -> 512: 815 and 623, the
  // XCDs' load even in both).
  const int64_t wide = 4 * ceil_div(outputs, 256) * ceil_div(features, 256);
  const int64_t narrow = ceil_div(outputs, 128) * ceil_div(features, 128);
  const bool large = outputs > 128 && features > 128 && 10 * wide <= 13 * narrow &&
                     double(rows) * double(outputs) * double(features) >=
                         (size == 2 ? 2e10 : 1e10);
  p.a = large ? (size == 2 ? 8 : 4) : outputs <= 64 ? 2 : 4;
  p.b = large ? 4 : features <= 64 ? 1 : 2;
  p.step = p.a == 2 ? 64 : 32;
  p.tiles_m = ceil_div(outputs, 32 * p.a);
  p.tiles_n = ceil_div(features, 64 * p.b);
  const int64_t tiles = p.tiles_m * p.tiles_n;
  p.splits = std::max<int64_t>(1, (large ? 256 : 512) / tiles);
  const int64_t least = tiles < 8 ? 64 : 128;
  p.share = ceil_div(std::max(ceil_div(rows, p.splits), least), p.step) * p.step;
  p.splits = ceil_div(rows, p.share);
  return p;
}

// C = x matrix through rows_kernel; `taken` is false where the matrix or the
// stride is too large for it, or k less than a lane's part of a fragment.
template <typename T, bool Transposed>
int launch_rows(const char* name, const void* x, int64_t stride, const void* w, const void* bias,
                int64_t rows, int64_t k, int64_t n, void* out, void* values, void* exponents,
                hipStream_t stream, bool& taken) {
  const int fragments = panel_fragments(sizeof(T), rows, k, n);
  const int64_t panels = fragments ? ceil_div(n, 16 * fragments) : 0;
  taken = fragments && panels <= 32 && stride < (1 << 24) && k >= kPart<T>;
  if (!taken) return GS_OK;
  using std::integral_constant;
  auto launch = [&](auto tm, auto tn, auto ahead, auto keep, auto tail) {
    RowsProduct p{rows, stride, int(k), int(n), int(panels), 0, int(steps_of(sizeof(T), k))};
    static_assert(16 * tm.value == kRowTile, "tiles");
    const int64_t tiles = ceil_div(rows, kRowTile);
    p.workers = int(std::min<int64_t>(32 / panels * 8, tiles));
    const dim3 grid{unsigned(ceil_div(p.workers, 8) * panels * 8)};
    const size_t lds = size_t(p.steps) * 2 * tn.value * 1024;
    auto* const kernel =
        &rows_kernel<T, tm.value, tn.value, ahead.value, Transposed, keep.value, tail.value>;
    GS_CHECK(allow_lds(reinterpret_cast<const void*>(kernel), lds));
    kernel<<<grid, kRowThreads, lds, stream>>>(
        static_cast<const T*>(x), static_cast<const T*>(w), static_cast<const T*>(bias), p,
        static_cast<T*>(out), static_cast<uint8_t*>(values), static_cast<uint8_t*>(exponents));
    GS_LAUNCHED(name);
    return GS_OK;
  };
  using one = integral_constant<int, 1>;
  using two = integral_constant<int, 2>;
  using four = integral_constant<int, 4>;
  auto by_ahead = [&](auto tm, auto tn, auto keep) {
    const int64_t steps = steps_of(sizeof(T), k);
    if (k != steps * kStep<T>)
      switch (ahead_of(steps)) {
        case 1: return launch(tm, tn, one{}, keep, std::true_type{});
        case 2: return launch(tm, tn, two{}, keep, std::true_type{});
        default: return launch(tm, tn, four{}, keep, std::true_type{});
      }
    switch (ahead_of(steps)) {
      case 1: return launch(tm, tn, one{}, keep, std::false_type{});
      case 2: return launch(tm, tn, two{}, keep, std::false_type{});
      default: return launch(tm, tn, four{}, keep, std::false_type{});
    }
  };
  auto by_keep = [&](auto tm, auto tn) {
    if constexpr (!Transposed)
      if (values) return by_ahead(tm, tn, std::true_type{});
    return by_ahead(tm, tn, std::false_type{});
  };
  switch (fragments) {
    case 8: return by_keep(two{}, integral_constant<int, 8>{});
    case 4: return by_keep(two{}, four{});
    default:
      if constexpr (sizeof(T) == 4)
        return by_keep(two{}, two{});
      else
        return int(GS_OK);  // not reached: panel_fragments gives no such panel
  }
}

// --------------------------------------------------------------------------
// y of a few rows: a wave to an output, its lanes along the features. Each
// weight is read once, by as many workgroups as a quarter of the outputs,
// while the matrix instructions would wait for a panel in LDS first: 1 x 1024
// -> 1024 bfloat16 3.0 us against 9.7, eight rows 5.0 against 10.9. From nine
// rows on the panel's time is shared by enough of them.

constexpr int kFewRows = 8;

template <typename T, int Rows>
__global__ __launch_bounds__(kThreads) void few_rows_kernel(
    const T* __restrict__ x, int64_t stride, const T* __restrict__ w, const T* __restrict__ bias,
    int k, int n, T* __restrict__ y) {
  const int lane = threadIdx.x & 63;
  const int output = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (output >= n) return;
  const T* const row = w + int64_t(output) * k;
  float sum[Rows] = {};
#pragma unroll 4
  for (int c = lane * kChunk; c < k; c += 64 * kChunk) {
    const int valid = min(k - c, kChunk);
    float a[kChunk], b[Rows][kChunk];
    load8<T>(row + c, valid, a);
#pragma unroll
    for (int r = 0; r < Rows; ++r) load8<T>(x + r * stride + c, valid, b[r]);
#pragma unroll
    for (int r = 0; r < Rows; ++r)
#pragma unroll
      for (int j = 0; j < kChunk; ++j) sum[r] = __builtin_fmaf(a[j], b[r][j], sum[r]);
  }
  const float offset = bias ? float(bias[output]) : 0.f;
#pragma unroll
  for (int r = 0; r < Rows; ++r) {
#pragma unroll
    for (int step = 32; step; step >>= 1) sum[r] += __shfl_xor(sum[r], step);
    if (lane == 0) y[int64_t(r) * n + output] = T(sum[r] + offset);
  }
}

template <typename T>
int launch_few_rows(const void* x, int64_t stride, const void* w, const void* bias, int64_t rows,
                    int64_t k, int64_t n, void* y, hipStream_t stream) {
  const dim3 grid{unsigned(ceil_div(n, kThreads / 64))};
  auto launch = [&](auto count) {
    few_rows_kernel<T, count.value><<<grid, kThreads, 0, stream>>>(
        static_cast<const T*>(x), stride, static_cast<const T*>(w), static_cast<const T*>(bias),
        int(k), int(n), static_cast<T*>(y));
  };
  switch (rows) {
    case 1: launch(std::integral_constant<int, 1>{}); break;
    case 2: launch(std::integral_constant<int, 2>{}); break;
    case 3: launch(std::integral_constant<int, 3>{}); break;
    case 4: launch(std::integral_constant<int, 4>{}); break;
    case 5: launch(std::integral_constant<int, 5>{}); break;
    case 6: launch(std::integral_constant<int, 6>{}); break;
    case 7: launch(std::integral_constant<int, 7>{}); break;
    default: launch(std::integral_constant<int, 8>{}); break;
  }
  GS_LAUNCHED("few_rows_kernel");
  return GS_OK;
}

int check_linear(const char* name, int32_t dtype, int64_t rows, int64_t features,
                 int64_t outputs) {
  GS_CHECK(check_rows(name, dtype, rows, features, features));
  GS_CHECK(check_rows(name, dtype, rows, outputs, outputs));
  GS_REQUIRE(outputs <= kMostFeatures / 64 && features <= kMostFeatures / 64, GS_ERR_ARGUMENT,
             "%s: at most %lld features and outputs", name, (long long)(kMostFeatures / 64));
  return GS_OK;
}

// A launch takes less than 2^32 threads.
int check_launch(const char* name, int64_t blocks, int64_t threads) {
  GS_REQUIRE(blocks < (int64_t(1) << 32) / threads, GS_ERR_OVERFLOW, "%s: too many rows", name);
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
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (rows <= kFewRows) {  // with and without the 8-bit form: y is the same
      if (values)
        GS_CHECK(gs_checkpoint8_write(dtype, x, row_stride, rows, features, values, exponents,
                                      stream));
      return launch_few_rows<T>(x, row_stride, weight, bias, rows, features, outputs, y,
                                static_cast<hipStream_t>(stream));
    }
    bool taken = false;
    GS_CHECK((launch_rows<T, false>("linear forward", x, row_stride, weight, bias, rows, features,
                                    outputs, y, values, exponents,
                                    static_cast<hipStream_t>(stream), taken)));
    if (taken) return int(GS_OK);
    if (values)
      GS_CHECK(gs_checkpoint8_write(dtype, x, row_stride, rows, features, values, exponents,
                                    stream));
    const Side<T> ms{static_cast<const T*>(x), row_stride, rows, features};
    const Side<T> ns{static_cast<const T*>(weight), features, outputs, features};
    const Product p{rows, outputs, features, ceil_div(outputs, kEdge)};
    GS_CHECK(check_launch("gs_linear_forward", ceil_div(rows, kEdge) * p.tiles_n, kThreads));
    const dim3 grid{unsigned(ceil_div(rows, kEdge) * p.tiles_n)};
    product_kernel<T, true><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        ms, ns, p, static_cast<const T*>(bias), static_cast<T*>(y));
    GS_LAUNCHED("linear forward");
    return int(GS_OK);
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
    bool taken = false;
    GS_CHECK((launch_rows<T, true>("linear backward input", grad_y, grad_stride, weight, nullptr,
                                   rows, outputs, features, grad_x, nullptr, nullptr,
                                   static_cast<hipStream_t>(stream), taken)));
    if (taken) return int(GS_OK);
    const Side<T> ms{static_cast<const T*>(grad_y), grad_stride, rows, outputs};
    const Side<T> ns{static_cast<const T*>(weight), features, outputs, features};
    const Product p{rows, features, outputs, ceil_div(features, kEdge)};
    GS_CHECK(
        check_launch("gs_linear_backward_input", ceil_div(rows, kEdge) * p.tiles_n, kThreads));
    const dim3 grid{unsigned(ceil_div(rows, kEdge) * p.tiles_n)};
    product_kernel<T, false><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        ms, ns, p, static_cast<const T*>(nullptr), static_cast<T*>(grad_x));
    GS_LAUNCHED("linear backward input");
    return int(GS_OK);
  });
}

size_t gs_linear_backward_weight_workspace_size(int32_t dtype, int64_t rows, int64_t features,
                                                int64_t outputs) {
  using namespace gs;
  if (rows <= 0 || features <= 0 || outputs <= 0) return 0;
  const size_t size = dtype == GS_FLOAT32 ? 4 : 2;
  auto bytes = [&](int64_t planned, int64_t values) {
    return size_t(sum_plan(size, rows, planned, outputs).splits) * size_t(outputs * values) *
           sizeof(float);
  };
  return std::max(bytes(features, features + 1), bytes(1, 1));
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
  GS_REQUIRE(rows == 0 || (grad_y && ((values && exponents) || !grad_weight)), GS_ERR_ARGUMENT,
             "null pointer passed to gs_linear_backward_weight");
  const size_t need =
      gs_linear_backward_weight_workspace_size(dtype, rows, features, outputs);
  GS_REQUIRE(rows == 0 || (workspace && workspace_bytes >= need), GS_ERR_WORKSPACE,
             "workspace too small for gs_linear_backward_weight");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    int64_t splits = 0;
    const int64_t across = grad_weight ? features : 0;
    if (rows > 0) {
      const SumPlan plan = sum_plan(sizeof(T), rows, grad_weight ? features : 1, outputs);
      splits = plan.splits;
      const SumProduct p{rows, grad_stride, int(outputs), int(across), int(plan.tiles_m),
                         int(plan.tiles_n), int(splits), plan.share};
      const int64_t blocks =
          (splits >= 8 ? ceil_div(splits, 8) * 8 : splits) * plan.tiles_m * plan.tiles_n;
      GS_CHECK(check_launch("gs_linear_backward_weight", blocks, kSumThreads));
      auto launch = [&](auto a, auto b, auto narrow) {
        constexpr int step = a.value == 2 ? 64 : 32;
        constexpr int pitches = kParts<T> * (32 * a.value + 16) + 64 * b.value + 16;
        const size_t lds = std::max<size_t>(2 * size_t(step) * pitches * 2,
                                            size_t(kSumThreads) * 8 * sizeof(float));
        auto* const kernel = &sum_kernel<T, a.value, b.value, step, narrow.value>;
        GS_CHECK(allow_lds(reinterpret_cast<const void*>(kernel), lds));
        kernel<<<dim3{unsigned(blocks)}, kSumThreads, lds, s>>>(
            static_cast<const T*>(grad_y), static_cast<const uint8_t*>(values),
            static_cast<const uint8_t*>(exponents), p, static_cast<float*>(workspace));
        GS_LAUNCHED("linear backward weight");
        return int(GS_OK);
      };
      using std::integral_constant;
      using one = integral_constant<int, 1>;
      using two = integral_constant<int, 2>;
      using four = integral_constant<int, 4>;
      const int shape = plan.a * 10 + plan.b;
      using wide = std::false_type;
      using narrow = std::true_type;
      if (shape == 21 && outputs < 8) GS_CHECK(launch(two{}, one{}, narrow{}));
      if (shape == 22 && outputs < 8) GS_CHECK(launch(two{}, two{}, narrow{}));
      if (shape == 21 && outputs >= 8) GS_CHECK(launch(two{}, one{}, wide{}));
      if (shape == 22 && outputs >= 8) GS_CHECK(launch(two{}, two{}, wide{}));
      if (shape == 41) GS_CHECK(launch(four{}, one{}, wide{}));
      if (shape == 42) GS_CHECK(launch(four{}, two{}, wide{}));
      if constexpr (sizeof(T) == 2) {
        if (shape == 84) GS_CHECK(launch(integral_constant<int, 8>{}, four{}, wide{}));
      } else {
        if (shape == 44) GS_CHECK(launch(four{}, four{}, wide{}));
      }
    }
    const int64_t weights = outputs * across, size = weights + outputs;
    // Enough workgroups to fill the chip with few values, too: 65,792 values of
    // 128 partial results take 9.2 us with one slice and 6.2 with four, 147,840
    // 7.1 and 7.2.
    auto join = [&](auto slices) {
      join_kernel<T, slices.value>
          <<<dim3{unsigned(std::min(ceil_div(size, kThreads / slices.value), kJoinBlocks))},
             kThreads, 0, s>>>(
              static_cast<const float*>(workspace), int(splits), size, weights,
              static_cast<T*>(grad_weight), static_cast<T*>(grad_bias));
    };
    if (size >= 512 * kThreads)
      join(std::integral_constant<int, 1>{});
    else if (size >= 256 * kThreads)
      join(std::integral_constant<int, 4>{});
    else
      join(std::integral_constant<int, 16>{});
    GS_LAUNCHED("join_kernel");
    return int(GS_OK);
  });
}

}  // extern "C"
