// A dense layer on rows of vertices and its gradients.
//   z = x w^T + bias, y = residual + drop(act(z))
//   dz = drop(g) act'(z) with z computed again, gx = dz w, gw = dz^T x, gb = column sums of dz
#include <algorithm>

#include "launch_size.hpp"
#include "layers.hpp"
#include "tiles.hpp"

namespace nts {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// What a product's result becomes.
enum Use { kLayer, kSlope, kRows, kWeight };

struct DenseArgs {
  const void *a, *b;  // result [M, N] = sum over K terms
  uint32_t M, N, K, a_stride, b_stride;
  void *out;
  const void *bias, *more;  // more: the residual, or the gradient of y
  float *sums;              // kSlope: column sums of every row of tiles [tiles_m, N]; kWeight: the parts' results [parts, M, N], if there are several
  int act;
  DropArgs drop;
  uint32_t row0;  // of the launch, where dropout counts from
  uint32_t tiles_m, tiles_n, part_terms;
  bool streamed;
};

__device__ __forceinline__ float activate(float z, int act) {
  if (act == NTS_ACT_RELU) return z <= 0.0f ? 0.0f : z;
  if (act == NTS_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678f));
  if (act == NTS_ACT_SILU) return z / (1.0f + expf(-z));
  return z;
}
__device__ __forceinline__ float slope(float z, int act) {
  if (act == NTS_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;
  if (act == NTS_ACT_GELU) return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * expf(-0.5f * z * z) * 0.39894228f;
  if (act == NTS_ACT_SILU) {
    const float f = 1.0f / (1.0f + expf(-z));
    return f * (1.0f + z * (1.0f - f));
  }
  return 1.0f;
}

// Up to four neighbouring values of a row, those behind its end 0.
template <typename T>
__device__ __forceinline__ void get_columns(const T *at, uint32_t count, float *v) {
  if (count >= 4u) {
    get_values<4>(at, v);
  } else {
#pragma unroll
    for (uint32_t c = 0; c < 3; ++c) v[c] = c < count ? get_value(at + c) : 0.0f;
    v[3] = 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void put_columns(T *at, uint32_t count, const float *v, bool streamed) {
  if (count >= 4u) {
    put_values<4>(at, v, streamed);
  } else {
#pragma unroll
    for (uint32_t c = 0; c < 3; ++c)
      if (c < count) put_value(at + c, v[c]);
  }
}
// Drops of the four columns of a row from c on, a multiple of 4.
__device__ __forceinline__ void drop_columns(const DropArgs &d, uint32_t step, uint32_t row, uint32_t c, float *v) {
  if (!d.threshold) return;
  const uint4 n = row_numbers(d, step, row, c >> 3);
  const uint32_t w0 = c & 4u ? n.z : n.x, w1 = c & 4u ? n.w : n.y;
  v[0] = (w0 & 0xFFFFu) >= d.threshold ? v[0] * d.scale : 0.0f;
  v[1] = (w0 >> 16) >= d.threshold ? v[1] * d.scale : 0.0f;
  v[2] = (w1 & 0xFFFFu) >= d.threshold ? v[2] * d.scale : 0.0f;
  v[3] = (w1 >> 16) >= d.threshold ? v[3] * d.scale : 0.0f;
}
// Columns c .. c + 3 of row i, sums of products in v: the layer's output, or the gradient of its sums, which v keeps.
template <typename T, int USE>
__device__ __forceinline__ void finish_columns(const DenseArgs &p, uint32_t step, uint64_t i, uint32_t c, float *v) {
  const uint32_t count = p.N - c;
  T *const to = static_cast<T *>(p.out) + i * p.N + c;
  if (USE == kLayer || USE == kSlope) {
    if (p.bias) {
      float bias[4];
      get_columns(static_cast<const T *>(p.bias) + c, count, bias);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += bias[k];
    }
    float more[4] = {};
    if (p.more) get_columns(static_cast<const T *>(p.more) + i * p.N + c, count, more);
    if (USE == kLayer) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = activate(v[k], p.act);
      drop_columns(p.drop, step, p.row0 + static_cast<uint32_t>(i), c, v);
      if (p.more) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += more[k];
      }
    } else {
      drop_columns(p.drop, step, p.row0 + static_cast<uint32_t>(i), c, more);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = k < static_cast<int>(count) ? more[k] * slope(v[k], p.act) : 0.0f;
    }
  }
  put_columns(to, count, v, p.streamed);
}

// ---- tiles ------------------------------------------------------------------------------------------
// A block of four wavefronts takes 128 rows of the result by 128 columns, 32 terms at a time through LDS, where both operands lie
// with the terms of a row or column side by side.  Operands of 32 bits are split into three bf16 parts, each the nearest to what the ones
// before it leave: x = hi + mid + lo up to 2^-27 of x, and of the nine products the three that are below 2^-26 of the whole are
// left out, so that the sums in 32 bits are as good as a 32-bit product's.  An infinity's mid part is NaN: elements that are not finite
// are computed again term by term.
constexpr uint32_t kTile = 128, kTerms = 32;
// Where 8 of a row's 32 terms lie: the 16 lanes that read one part of 16 rows meet all banks once.
__device__ __forceinline__ uint32_t tile_at(uint32_t row, uint32_t part) { return row * kTerms + ((part ^ (row >> 2)) & 3u) * 8u; }

template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;

template <typename T>
__device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 multiply<F16>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Sixteen terms of one row (ALONG: the terms lie side by side) or column of an operand, on their way from memory to LDS.
template <typename T, bool ALONG>
struct Terms {
  typedef typename ValueOf<T>::raw raw;
  raw v[16];
  __device__ __forceinline__ void request(const T *from, uint32_t stride) {  // of the first of the sixteen
    if (ALONG) {
      constexpr int N = 16 / sizeof(raw);
#pragma unroll
      for (int i = 0; i < 16; i += N) {
        const typename Pack<T, N>::type q = *reinterpret_cast<const typename Pack<T, N>::type *>(from + i);
#pragma unroll
        for (int k = 0; k < N; ++k) v[i + k] = q[k];
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) v[i] = *reinterpret_cast<const raw *>(from + static_cast<uint64_t>(i) * stride);
    }
  }
  __device__ __forceinline__ void request_some(const T *from, uint32_t stride, uint32_t count) {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      v[i] = i < count ? *reinterpret_cast<const raw *>(from + (ALONG ? i : static_cast<uint64_t>(i) * stride)) : static_cast<raw>(0);
  }
};
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
}
// Eight terms to the planes at `to`.
__device__ __forceinline__ void keep(const float *v, uint16_t *to, uint32_t plane) {
  u32x4 w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      w[c][i] = pair_of(a, b);
      a -= __uint_as_float(w[c][i] << 16), b -= __uint_as_float(w[c][i] & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int c = 0; c < 3; ++c) *reinterpret_cast<u32x4 *>(to + c * plane) = w[c];
}
__device__ __forceinline__ void keep(const uint16_t *v, uint16_t *to, uint32_t) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = v[2 * i] | static_cast<uint32_t>(v[2 * i + 1]) << 16;
  *reinterpret_cast<u32x4 *>(to) = w;
}

template <typename T, int USE>
__global__ __launch_bounds__(256, 2) void dense_tile_kernel(DenseArgs p) {
  constexpr bool kAlongA = USE != kWeight, kAlongB = USE == kLayer || USE == kSlope;
  constexpr int P = kPlanes<T>;
  constexpr uint32_t kPlane = kTile * kTerms;
  __shared__ __attribute__((aligned(16))) uint16_t tile[2 * P * kPlane > 8192 ? 2 * P * kPlane : 8192];
  uint16_t *const ta = tile, *const tb = tile + P * kPlane;
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = wave_of_block(), r = lane & 15u, part = lane >> 4;
  uint32_t tm, tn;
  tile_of(p.tiles_n, p.tiles_m >= kXcdTiles, 1, &tm, &tn);
  if (tm >= p.tiles_m) return;
  const uint32_t step = USE == kLayer || USE == kSlope ? drop_step(p.drop) : 0u;
  if (USE == kLayer && p.drop.step_kept && blockIdx.x == 0 && t == 0) *p.drop.step_kept = step;
  const uint64_t m0 = static_cast<uint64_t>(tm) * kTile;
  const uint32_t n0 = tn * kTile;
  const uint64_t begin = static_cast<uint64_t>(blockIdx.z) * p.part_terms, end = min(static_cast<uint64_t>(p.K), begin + p.part_terms);
  // Two threads take a row's 32 terms where they lie side by side, otherwise neighbouring threads have neighbouring columns.  Rows and
  // columns that the result does not have read some other of it.
  const uint32_t ra = kAlongA ? t >> 1 : t & 127u, ka = kAlongA ? (t & 1u) * 16u : (t >> 7) * 16u;
  const uint32_t rb = kAlongB ? t >> 1 : t & 127u, kb = kAlongB ? (t & 1u) * 16u : (t >> 7) * 16u;
  const uint64_t ma = min(m0 + ra, static_cast<uint64_t>(p.M - 1u)), nb = min(n0 + rb, p.N - 1u);
  const T *const from_a = static_cast<const T *>(p.a) + (kAlongA ? ma * p.a_stride + ka : ka * static_cast<uint64_t>(p.a_stride) + ma);
  const T *const from_b = static_cast<const T *>(p.b) + (kAlongB ? nb * p.b_stride + kb : kb * static_cast<uint64_t>(p.b_stride) + nb);
  Terms<T, kAlongA> va;
  Terms<T, kAlongB> vb;
  auto request = [&](uint64_t k) __attribute__((always_inline)) {
    const T *const at_a = from_a + (kAlongA ? k : k * p.a_stride), *const at_b = from_b + (kAlongB ? k : k * p.b_stride);
    if (k + kTerms <= end) {
      va.request(at_a, p.a_stride);
      vb.request(at_b, p.b_stride);
    } else {
      const uint32_t left = k < end ? static_cast<uint32_t>(end - k) : 0u;
      va.request_some(at_a, p.a_stride, left > ka ? left - ka : 0u);
      vb.request_some(at_b, p.b_stride, left > kb ? left - kb : 0u);
    }
  };
  const uint32_t wm = wave / 2u * 64u, wn = wave % 2u * 64u;
  f32x4 acc[4][4] = {};
  request(begin);
  for (uint64_t k = begin; k < end; k += kTerms) {
#pragma unroll
    for (uint32_t i = 0; i < 16; i += 8) {
      keep(va.v + i, ta + tile_at(ra, (ka + i) / 8u), kPlane);
      keep(vb.v + i, tb + tile_at(rb, (kb + i) / 8u), kPlane);
    }
    __syncthreads();
    if (k + kTerms < end) request(k + kTerms);
    u32x4 b[P][4];
#pragma unroll
    for (int c = 0; c < P; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) b[c][j] = *reinterpret_cast<const u32x4 *>(tb + c * kPlane + tile_at(wn + j * 16 + r, part));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 a[P];
#pragma unroll
      for (int c = 0; c < P; ++c) a[c] = *reinterpret_cast<const u32x4 *>(ta + c * kPlane + tile_at(wm + i * 16 + r, part));
      // b is the first operand: a lane then ends up with four neighbouring columns of one row of the result
#pragma unroll
      for (int s = P - 1; s >= 0; --s)
#pragma unroll
        for (int c = 0; c <= s; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = multiply<T>(b[s - c][j], a[c], acc[i][j]);
    }
    __syncthreads();
  }
  // A lane has four columns of 16 rows: through LDS, 16 rows at a time, they become lines of 64 columns (part c of row r at c ^ r).
  f32x4 *const mine = reinterpret_cast<f32x4 *>(tile) + wave * 256u;
  float sums[4] = {};
#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[r * 16u + ((j * 4u + part) ^ r)] = acc[m][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
      const uint32_t row = q * 4u + lane / 16u, c = n0 + wn + (lane & 15u) * 4u;
      const uint64_t i = m0 + wm + m * 16u + row;
      const f32x4 got = mine[row * 16u + ((lane & 15u) ^ row)];
      if (i >= p.M || c >= p.N) continue;
      float v[4] = {got.x, got.y, got.z, got.w};
      if (P == 3) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          if (fabsf(v[k]) < INFINITY || c + k >= p.N) continue;
          const float *x = static_cast<const float *>(p.a) + (kAlongA ? i * p.a_stride : i), *y = static_cast<const float *>(p.b) + (kAlongB ? static_cast<uint64_t>(c + k) * p.b_stride : c + k);
          v[k] = 0.0f;
          for (uint64_t f = begin; f < end; ++f) v[k] = fmaf(x[kAlongA ? f : f * p.a_stride], y[kAlongB ? f : f * p.b_stride], v[k]);
        }
      }
      if (USE == kWeight && p.sums) {
        put_columns(p.sums + (static_cast<uint64_t>(blockIdx.z) * p.M + i) * p.N + c, p.N - c, v, false);
        continue;
      }
      finish_columns<T, USE>(p, step, i, c, v);
      if (USE == kSlope) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[k] += v[k];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (USE != kSlope || !p.sums) return;
  __syncthreads();
  float(*const both)[kTile] = reinterpret_cast<float(*)[kTile]>(tile);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    sums[k] += __shfl_xor(sums[k], 16, kWave);
    sums[k] += __shfl_xor(sums[k], 32, kWave);
    if (lane < 16u) both[wave / 2u][wn + lane * 4u + k] = sums[k];
  }
  __syncthreads();
  if (t < kTile && n0 + t < p.N) p.sums[static_cast<uint64_t>(tm) * p.N + n0 + t] = both[0][t] + both[1][t];
}

// ---- few rows ---------------------------------------------------------------------------------------
// A prediction for some vertices: the weight is what has to be read, once.  A wavefront takes a column of the result for R rows; its
// lanes take 8 terms each at a time, in 32 bits.
constexpr uint32_t kFewRows = 8, kFewWaves = 4;
template <typename T, int R>
__global__ __launch_bounds__(kFewWaves *kWave) void dense_few_kernel(DenseArgs p) {
  const uint32_t lane = threadIdx.x & (kWave - 1), c = blockIdx.x * kFewWaves + wave_of_block();
  const uint64_t i0 = static_cast<uint64_t>(blockIdx.y) * R, last = p.M - 1u;
  const uint32_t step = drop_step(p.drop);
  if (p.drop.step_kept && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.drop.step_kept = step;
  if (c >= p.N) return;
  const T *const x = static_cast<const T *>(p.a), *const w = static_cast<const T *>(p.b) + static_cast<uint64_t>(c) * p.K;
  float acc[R] = {};
  for (uint32_t k = lane * 8u; k < p.K; k += kWave * 8u) {
    float wv[8], xv[R][8];
    const uint32_t count = p.K - k;
#pragma unroll
    for (int i = 0; i < 8; ++i) wv[i] = 0.0f;
    if (count >= 8u) {
      get_values<8>(w + k, wv);
#pragma unroll
      for (int q = 0; q < R; ++q) get_values<8>(x + min(i0 + q, last) * p.K + k, xv[q]);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        if (i < count) wv[i] = get_value(w + k + i);
#pragma unroll
        for (int q = 0; q < R; ++q) xv[q][i] = i < count ? get_value(x + min(i0 + q, last) * p.K + k + i) : 0.0f;
      }
    }
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[q] = fmaf(wv[i], xv[q][i], acc[q]);
  }
#pragma unroll
  for (int q = 0; q < R; ++q) acc[q] = group_sum<kWave>(acc[q]);
  float v = acc[0];
#pragma unroll
  for (int q = 1; q < R; ++q) v = lane == static_cast<uint32_t>(q) ? acc[q] : v;
  const uint64_t i = i0 + lane;
  if (lane >= R || i >= p.M) return;
  if (p.bias) v += get_value(static_cast<const T *>(p.bias) + c);
  v = activate(v, p.act);
  if (p.drop.threshold) {
    const uint4 n = row_numbers(p.drop, step, static_cast<uint32_t>(i), c >> 3);
    const uint32_t word = c & 4u ? (c & 2u ? n.w : n.z) : (c & 2u ? n.y : n.x);
    v = (c & 1u ? word >> 16 : word & 0xFFFFu) >= p.drop.threshold ? v * p.drop.scale : 0.0f;
  }
  if (p.more) v += get_value(static_cast<const T *>(p.more) + i * p.N + c);
  put_value(static_cast<T *>(p.out) + i * p.N + c, v);
}

// ---- sums -------------------------------------------------------------------------------------------
// The gradient of y where the activation's slope is 1: dropped (if out is not null) and summed by columns.  A block takes 64 columns and
// every gridDim.y-th group of 4 rows.
template <typename T>
__global__ __launch_bounds__(256) void dense_columns_kernel(DenseArgs p) {
  __shared__ float sums[4][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block(), c = blockIdx.x * kWave + lane;
  const uint32_t step = drop_step(p.drop);
  float sum = 0.0f;
  if (c < p.N) {
    for (uint64_t i = blockIdx.y * 4ull + wave; i < p.M; i += gridDim.y * 4ull) {
      float v = get_value(static_cast<const T *>(p.more) + i * p.N + c);
      if (p.drop.threshold) {
        const uint4 n = row_numbers(p.drop, step, static_cast<uint32_t>(i), c >> 3);
        const uint32_t word = c & 4u ? (c & 2u ? n.w : n.z) : (c & 2u ? n.y : n.x);
        v = (c & 1u ? word >> 16 : word & 0xFFFFu) >= p.drop.threshold ? v * p.drop.scale : 0.0f;
      }
      if (p.out) put_value(static_cast<T *>(p.out) + i * p.N + c, v);
      sum += v;
    }
  }
  if (!p.sums) return;
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < p.N) p.sums[static_cast<uint64_t>(blockIdx.y) * p.N + c] = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
}

// out = the sum of `parts` arrays of `count` floats, in order: the wavefronts take every kSumWaves-th part of 64 values, and the first
// adds up what they have.
constexpr uint32_t kSumWaves = 16;
template <typename T>
__global__ __launch_bounds__(kSumWaves *kWave) void dense_sum_kernel(T *__restrict__ out, const float *__restrict__ from, uint64_t count, uint32_t parts) {
  __shared__ float sums[kSumWaves][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block();
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * kWave + lane;
  float sum = 0.0f;
  if (i < count) {
#pragma unroll 8
    for (uint32_t k = wave; k < parts; k += kSumWaves) sum += from[k * count + i];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave || i >= count) return;
#pragma unroll
  for (uint32_t w = 1; w < kSumWaves; ++w) sum += sums[w][lane];
  put_value(out + i, sum);
}

// ---- launches ---------------------------------------------------------------------------------------
constexpr uint64_t kStreamed = 32ull << 20;  // an output from this size on is more than the L2s hold

template <int USE>
int launch_tiles(DenseArgs p, int type, uint32_t parts, hipStream_t stream) {
  p.tiles_n = ceil_div(p.N, kTile);
  const size_t size = type_size(type);
  p.streamed = static_cast<uint64_t>(p.M) * p.N * size >= kStreamed;
  // launches of at most 2^24 - 1 blocks: rows of the result in turns
  const uint64_t turn = USE == kWeight ? p.M : static_cast<uint64_t>(kMostBlocks / p.tiles_n - kXcdTiles) * kTile;
  for (uint64_t first = 0; first < p.M; first += turn) {
    DenseArgs q = p;
    q.M = static_cast<uint32_t>(std::min<uint64_t>(turn, p.M - first));
    q.tiles_m = ceil_div(q.M, kTile);
    q.row0 = static_cast<uint32_t>(first);
    if (first) {
      q.a = static_cast<const char *>(p.a) + first * p.a_stride * size;
      q.out = static_cast<char *>(p.out) + first * p.N * size;
      if (p.more) q.more = static_cast<const char *>(p.more) + first * p.N * size;
      if (p.sums) q.sums = p.sums + first / kTile * p.N;
    }
    const dim3 grid(tile_blocks(q.tiles_m, q.tiles_n, 1), 1, parts);
    if (type == NTS_F32) hipLaunchKernelGGL((dense_tile_kernel<float, USE>), grid, dim3(256), 0, stream, q);
    else if (type == NTS_BF16) hipLaunchKernelGGL((dense_tile_kernel<Bf16, USE>), grid, dim3(256), 0, stream, q);
    else hipLaunchKernelGGL((dense_tile_kernel<F16, USE>), grid, dim3(256), 0, stream, q);
    NTS_LAUNCH_CHECK("dense_tile_kernel");
  }
  return NTS_OK;
}
template <typename T>
void launch_few(const DenseArgs &p, hipStream_t stream) {
  const dim3 grid(ceil_div(p.N, kFewWaves), ceil_div(p.M, kFewRows)), block(kFewWaves * kWave);
  if (p.M == 1) hipLaunchKernelGGL((dense_few_kernel<T, 1>), dim3(grid.x, 1), block, 0, stream, p);
  else hipLaunchKernelGGL((dense_few_kernel<T, kFewRows>), grid, block, 0, stream, p);
}
int launch_sum(void *out, int type, const float *from, uint64_t count, uint32_t parts, hipStream_t stream) {
  const dim3 grid(ceil_div(count, kWave)), block(kSumWaves * kWave);
  if (type == NTS_F32) hipLaunchKernelGGL(dense_sum_kernel<float>, grid, block, 0, stream, static_cast<float *>(out), from, count, parts);
  else if (type == NTS_BF16) hipLaunchKernelGGL(dense_sum_kernel<Bf16>, grid, block, 0, stream, static_cast<Bf16 *>(out), from, count, parts);
  else hipLaunchKernelGGL(dense_sum_kernel<F16>, grid, block, 0, stream, static_cast<F16 *>(out), from, count, parts);
  NTS_LAUNCH_CHECK("dense_sum_kernel");
  return NTS_OK;
}

// Parts of the weight's gradient, of few results and many terms: 512 blocks, two for a compute unit, and none of fewer than 256 terms.
struct Parts {
  uint32_t count, terms;
};
Parts weight_parts(uint32_t n, uint32_t N, uint32_t F) {
  const uint64_t tiles = static_cast<uint64_t>(ceil_div(N, kTile)) * ceil_div(F, kTile);
  const uint64_t want = std::max<uint64_t>(1, std::min<uint64_t>(512 / tiles, n / 256));
  const uint64_t terms = (n + want - 1) / want;
  Parts p;
  p.terms = static_cast<uint32_t>(std::min<uint64_t>((terms + kTerms - 1) / kTerms * kTerms, 0xFFFFFFE0u));
  p.count = std::max(1u, ceil_div(n, std::max(p.terms, 1u)));
  return p;
}

// The gradient's work: dz, the parts of the bias's sums and of the weight's.
struct Work {
  size_t sums, parts, bytes;
  uint32_t sum_parts;
  Parts weight;
};
Work grad_work(int type, uint32_t n, uint32_t N, uint32_t F, int act, bool dropout, bool rows, bool weight, bool bias) {
  Work w{};
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const bool keeps = (act != NTS_ACT_NONE || dropout) && n;
  w.sums = keeps ? up(static_cast<size_t>(n) * N * type_size(type)) : 0;
  w.sum_parts = act != NTS_ACT_NONE ? ceil_div(n, kTile) : static_cast<uint32_t>(std::min<uint64_t>(1024, ceil_div(n, 64)));
  w.parts = w.sums + (bias ? up(static_cast<size_t>(w.sum_parts) * N * sizeof(float)) : 0);
  w.weight = weight_parts(n, N, F);
  w.bytes = w.parts + (weight && w.weight.count > 1 ? static_cast<size_t>(w.weight.count) * N * F * sizeof(float) : 0);
  (void)rows;
  return w;
}

const char *bad_shapes(int type, uint32_t N, uint32_t F, int act, const nts_dropout_t *dropout) {
  if (!known_type(type)) return "unknown type";
  if (N == 0 || N > kMostColumns || F == 0 || F > kMostColumns) return "N or F is 0 or above 2^17";
  if (act < NTS_ACT_NONE || act > NTS_ACT_SILU) return "unknown activation";
  return bad_dropout(dropout);
}
int fail_in(const char *call, const char *why) {
  char text[160];
  snprintf(text, sizeof(text), "%s: %s", call, why);
  return fail(NTS_ERR_INVALID, text);
}

}  // namespace
}  // namespace nts

using namespace nts;

extern "C" {

int nts_dense(void *y, const void *x, const void *w, const void *bias, const void *residual, int type, uint32_t n, uint32_t N,
              uint32_t F, int activation, const nts_dropout_t *dropout, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_dense");
  if (const char *why = bad_shapes(type, N, F, activation, dropout)) return fail_in("nts_dense", why);
  if (n == 0) return NTS_OK;
  if (!y || !x || !w) return fail_in("nts_dense", "null pointer");
  for (const void *at : {static_cast<const void *>(y), x, w, bias, residual})
    if (!aligned_to(at, type_size(type))) return fail_in("nts_dense", "a value's alignment");
  DenseArgs p{};
  p.a = x, p.b = w, p.M = n, p.N = N, p.K = F, p.a_stride = F, p.b_stride = F, p.out = y, p.bias = bias, p.more = residual;
  p.act = activation, p.drop = drop_args(dropout), p.part_terms = F;
  if (n <= kFewRows) {
    if (type == NTS_F32) launch_few<float>(p, stream);
    else if (type == NTS_BF16) launch_few<Bf16>(p, stream);
    else launch_few<F16>(p, stream);
    NTS_LAUNCH_CHECK("nts_dense");
    return NTS_OK;
  }
  return launch_tiles<kLayer>(p, type, 1, stream);
}

size_t nts_dense_grad_work_bytes(int type, uint32_t n, uint32_t N, uint32_t F, int activation, int with_dropout, int with_rows, int with_weight, int with_bias) {
  if (bad_shapes(type, N, F, activation, nullptr)) return 0;
  return grad_work(type, n, N, F, activation, with_dropout != 0, with_rows != 0, with_weight != 0, with_bias != 0).bytes;
}

int nts_dense_grad(void *gx, void *gw, void *gb, const void *g, const void *x, const void *w, const void *bias, int type, uint32_t n,
                   uint32_t N, uint32_t F, int activation, const nts_dropout_t *dropout, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_dense_grad");
  const char *const name = "nts_dense_grad";
  if (const char *why = bad_shapes(type, N, F, activation, dropout)) return fail_in(name, why);
  if ((n == 0 || !gx) && !gw && !gb) return NTS_OK;
  const bool again = activation != NTS_ACT_NONE;  // z is needed
  if (n && (!g || ((gw || again) && !x) || ((gx || again) && !w))) return fail_in(name, "null pointer");
  for (const void *at : {static_cast<const void *>(gx), static_cast<const void *>(gw), static_cast<const void *>(gb), g, x, w, bias})
    if (!aligned_to(at, type_size(type))) return fail_in(name, "a value's alignment");
  const Work layout = grad_work(type, n, N, F, activation, dropout != nullptr, gx != nullptr, gw != nullptr, gb != nullptr);
  if (layout.bytes && (!work || !aligned_to(work, 16))) return fail_in(name, "needs nts_dense_grad_work_bytes of 16-byte-aligned work");
  char *const base = static_cast<char *>(work);
  float *const sums = gb ? reinterpret_cast<float *>(base + layout.sums) : nullptr;
  const void *dz = g;
  DenseArgs p{};
  p.drop = drop_args(dropout), p.act = activation;
  p.drop.step_kept = nullptr;
  if (n && (again || dropout || gb)) {
    DenseArgs q = p;
    q.more = g, q.M = n, q.N = N, q.sums = sums;
    if (again || dropout) dz = q.out = work;
    if (again) {
      q.a = x, q.b = w, q.K = F, q.a_stride = F, q.b_stride = F, q.bias = bias, q.part_terms = F;
      if (const int status = launch_tiles<kSlope>(q, type, 1, stream)) return status;
    } else {
      const dim3 grid(ceil_div(N, kWave), layout.sum_parts);
      if (type == NTS_F32) hipLaunchKernelGGL(dense_columns_kernel<float>, grid, dim3(256), 0, stream, q);
      else if (type == NTS_BF16) hipLaunchKernelGGL(dense_columns_kernel<Bf16>, grid, dim3(256), 0, stream, q);
      else hipLaunchKernelGGL(dense_columns_kernel<F16>, grid, dim3(256), 0, stream, q);
      NTS_LAUNCH_CHECK("dense_columns_kernel");
    }
  }
  if (gb)
    if (const int status = launch_sum(gb, type, sums, N, n ? layout.sum_parts : 0u, stream)) return status;
  if (gx && n) {
    DenseArgs q = p;
    q.a = dz, q.b = w, q.M = n, q.N = F, q.K = N, q.a_stride = N, q.b_stride = F, q.out = gx, q.part_terms = N;
    if (const int status = launch_tiles<kRows>(q, type, 1, stream)) return status;
  }
  if (gw) {
    DenseArgs q = p;
    q.a = dz, q.b = x, q.M = N, q.N = F, q.K = n, q.a_stride = N, q.b_stride = F, q.out = gw, q.part_terms = layout.weight.terms;
    const uint32_t parts = layout.weight.count;
    q.sums = parts > 1 ? reinterpret_cast<float *>(base + layout.parts) : nullptr;
    if (const int status = launch_tiles<kWeight>(q, type, parts, stream)) return status;
    if (parts > 1)
      if (const int status = launch_sum(gw, type, q.sums, static_cast<uint64_t>(N) * F, parts, stream)) return status;
  }
  return NTS_OK;
}

}  // extern "C"
