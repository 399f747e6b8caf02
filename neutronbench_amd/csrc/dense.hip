// A dense layer on rows of vertices and its gradients.
//   z = x w^T + bias, y = residual + drop(act(z))
//   dz = drop(g) act'(z) with z computed again, gx = dz w, gw = dz^T x, gb = column sums of dz
// With relu and no residual y says what dz needs: it is above 0 where z is and the value was kept.  Then z is not computed again, and rows of up
// to 128 values have dz never stored: both products make it from g and y as they read them.  dz of 16-bit operands is not rounded to 16 bits, which
// would add an error as large as the results' own rounding: dz of a computed z is stored in 32 bits and multiplied as three bf16 parts, with as
// many parts of the other operand as it has (bf16 one, fp16 two), and otherwise the products are of g itself, dropped, and the scale of what is
// kept comes after the sums.  (Two parts of the operands' own type take as much memory and one matrix instruction less, but hold 16 to 17
// bits in bf16, and in fp16 nothing below 2^-25 or above 65,504.)
#include <algorithm>
#include <type_traits>

#include "dense_layout.hpp"
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
enum Use { kLayer, kSlope, kRows };

struct DenseArgs {
  const void *a, *b;  // result [M, N] = sum over K terms; b: the weight as prepared, or the second operand of the weight's gradient
  const void *w;      // the weight itself
  const void *y;      // masked gradients: a is g, and counts where y is not 0 or below, times mask_scale
  float mask_scale;
  float after;  // the products of 16-bit values for gx and gw, times this
  bool dz32;    // a is dz in 32 bits, the other operand and the result are of 16
  uint32_t M, N, K, a_stride, b_stride;
  void *out;
  const void *bias, *more;  // more: the residual, or the gradient of y
  float *sums;              // the workers' column sums [workers, N], or the parts of the weight's gradient [parts, M, N]; may be null
  float *column_sums;       // the weight's gradient: the parts' sums of a's columns [parts, M], may be null
  int act;
  DropArgs drop;
  uint32_t tiles_m, tiles_n, workers, part_terms;
  bool streamed;
};

// The normal distribution's share below z, and density * sqrt(2 pi).  The share behind |z| is density * t * (a polynomial of t = 1 / (1 + 0.265
// |z|)), so that it keeps its bits where it is small: below -3 it is off by 6e-7 of itself, of which the density's argument makes
// most.  Near 0, where that is off by 2e-7 at most, operands of 32 bits take 1/2 + z * (a polynomial of z^2) instead: for normally distributed z
// GELU is then off by 3.8e-8 of the whole and its slope by 3.9e-8, as with a 32-bit erf.  The polynomials are fitted to erfcx and erf, with a
// relative error of 1.2e-8.  (M. Abramowitz and I. Stegun's 7.1.26, four terms shorter than the first: 8.5e-8, 9.9e-8, and 5e-5 below -3.)
// 169,343 rows of 128 by 128 in bf16: 44 us forward, with 7.1.26 42 and with both polynomials 47; in 32 bits 75 and with 7.1.26 70.
template <typename T>
__device__ __forceinline__ float normal_below(float z, float *bell) {
  constexpr float kNear[] = {-6.80948867e-06f, 0.000111041116f, -0.00118383714f, 0.00997228272f, -0.0664902079f, 0.398942277f};
  constexpr float kFar[] = {0.0308208912f, -0.144228774f, 0.217815231f, -0.116362888f, 0.137953277f, 0.06031304f, 0.102700998f, 0.105246662f, 0.105741564f};
  const float a = fabsf(z), square = z * z, t = __builtin_amdgcn_rcpf(fmaf(a, 0.265f, 1.0f)), e = __builtin_amdgcn_exp2f(square * -0.72134752f);
  float far = kFar[0];
#pragma unroll
  for (int i = 1; i < 9; ++i) far = fmaf(far, t, kFar[i]);
  *bell = e;
  far *= t * e;
  if (sizeof(T) == 4) {
    float near = kNear[0];
#pragma unroll
    for (int i = 1; i < 6; ++i) near = fmaf(near, square, kNear[i]);
    if (a < 1.25f) return fmaf(z, near, 0.5f);
  }
  return z < 0.0f ? far : 1.0f - far;
}
// 1 / (1 + e^-z).  z log2 e is rounded by as much as it is large, which the exponential of 16 is off by 1e-6 for.  For operands of 32 bits what
// that leaves goes into a factor near 1 (beyond 200 nothing changes, and the factor is a number there); results of 16 bits do not see it, and
// forward 169,343 rows of 128 by 128 in bf16 would take 31.4 us instead of 29.1.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
  const float to = __builtin_amdgcn_fmed3f(z, -200.0f, 200.0f), x = to * -1.44269504f;
  const float rest = fmaf(to, -1.92596299e-8f, fmaf(to, -1.44269504f, -x));
  return __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(x), fmaf(rest, 0.693147181f, 1.0f), 1.0f));
}
template <typename T, int N>
__device__ __forceinline__ void activate(float *z, int act) {
  if (act == NTS_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = z[k] <= 0.0f ? 0.0f : z[k];
  } else if (act == NTS_ACT_GELU) {
    float bell;
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] *= normal_below<T>(z[k], &bell);
  } else if (act == NTS_ACT_SILU) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] *= sigmoid<T>(z[k]);
  }
}
// g times the activation's slopes at z.
template <typename T>
__device__ __forceinline__ void through_slope(float *z, const float *g, int act) {
  if (act == NTS_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = z[k] <= 0.0f ? 0.0f : g[k];
  } else if (act == NTS_ACT_GELU) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float bell;
      const float below = normal_below<T>(z[k], &bell);
      z[k] = g[k] * fmaf(z[k] * 0.39894228f, bell, below);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = sigmoid<T>(z[k]);
      z[k] = g[k] * (f * fmaf(z[k], 1.0f - f, 1.0f));
    }
  }
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
__device__ __forceinline__ float dropped(uint32_t number, const DropArgs &d, float v) { return number >= d.threshold ? v * d.scale : 0.0f; }
// Drops of the four columns from c on (a multiple of 4, neighbouring lanes take neighbouring fours) of two rows: a lane draws the eight
// numbers of one of them, of the second one where its columns are the upper four, and neighbours exchange what the other needs.
__device__ __forceinline__ void drop_two_rows(const DropArgs &d, uint32_t step, uint32_t row0, uint32_t row1, uint32_t c, float *v0, float *v1) {
  const bool upper = (c & 4u) != 0;
  const uint4 n = row_numbers(d, step, upper ? row1 : row0, c >> 3);
  const int give0 = static_cast<int>(upper ? n.x : n.z), give1 = static_cast<int>(upper ? n.y : n.w);
  const uint32_t got0 = __builtin_amdgcn_update_dpp(0, give0, 0xB1, 0xF, 0xF, true), got1 = __builtin_amdgcn_update_dpp(0, give1, 0xB1, 0xF, 0xF, true);
  const uint32_t a0 = upper ? got0 : n.x, a1 = upper ? got1 : n.y, b0 = upper ? n.z : got0, b1 = upper ? n.w : got1;
  v0[0] = dropped(a0 & 0xFFFFu, d, v0[0]), v0[1] = dropped(a0 >> 16, d, v0[1]);
  v0[2] = dropped(a1 & 0xFFFFu, d, v0[2]), v0[3] = dropped(a1 >> 16, d, v0[3]);
  v1[0] = dropped(b0 & 0xFFFFu, d, v1[0]), v1[1] = dropped(b0 >> 16, d, v1[1]);
  v1[2] = dropped(b1 & 0xFFFFu, d, v1[2]), v1[3] = dropped(b1 >> 16, d, v1[3]);
}

// ---- products ---------------------------------------------------------------------------------------
// Matrix instructions take 16 rows by 16 columns, 32 terms at a time.  Operands of 32 bits are split into three bf16 parts, each the nearest
// to what the ones before it leave: x = hi + mid + lo up to 2^-27 of x, and of the nine products the three that are below 2^-26 of the whole
// are left out, so that the sums in 32 bits are as good as a 32-bit product's.  An infinity's mid part is NaN: elements that are not
// finite are computed again term by term.
// Where 8 of a row's 32 terms lie in LDS.  A read of 16 bytes by a wavefront goes in quarters of 16 lanes, four neighbours' worth each of two
// parts (rows 0..3 and 12..15 of one with 4..11 of the next, and so on): with the four groups of rows at 0, 2, 3, 1 such a quarter meets
// every bank once, as 16 rows of one part do.  At 0, 1, 2, 3 every read took half as long again.
__host__ __device__ __forceinline__ uint32_t part_at(uint32_t row, uint32_t part) { return (part ^ (0x78u >> ((row >> 2 & 3u) * 2u))) & 3u; }
__host__ __device__ __forceinline__ uint32_t tile_at(uint32_t row, uint32_t part) { return row * kTerms + part_at(row, part) * 8u; }

template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;
// Parts of an operand of T that is multiplied by one of A: fp16 is two bf16 parts, whose exponents reach as far.
template <typename A, typename T>
constexpr int kPlanesBeside = sizeof(A) == sizeof(T) ? kPlanes<T> : 1;
template <>
constexpr int kPlanesBeside<float, F16> = 2;

template <typename T>
__device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 multiply<F16>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
}
// The parts of eight terms.
__device__ __forceinline__ void split8(const float *v, u32x4 *w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      const uint32_t both = pair_of(a, b);
      w[c][i] = both;
      a -= __uint_as_float(both << 16), b -= __uint_as_float(both & 0xFFFF0000u);
    }
  }
}
__device__ __forceinline__ void split8(const uint16_t *v, u32x4 *w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[0][i] = v[2 * i] | static_cast<uint32_t>(v[2 * i + 1]) << 16;
}
// The sum of an element's products term by term, as far as it is not NaN; mask: as DenseArgs' y, null for none.
template <typename T>
__device__ __forceinline__ float sum_of_terms(const float *x, const float *mask, float scale, uint64_t x_step, const T *y, uint64_t y_step, uint64_t count) {
  float sum = 0.0f;
  for (uint64_t f = 0; f < count && sum == sum; ++f) {
    const float v = !mask ? x[f * x_step] : mask[f * x_step] <= 0.0f ? 0.0f : x[f * x_step] * scale;
    sum = fmaf(v, get_value(y + f * y_step), sum);
  }
  return sum;
}

// The weight as the products want it: for every 128 columns of the result and 32 terms its parts, as they lie in LDS, zeros behind the
// ends.  ALONG: a column's terms lie side by side.  A thread takes eight terms.
struct PrepareArgs {
  const void *from;
  uint16_t *to;
  uint32_t columns, terms, stride, stages, tiles;
};
template <typename T, int P, bool ALONG>
__global__ __launch_bounds__(256) void dense_prepare_kernel(PrepareArgs p) {
  typedef typename ValueOf<T>::raw raw;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  // neighbouring threads have neighbouring terms or columns, as they lie in memory
  const uint32_t part = ALONG ? i % 4u : i / kTile % 4u, row = ALONG ? i / 4u % kTile : i % kTile, block = i / (4u * kTile);
  if (block >= p.stages * p.tiles) return;
  const uint32_t tile = block / p.stages, stage = block - tile * p.stages;
  const uint32_t column = tile * kTile + row, term = stage * kTerms + part * 8u;
  raw v[8];
  if (ALONG && column < p.columns && term + 8u <= p.terms) {
    const typename Pack<T, 8>::type got = *reinterpret_cast<const typename Pack<T, 8>::type *>(static_cast<const raw *>(p.from) + static_cast<uint64_t>(column) * p.stride + term);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = got[k];
  } else {
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k) {
    const uint64_t at = ALONG ? static_cast<uint64_t>(column) * p.stride + term + k : static_cast<uint64_t>(term + k) * p.stride + column;
    v[k] = column < p.columns && term + k < p.terms ? static_cast<const raw *>(p.from)[at] : static_cast<raw>(0);
  }
  }
  u32x4 w[3];
  if constexpr (P == 2) {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = ValueOf<T>::get(v[k]);
    split8(f, w);
  } else {
    split8(v, w);
  }
#pragma unroll
  for (int c = 0; c < P; ++c) *reinterpret_cast<u32x4 *>(p.to + (static_cast<uint64_t>(block) * P + c) * kPlane + tile_at(row, part)) = w[c];
}

typedef __attribute__((address_space(3))) void *LdsPointer;
// 16 bytes a lane to 1,024 consecutive bytes of LDS.
__device__ __forceinline__ void load_to_lds(const uint16_t *from, uint16_t *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (LdsPointer)to, 16, 0, 0);
}
// Waits for the wavefront's loads and LDS accesses, then for the block.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The block has read what it wanted from LDS, and the compiler moves no access past that; loads that are on their way stay so.
__device__ __forceinline__ void block_has_read() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// What a wavefront's 16 * MR rows by 128 columns of sums become.  Through LDS (`mine`, 4 KB), 16 rows by 64 columns at a time, a lane's columns
// become lines (part c of row r at c ^ r).  sums: of the columns, kept over tiles.
template <typename A, typename T, int USE, int MR, bool MASKED>
__device__ __forceinline__ void finish_tile(const DenseArgs &p, uint32_t step, f32x4 (&acc)[MR][8], f32x4 *mine, uint64_t first_row, uint32_t column0,
                                            const float (&bias)[2][4], float (&sums)[2][4]) {
  const uint32_t lane = threadIdx.x & (kWave - 1), r = lane & 15u, part = lane >> 4;
#pragma unroll
  for (int i = 0; i < MR; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 4; ++j) mine[r * 16u + ((j * 4u + part) ^ r)] = acc[i][h * 4 + j];
      __builtin_amdgcn_wave_barrier();
      const uint32_t c = column0 + h * 64u + (lane & 15u) * 4u;
      const uint64_t row0 = first_row + i * 16u + lane / 16u;
      // two rows of a lane at a time, the next ones' second operand on its way; not unrolled, or the registers do not hold what is behind it
      float ahead[2][4] = {};
      auto read = [&](uint32_t q) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u)
          if (USE != kRows && p.more && row0 + (q + u) * 4u < p.M && c < p.N)
            get_columns(static_cast<const T *>(p.more) + (row0 + (q + u) * 4u) * p.N + c, p.N - c, ahead[u]);
      };
      read(0);
      // nothing for 64 columns that are not there: a step of 183,672 rows of 39 by 22 in bf16 takes 134 us and some 20 more with them
      const uint32_t turns = column0 + h * 64u < p.N ? 4u : 0u;
#pragma unroll 1
      for (uint32_t q = 0; q < turns; q += 2) {
        float v[2][4], more[2][4];
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
          const uint32_t row = (q + u) * 4u + lane / 16u;
          const uint64_t at = row0 + (q + u) * 4u;
          const f32x4 got = mine[row * 16u + ((lane & 15u) ^ row)];
          v[u][0] = got.x, v[u][1] = got.y, v[u][2] = got.z, v[u][3] = got.w;
#pragma unroll
          for (int k = 0; k < 4; ++k) more[u][k] = ahead[u][k];
          if (sizeof(A) == 4) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
              if (fabsf(v[u][k]) < INFINITY || at >= p.M || c + k >= p.N) continue;
              const T *const b = static_cast<const T *>(p.w);
              v[u][k] = sum_of_terms(static_cast<const float *>(p.a) + at * p.a_stride,
                                     MASKED ? static_cast<const float *>(p.y) + at * p.a_stride : nullptr, p.mask_scale, 1,
                                     USE == kRows ? b + c + k : b + static_cast<uint64_t>(c + k) * p.K, USE == kRows ? p.N : 1u, p.K);
            }
          }
          if (USE != kRows) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[u][k] += bias[h][k];
          }
          if (USE == kLayer) activate<T, 4>(v[u], p.act);
        }
        if (q == 0) read(2);
        if (USE != kRows && p.drop.threshold) {
          float(*const dropping)[4] = USE == kLayer ? v : more;
          drop_two_rows(p.drop, step, static_cast<uint32_t>(row0) + q * 4u, static_cast<uint32_t>(row0) + q * 4u + 4u, c, dropping[0], dropping[1]);
        }
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
          const uint64_t at = row0 + (q + u) * 4u;
          if (USE == kLayer && p.more) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[u][k] += more[u][k];
          }
          if (USE == kSlope) through_slope<T>(v[u], more[u], p.act);
          if (at >= p.M || c >= p.N) continue;
          if (USE == kSlope) {
            put_columns(static_cast<float *>(p.out) + at * p.N + c, p.N - c, v[u], p.streamed);
          } else {
            if (USE == kRows && sizeof(A) == 2) {
#pragma unroll
              for (int k = 0; k < 4; ++k) v[u][k] *= p.after;
            }
            put_columns(static_cast<T *>(p.out) + at * p.N + c, p.N - c, v[u], p.streamed);
          }
          if (USE == kSlope) {  // columns that are not there are summed and not stored
#pragma unroll
            for (int k = 0; k < 4; ++k) sums[h][k] += v[u][k];
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
}

template <typename T>
__device__ __forceinline__ void bias_of_columns(const DenseArgs &p, uint32_t column0, float (&bias)[2][4]) {
  if (!p.bias) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t c = column0 + h * 64u + (threadIdx.x & 15u) * 4u;
    if (c < p.N) get_columns(static_cast<const T *>(p.bias) + c, p.N - c, bias[h]);
  }
}
// The block's column sums to row `to` of p.sums: of a wavefront's four rows of lanes, then of the ROWS wavefronts of rows of each group of 128
// columns.
template <int WAVES, int ROWS>
__device__ __forceinline__ void block_sums(const DenseArgs &p, const float (&sums)[2][4], float (*of_wave)[kTile], uint32_t to, uint32_t column0) {
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = wave_of_block();
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float v = sums[h][k];
      v += __shfl_xor(v, 16, kWave);
      v += __shfl_xor(v, 32, kWave);
      if (lane < 16u) of_wave[wave][h * 64u + lane * 4u + k] = v;
    }
  __syncthreads();
  if (t < kTile * (WAVES / ROWS)) {
    const uint32_t group = t / kTile, c = column0 + t;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < ROWS; ++w) v += of_wave[group * ROWS + w][t % kTile];
    if (c < p.N) p.sums[static_cast<uint64_t>(to) * p.N + c] = v;
  }
}

// Many rows.  A block of four wavefronts takes 64 * MR rows by 128 columns, a stage of 32 terms after the other, and then its next rows.  Rows
// go from memory to the registers that the matrix instructions read, each to the one wavefront that needs them, and are split there; the
// prepared weight goes to LDS by loads that write it themselves.  Both are a stage ahead, past the end of a tile too.
// MR: 16 rows each, of a wavefront.
// 232,965 rows of 602 by 256 in 32 bits take 440-500 us, 72 GFLOP at 145-160 TFLOP/s, as the library's product of such size (152): six matrix
// instructions a product, which are under way for half of the time, and the splitting for most of the other half; the clock falls to 1.8 GHz
// (splitting one tile between the instructions of the other, or three blocks to a compute unit, which spill, did not help).  169,343 rows of
// 128 by 128 in bf16 with GELU, drops and residual take 56 us, 2.4 TB/s: vector instructions of the epilogue for half of the time.
// A: the rows' type.
template <typename A, typename T, int USE, int MR, bool MASKED>
__device__ __forceinline__ void rows_of_tiles(DenseArgs p) {
  constexpr int P = kPlanes<A>, PB = kPlanesBeside<A, T>;
  constexpr uint32_t kTileRows = 64 * MR, kStage = PB * kPlane;
  // results are turned where the stage of the weight was that has been used last, if it is large enough
  constexpr bool kApart = kStage * sizeof(uint16_t) < 4u * 4096u;
  __shared__ __attribute__((aligned(16))) uint16_t weight0[kStage], weight1[kStage], apart[kApart ? 4 * 2048 : 8];
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = wave_of_block(), r = lane & 15u, part = lane >> 4;
  // neighbouring blocks of a chiplet take the columns of one worker's rows
  const uint32_t x = blockIdx.x / 8u, tn = x % p.tiles_n, worker = x / p.tiles_n * 8u + blockIdx.x % 8u;
  const uint32_t stages = (p.K + kTerms - 1u) / kTerms;
  const uint32_t step = USE == kLayer || USE == kSlope ? drop_step(p.drop) : 0u;
  if (USE == kLayer && p.drop.step_kept && blockIdx.x == 0 && t == 0) *p.drop.step_kept = step;
  if (!has_rows(worker, p.workers)) return;
  const uint16_t *const weight = static_cast<const uint16_t *>(p.b) + static_cast<uint64_t>(tn) * stages * PB * kPlane;
  const A *const rows = static_cast<const A *>(p.a);
  // stage s of the weight
  auto request_weight = [&](uint16_t *to, uint32_t s) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < 2 * PB; ++i) {
      const uint32_t piece = i * 4 + wave;  // 512 values each
      load_to_lds(weight + (static_cast<uint64_t>(s) * PB * kPlane + piece * 512u + lane * 8u), to + piece * 512u);
    }
  };
  typedef typename ValueOf<A>::raw raw;
  constexpr int L = 8 * sizeof(raw) / 16;  // loads of a lane's eight terms
  constexpr int S = MASKED ? 2 : 1;  // operands: g and y
  u32x4 next[S][MR][L];
  const A *row_at[S][MR];
  auto place = [&](uint32_t tile) __attribute__((always_inline)) {  // rows that the result does not have read the last one
#pragma unroll
    for (int i = 0; i < MR; ++i) {
      const uint64_t row = static_cast<uint64_t>(tile) * kTileRows + wave * (16u * MR) + i * 16u + r;
#pragma unroll
      for (int o = 0; o < S; ++o)
        row_at[o][i] = (o ? static_cast<const A *>(p.y) : rows) + min(row, static_cast<uint64_t>(p.M - 1u)) * p.a_stride + part * 8u;
    }
  };
  auto request_rows = [&](uint32_t s) __attribute__((always_inline)) {
    typedef typename Pack<A, 16 / sizeof(raw)>::type Whole;
    const uint32_t k = s * kTerms;
    if (k + kTerms <= p.K) {
#pragma unroll
      for (int o = 0; o < S; ++o)
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int l = 0; l < L; ++l) {
            const Whole got = *reinterpret_cast<const Whole *>(row_at[o][i] + k + l * (16 / sizeof(raw)));
            next[o][i][l] = __builtin_bit_cast(u32x4, got);
          }
    } else {
      const uint32_t from = k + part * 8u, count = from < p.K ? min(p.K - from, 8u) : 0u;
#pragma unroll
      for (int o = 0; o < S; ++o)
#pragma unroll
        for (int i = 0; i < MR; ++i) {
          raw v[8];
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e) v[e] = e < count ? reinterpret_cast<const raw *>(row_at[o][i] + k)[e] : static_cast<raw>(0);
          if (sizeof(raw) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) next[o][i][e / 4 % L][e % 4] = __float_as_uint(v[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) next[o][i][0][e] = static_cast<uint32_t>(v[2 * e]) | static_cast<uint32_t>(v[2 * e + 1]) << 16;
          }
        }
    }
  };
  // value e of the eight of fragment i
  auto value = [&](int o, int i, int e) __attribute__((always_inline)) {
    if (sizeof(raw) == 4) {
      const uint32_t bits = next[o][i][e / 4 % L][e % 4];
      return __uint_as_float(bits);
    }
    const uint32_t both = next[o][i][0][e / 2 % 4];
    return ValueOf<A>::get(static_cast<raw>(e & 1 ? both >> 16 : both));
  };
  f32x4 acc[MR][8];
  uint32_t half = 0;
  float bias[2][4] = {};
  if (USE != kRows) bias_of_columns<T>(p, tn * kTile, bias);
  float sums[2][4] = {};
  place(worker);
  request_weight(weight0, 0);
  request_rows(0);
  for (uint32_t tile = worker; tile < p.tiles_m; tile += p.workers) {
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    for (uint32_t s = 0; s < stages; ++s) {
      u32x4 a[MR][P];
      stage_barrier();
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        if (P == 3 || MASKED) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = value(0, i, e);
            if (MASKED) v[e] = value(S - 1, i, e) <= 0.0f ? 0.0f : P == 3 ? v[e] * p.mask_scale : v[e];
          }
          if constexpr (P == 3) {
            split8(v, a[i]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) a[i][0][e] = ValueOf<A>::put(v[2 * e]) | static_cast<uint32_t>(ValueOf<A>::put(v[2 * e + 1])) << 16;
          }
        } else {
          a[i][0] = next[0][i][0];
        }
      }
      const bool last = s + 1u == stages;
      if (!last || tile + p.workers < p.tiles_m) {
        if (last) place(tile + p.workers);
        request_weight(half ? weight0 : weight1, last ? 0u : s + 1u);
        request_rows(last ? 0u : s + 1u);
      }
      const uint16_t *const w = half ? weight1 : weight0;
      half ^= 1u;
      u32x4 b[2][PB];
#pragma unroll
      for (int c = 0; c < PB; ++c) b[0][c] = *reinterpret_cast<const u32x4 *>(w + c * kPlane + tile_at(r, part));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < 7) {
#pragma unroll
          for (int c = 0; c < PB; ++c) b[(j + 1) & 1][c] = *reinterpret_cast<const u32x4 *>(w + c * kPlane + tile_at((j + 1) * 16 + r, part));
        }
        // the weight is the first operand: a lane then ends up with four neighbouring columns of one row; small products first
#pragma unroll
        for (int q = P - 1; q >= 0; --q)
#pragma unroll
          for (int c = q >= PB ? q - PB + 1 : 0; c <= q; ++c)
#pragma unroll
            for (int i = 0; i < MR; ++i) acc[i][j] = multiply<A>(b[j & 1][q - c], a[i][c], acc[i][j]);
      }
    }
    if (!kApart) block_has_read();
    finish_tile<A, T, USE, MR, MASKED>(p, step, acc, reinterpret_cast<f32x4 *>(kApart ? apart : half ? weight0 : weight1) + wave * 256u,
                                    static_cast<uint64_t>(tile) * kTileRows + wave * (16u * MR), tn * kTile, bias, sums);
  }
  if (USE == kSlope && p.sums) block_sums<4, 4>(p, sums, reinterpret_cast<float(*)[kTile]>(kApart ? apart : weight0), worker, tn * kTile);
}
template <typename T, int USE, int MR, bool MASKED>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) void dense_rows_kernel(DenseArgs p) {
  rows_of_tiles<T, T, USE, MR, MASKED>(p);
}
// Rows of dz in 32 bits times a weight of 16.  169,343 rows of 128 by 128: 34 us in bf16, 3.8 TB/s, as with two bf16 parts of dz, whose products
// read the weight twice from LDS; 49 in fp16.  Large products go this way, too: 65,536 x 4,096 x 4,096 in bf16 5.7 ms, three products at
// 1,160 TFLOP/s, where large tiles took 3.5 for two parts; in fp16 8.9.
template <typename T>
__global__ __launch_bounds__(256, 2) void dense_dz_kernel(DenseArgs p) {
  rows_of_tiles<float, T, kRows, 2, false>(p);
}

// Large products of 16-bit values whose rows begin at multiples of 16 bytes: a block of eight wavefronts takes 256 rows by 256 columns, 32
// terms at a time, which loads write to LDS themselves, three stages ahead of the one that is multiplied.  Both operands lie as they do in
// memory: b's row j holds column j's terms; in LDS as tile_at says.  65,536 rows of 4,096 by 4,096 with GELU, drops and a residual take 2,110
// us, 1,040 TF/s.  LDS bounds it: a stage's 96 reads and 32 KB of writes hold it for 1,024 cycles, as long as the matrix instructions take.
// (Four wavefronts of 128 by 128 read a third less, but their 256 sums leave too few registers: 3,170 us, moves between the two halves of the
// register file; all wavefronts in step: 2,510; dense_rows_kernel: 2,830.)
constexpr uint32_t kWideStages = 4;
__device__ __attribute__((aligned(16))) uint16_t zero_part[8];
template <typename T, int USE>
__global__ __launch_bounds__(512, 2) void dense_wide_kernel(DenseArgs p) {
  constexpr uint32_t kOperand = kWideTile * kTerms;
  __shared__ __attribute__((aligned(16))) uint16_t stages[kWideStages][2 * kOperand];
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = wave_of_block(), r = lane & 15u, part = lane >> 4;
  uint32_t tm, tn;
  tile_of(p.tiles_n, p.tiles_m >= kXcdTiles, 8, &tm, &tn);
  if (tm >= p.tiles_m) return;
  const uint32_t step = USE == kRows ? 0u : drop_step(p.drop);
  if (USE == kLayer && p.drop.step_kept && blockIdx.x == 0 && t == 0) *p.drop.step_kept = step;
  // A load takes 16 rows' 64 bytes, and a wavefront every eighth of the 32 loads of a stage.  Rows that are not there read the last one.
  const uint64_t row_a = static_cast<uint64_t>(tm) * kWideTile, row_b = static_cast<uint64_t>(tn) * kWideTile;
  const char *const from_a = reinterpret_cast<const char *>(static_cast<const uint16_t *>(p.a) + row_a * p.a_stride);
  const char *const from_b = reinterpret_cast<const char *>(static_cast<const uint16_t *>(p.b) + row_b * p.b_stride);
  const uint32_t chunk = part_at(lane / 4u, lane & 3u);  // the same for all of the lane's rows, which are 16 apart
  uint32_t at[4];  // in bytes: below 2^26, as 256 rows of 2^17 values are
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t row = ((i & 1) * 8u + wave) * 16u + lane / 4u;
    at[i] = (i < 2 ? static_cast<uint32_t>(min(static_cast<uint64_t>(row), p.M - 1u - row_a)) * p.a_stride
                   : static_cast<uint32_t>(min(static_cast<uint64_t>(row), p.N - 1u - row_b)) * p.b_stride) * 2u + chunk * 16u;
  }
  auto request = [&](uint16_t *to, uint32_t k) __attribute__((always_inline)) {
    const char *const a = from_a + k * 2ull, *const b = from_b + k * 2ull;
    if (k + kTerms <= p.K) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_to_lds(reinterpret_cast<const uint16_t *>((i < 2 ? a : b) + at[i]), to + (i * 8u + wave) * 512u);
      return;
    }
    const bool inside = k + chunk * 8u < p.K;  // whole parts: rows are of multiples of eight
#pragma unroll
    for (int i = 0; i < 4; ++i)
      load_to_lds(inside ? reinterpret_cast<const uint16_t *>((i < 2 ? a : b) + at[i]) : zero_part, to + (i * 8u + wave) * 512u);
  };
  const uint32_t wr = wave & 3u, wc = wave >> 2;
  f32x4 acc[4][8] = {};
  u32x4 rows[4], columns[8];
#pragma unroll
  for (uint32_t s = 0; s < kWideStages - 1; ++s) request(stages[s], s * kTerms);
  // Two wavefronts share a SIMD, and while one multiplies the other reads LDS: those of the upper columns are half a stage behind.  A stage
  // is read by the lower ones in slot 2s and by the upper ones in slot 2s + 1, so its loads are waited for in the slots before, and its place
  // is written again three stages on.
  auto slot_ends = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // All LDS reads are done, and of the wavefront's loads all but those of two stages, eight.
  auto stage_comes = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0078);
  };
  stage_comes();
  if (wc) slot_ends();
  // Whole turns, so that the stages' places are constants; stages behind the last term are zeros that no memory is read for.
  for (uint32_t k = 0; k < p.K; k += kWideStages * kTerms) {
#pragma unroll
    for (uint32_t s = 0; s < kWideStages; ++s) {
      slot_ends();
      request(stages[(s + kWideStages - 1) % kWideStages], k + (s + kWideStages - 1) * kTerms);
#pragma unroll
      for (int i = 0; i < 4; ++i) rows[i] = *reinterpret_cast<const u32x4 *>(stages[s] + tile_at(wr * 64u + i * 16u + r, part));
#pragma unroll
      for (int j = 0; j < 8; ++j) columns[j] = *reinterpret_cast<const u32x4 *>(stages[s] + kOperand + wc * kPlane + tile_at(j * 16u + r, part));
      stage_comes();
      slot_ends();
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i][j] = multiply<T>(columns[j], rows[i], acc[i][j]);
    }
  }
  if (!wc) slot_ends();
  stage_barrier();  // no load may reach the LDS any more
  float bias[2][4] = {}, sums[2][4] = {};
  if (USE != kRows) bias_of_columns<T>(p, tn * kWideTile + wc * kTile, bias);
  finish_tile<T, T, USE, 4, false>(p, step, acc, reinterpret_cast<f32x4 *>(&stages[0][0]) + wave * 256u, static_cast<uint64_t>(tm) * kWideTile + wr * 64u,
                                tn * kWideTile + wc * kTile, bias, sums);
  if (USE == kSlope && p.sums) block_sums<8, 4>(p, sums, reinterpret_cast<float(*)[kTile]>(&stages[2][0]), tm, tn * kWideTile);
}
// The weight with rows and columns exchanged.
__global__ __launch_bounds__(256) void dense_turn_kernel(uint16_t *__restrict__ to, const uint16_t *__restrict__ from, uint32_t rows, uint32_t columns) {
  __shared__ uint16_t tile[64][66];
  const uint32_t x = threadIdx.x % 64u, y = threadIdx.x / 64u, c0 = blockIdx.x * 64u, r0 = blockIdx.y * 64u;
  for (uint32_t i = y; i < 64u; i += 4u) tile[i][x] = r0 + i < rows && c0 + x < columns ? from[static_cast<uint64_t>(r0 + i) * columns + c0 + x] : uint16_t{0};
  __syncthreads();
  for (uint32_t i = y; i < 64u; i += 4u)
    if (c0 + i < columns && r0 + x < rows) to[static_cast<uint64_t>(c0 + i) * rows + r0 + x] = tile[x][i];
}

// ---- the weight's gradient --------------------------------------------------------------------------
// Few results and many terms: blockIdx.z takes its part of the terms, the parts' sums are added in order by a second launch, so results do
// not depend on scheduling.  A block of four wavefronts takes 128 rows of the result by 128 columns, 32 terms at a time through LDS, where
// both operands are written with the terms of a row or column side by side.
// 232,965 terms of 256 by 602 in 32 bits: 500-550 us, 130-143 TFLOP/s, splitting half of the time and matrix instructions for two fifths;
// 169,343 of 128 by 128 in bf16: 19 us, 4.5 TB/s, and 33 with dz in 32 bits, three matrix instructions a product and the splitting; in
// fp16, with five, 38.
// Sixteen terms of one column of an operand, or eight of each of two neighbouring columns (PAIRS: rows of 16-bit values of an even number),
// on their way from memory to LDS, as P parts in planes of their own.  MASKED: as DenseArgs' y.
template <typename T, bool PAIRS, bool MASKED, int P>
struct Terms {
  typedef typename ValueOf<T>::raw raw;
  static constexpr int S = MASKED ? 2 : 1, N = PAIRS ? 8 : 16;
  typedef uint32_t Word __attribute__((aligned(2)));
  uint32_t v[S][N];
  const T *from[S];  // the operands' beginning, so that a row's address is a scalar, and the lane's place from there
  uint32_t lane_at, stride, column, first;  // the thread's column of 128, its first term of 32
  __device__ __forceinline__ void place(const void *a, const void *second, uint32_t row_stride, uint32_t first_column, uint32_t columns) {
    const uint32_t t = threadIdx.x;
    column = PAIRS ? t % 64u * 2u : t & 127u;
    first = PAIRS ? t / 64u * 8u : (t >> 7) * 16u;
    stride = row_stride;
    // neighbouring threads have neighbouring columns; columns that the operand does not have read some other of it
    const uint32_t c = min(first_column + column, columns - (PAIRS ? 2u : 1u));
    lane_at = first * stride + c;
    from[0] = static_cast<const T *>(a);
    if (S == 2) from[S - 1] = static_cast<const T *>(second);
  }
  template <bool SOME>
  __device__ __forceinline__ void request(uint64_t term, uint32_t left) {
#pragma unroll
    for (int o = 0; o < S; ++o) {
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        const T *const one = from[o] + (term + i) * stride + lane_at;
        if (SOME && first + i >= left) v[o][i] = 0u;
        else if (PAIRS) v[o][i] = *reinterpret_cast<const Word *>(one);
        else if (sizeof(raw) == 4) v[o][i] = *reinterpret_cast<const uint32_t *>(one);
        else v[o][i] = static_cast<uint32_t>(*reinterpret_cast<const raw *>(one));
      }
    }
  }
  // Term i of the thread's column, or of the second one of a pair.
  __device__ __forceinline__ float value(int i, int which) const {
    auto get = [&](uint32_t word) { return sizeof(raw) == 4 ? __uint_as_float(word) : ValueOf<T>::get(static_cast<raw>(which ? word >> 16 : word)); };
    const float x = get(v[0][i]);
    return !MASKED ? x : get(v[S - 1][i]) <= 0.0f ? 0.0f : x;
  }
  // To the planes; sums: of the columns' terms, times scale.
  __device__ __forceinline__ void keep(uint16_t *planes, float scale, float *sums) const {
#pragma unroll
    for (int which = 0; which < (PAIRS ? 2 : 1); ++which)
#pragma unroll
      for (int i = 0; i < N; i += 8) {
        u32x4 w[3];
        if (sizeof(raw) == 4 || MASKED || P == 2) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = value(i + e, which) * (MASKED && P == 3 ? scale : 1.0f);
            if (sums) sums[which] += MASKED && P == 1 ? f[e] * scale : f[e];
          }
          if constexpr (P > 1) {
            split8(f, w);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[0][e] = ValueOf<T>::put(f[2 * e]) | static_cast<uint32_t>(ValueOf<T>::put(f[2 * e + 1])) << 16;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = v[0][i + 2 * e], y = v[0][i + 2 * e + 1];
            w[0][e] = which ? __builtin_amdgcn_perm(y, x, 0x07060302u) : __builtin_amdgcn_perm(y, x, 0x05040100u);
          }
          if (sums) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[which] += value(i + e, which);
          }
        }
#pragma unroll
        for (int c = 0; c < P; ++c) *reinterpret_cast<u32x4 *>(planes + c * kPlane + tile_at(column + which, (first + i) / 8u)) = w[c];
      }
  }
};

// SOURCE, the first operand: g or dz as it is, g by y, dz in 32 bits beside operands of 16.
enum Source { kPlain, kMasked, kInWords };
template <typename T, bool PAIRS, int SOURCE>
__global__ __launch_bounds__(256, 2) void dense_weight_kernel(DenseArgs p) {
  typedef typename std::conditional<SOURCE == kInWords, float, T>::type A;
  constexpr bool MASKED = SOURCE == kMasked;
  constexpr int PA = kPlanes<A>, P = kPlanesBeside<A, T>;
  typedef Terms<A, PAIRS && sizeof(A) == 2, MASKED, PA> First;
  __shared__ __attribute__((aligned(16))) uint16_t tile[(PA + P) * kPlane];
  uint16_t *const ta = tile, *const tb = tile + PA * kPlane;
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = wave_of_block(), r = lane & 15u, part = lane >> 4;
  const uint32_t tm = blockIdx.x / p.tiles_n, tn = blockIdx.x % p.tiles_n;
  const uint32_t m0 = tm * kTile, n0 = tn * kTile;
  const uint64_t begin = static_cast<uint64_t>(blockIdx.z) * p.part_terms, end = min(static_cast<uint64_t>(p.K), begin + p.part_terms);
  First va;
  Terms<T, PAIRS, false, P> vb;
  va.place(p.a, p.y, p.a_stride, m0, p.M);
  vb.place(p.b, nullptr, p.b_stride, n0, p.N);
  float sums[2] = {};
  const bool summing = p.column_sums && tn == 0;
  auto request = [&](uint64_t k) __attribute__((always_inline)) {
    if (k + kTerms <= end) {
      va.template request<false>(k, 0u);
      vb.template request<false>(k, 0u);
    } else {
      const uint32_t left = k < end ? static_cast<uint32_t>(end - k) : 0u;
      va.template request<true>(k, left);
      vb.template request<true>(k, left);
    }
  };
  const uint32_t wm = wave / 2u * 64u, wn = wave % 2u * 64u;
  f32x4 acc[4][4] = {};
  request(begin);
  for (uint64_t k = begin; k < end; k += kTerms) {
    if (summing) va.keep(ta, p.mask_scale, sums);
    else va.keep(ta, p.mask_scale, nullptr);
    vb.keep(tb, 1.0f, nullptr);
    __syncthreads();
    if (k + kTerms < end) request(k + kTerms);
    u32x4 b[P][4];
#pragma unroll
    for (int c = 0; c < P; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) b[c][j] = *reinterpret_cast<const u32x4 *>(tb + c * kPlane + tile_at(wn + j * 16 + r, part));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 a[PA];
#pragma unroll
      for (int c = 0; c < PA; ++c) a[c] = *reinterpret_cast<const u32x4 *>(ta + c * kPlane + tile_at(wm + i * 16 + r, part));
#pragma unroll
      for (int s = PA - 1; s >= 0; --s)
#pragma unroll
        for (int c = s >= P ? s - P + 1 : 0; c <= s; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = multiply<A>(b[s - c][j], a[c], acc[i][j]);
    }
    __syncthreads();
  }
  // as the rows' kernel: lines of 64 columns
  f32x4 *const mine = reinterpret_cast<f32x4 *>(tile) + wave * 256u;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[r * 16u + ((j * 4u + part) ^ r)] = acc[m][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
      const uint32_t row = q * 4u + lane / 16u, c = n0 + wn + (lane & 15u) * 4u, i = m0 + wm + m * 16u + row;
      const f32x4 got = mine[row * 16u + ((lane & 15u) ^ row)];
      if (i >= p.M || c >= p.N) continue;
      float v[4] = {got.x, got.y, got.z, got.w};
      if (sizeof(A) == 4) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          if (fabsf(v[k]) < INFINITY || c + k >= p.N) continue;
          v[k] = sum_of_terms(static_cast<const float *>(p.a) + begin * p.a_stride + i, MASKED ? static_cast<const float *>(p.y) + begin * p.a_stride + i : nullptr,
                              p.mask_scale, p.a_stride, static_cast<const T *>(p.b) + begin * p.b_stride + c + k, p.b_stride, end - begin);
        }
      }
      if (sizeof(A) == 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] *= p.after;
      }
      if (p.sums) put_columns(p.sums + (static_cast<uint64_t>(blockIdx.z) * p.M + i) * p.N + c, p.N - c, v, false);
      else put_columns(static_cast<T *>(p.out) + static_cast<uint64_t>(i) * p.N + c, p.N - c, v, false);
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (!summing) return;
  __syncthreads();
  float(*const of_terms)[kTile] = reinterpret_cast<float(*)[kTile]>(tile);
  of_terms[va.first / First::N][va.column] = sums[0];
  if (First::N == 8) of_terms[va.first / 8u][va.column + 1u] = sums[1];
  __syncthreads();
  if (t < kTile && m0 + t < p.M) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < (First::N == 8 ? 4 : 2); ++i) sum += of_terms[i][t];
    p.column_sums[static_cast<uint64_t>(blockIdx.z) * p.M + m0 + t] = sum;
  }
}

// ---- few rows ---------------------------------------------------------------------------------------
// A prediction for some vertices: the weight is what has to be read, once.  A wavefront takes a column of the result for R rows; its
// lanes take 8 terms each at a time, in 32 bits.  One row of 602 by 256: 3.1-3.6 us, most of which a launch takes; on tiles of rows 9.
constexpr uint32_t kFewRows = 8, kFewWaves = 4;
template <typename T, int R>
__global__ __launch_bounds__(kFewWaves *kWave) void dense_few_kernel(DenseArgs p) {
  const uint32_t lane = threadIdx.x & (kWave - 1), c = blockIdx.x * kFewWaves + wave_of_block();
  const uint64_t i0 = static_cast<uint64_t>(blockIdx.y) * R, last = p.M - 1u;
  const uint32_t step = drop_step(p.drop);
  if (p.drop.step_kept && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.drop.step_kept = step;
  if (c >= p.N) return;
  const T *const x = static_cast<const T *>(p.a), *const w = static_cast<const T *>(p.w) + static_cast<uint64_t>(c) * p.K;
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
  activate<T, 1>(&v, p.act);
  if (p.drop.threshold) {
    const uint4 n = row_numbers(p.drop, step, static_cast<uint32_t>(i), c >> 3);
    const uint32_t word = c & 4u ? (c & 2u ? n.w : n.z) : (c & 2u ? n.y : n.x);
    v = (c & 1u ? word >> 16 : word & 0xFFFFu) >= p.drop.threshold ? v * p.drop.scale : 0.0f;
  }
  if (p.more) v += get_value(static_cast<const T *>(p.more) + i * p.N + c);
  put_value(static_cast<T *>(p.out) + i * p.N + c, v);
}

// ---- sums -------------------------------------------------------------------------------------------
// The gradient of y where no sums are needed: dropped, or by y as DenseArgs say (if out is not null), and summed by columns.  A lane has four
// columns, a wavefront four rows of 64; a block takes every gridDim.y-th group of 32 rows.  232,965 rows of 256 by y: 130 us, 5.5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void dense_columns_kernel(DenseArgs p) {
  __shared__ float of_wave[4][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block(), c = blockIdx.x * kWave + (lane & 15u) * 4u;
  const uint32_t step = drop_step(p.drop), count = c < p.N ? p.N - c : 0u;
  float sums[4] = {};
  // 16-bit values are stored as they are, and their sums scaled
  const float scale = p.y ? p.mask_scale : p.drop.scale, inside = kPlanes<T> == 3 ? scale : 1.0f, outside = kPlanes<T> == 3 ? 1.0f : scale;
  DropArgs drop = p.drop;
  drop.scale = inside;
  for (uint64_t i0 = blockIdx.y * 32ull + wave * 8u + lane / 16u; i0 < p.M; i0 += gridDim.y * 32ull) {
    float v[2][4] = {}, y[2][4] = {};
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      if (i0 + u * 4u >= p.M || !count) continue;
      get_columns(static_cast<const T *>(p.more) + (i0 + u * 4u) * p.N + c, count, v[u]);
      if (p.y) get_columns(static_cast<const T *>(p.y) + (i0 + u * 4u) * p.N + c, count, y[u]);
    }
    if (p.y) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[u][k] = y[u][k] <= 0.0f ? 0.0f : v[u][k] * inside;
    } else if (p.drop.threshold) {
      drop_two_rows(drop, step, static_cast<uint32_t>(i0), static_cast<uint32_t>(i0) + 4u, c, v[0], v[1]);
    }
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      if (i0 + u * 4u >= p.M || !count) continue;
      if (p.out) put_columns(static_cast<T *>(p.out) + (i0 + u * 4u) * p.N + c, count, v[u], false);
#pragma unroll
      for (int k = 0; k < 4; ++k) sums[k] += v[u][k];
    }
  }
  if (!p.sums) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    sums[k] *= outside;
    sums[k] += __shfl_xor(sums[k], 16, kWave);
    sums[k] += __shfl_xor(sums[k], 32, kWave);
    if (lane < 16u) of_wave[wave][lane * 4u + k] = sums[k];
  }
  __syncthreads();
  const uint32_t column = blockIdx.x * kWave + threadIdx.x;
  if (threadIdx.x < kWave && column < p.N)
    p.sums[static_cast<uint64_t>(blockIdx.y) * p.N + column] = (of_wave[0][threadIdx.x] + of_wave[1][threadIdx.x]) + (of_wave[2][threadIdx.x] + of_wave[3][threadIdx.x]);
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

template <bool ALONG>
int launch_prepare(void *to, const void *w, int type, uint32_t planes, uint32_t columns, uint32_t terms, uint32_t stride, hipStream_t stream) {
  const PrepareArgs p{w, static_cast<uint16_t *>(to), columns, terms, stride, ceil_div(terms, kTerms), ceil_div(columns, kTile)};
  const dim3 grid(ceil_div(prepare_threads(columns, terms), 256));
  if (type == NTS_F32) hipLaunchKernelGGL((dense_prepare_kernel<float, 3, ALONG>), grid, dim3(256), 0, stream, p);
  else if (!ALONG && planes == 2) hipLaunchKernelGGL((dense_prepare_kernel<F16, 2, false>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((dense_prepare_kernel<Bf16, 1, ALONG>), grid, dim3(256), 0, stream, p);  // the bits of both 16-bit types are copied
  NTS_LAUNCH_CHECK("dense_prepare_kernel");
  return NTS_OK;
}

template <typename T, int USE, bool MASKED = false>
void launch_rows(const DenseArgs &p, const Share &share, hipStream_t stream) {
  hipLaunchKernelGGL((dense_rows_kernel<T, USE, 2, MASKED>), dim3(launched_workers(share) * p.tiles_n), dim3(256), 0, stream, p);
}
template <typename T, int USE>
void launch_product_of(const DenseArgs &p, const Share &share, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (share.wide) {
      hipLaunchKernelGGL((dense_wide_kernel<T, USE>), dim3(tile_blocks(p.tiles_m, p.tiles_n, 8)), dim3(512), 0, stream, p);
      return;
    }
  }
  if constexpr (USE == kRows && sizeof(T) == 2) {
    if (p.dz32) {
      hipLaunchKernelGGL((dense_dz_kernel<T>), dim3(launched_workers(share) * p.tiles_n), dim3(256), 0, stream, p);
      return;
    }
  }
  if constexpr (USE == kRows) {
    if (p.y) return launch_rows<T, USE, true>(p, share, stream);
  }
  launch_rows<T, USE>(p, share, stream);
}
template <int USE>
Share share_for(const DenseArgs &p, int type) {
  return share_of(type, p.M, p.N, p.K, !p.y && !p.dz32 && aligned_to(p.a, 16) && (USE == kRows || aligned_to(p.w, 16)));
}
// The product of p.a and the weight p.w, whose form for it goes to `work`.
template <int USE>
int launch_product(DenseArgs p, int type, void *work, hipStream_t stream) {
  const Share share = share_for<USE>(p, type);
  p.tiles_m = share.tiles_m, p.tiles_n = share.tiles_n, p.workers = share.workers;
  p.streamed = static_cast<uint64_t>(p.M) * p.N * (USE == kSlope ? sizeof(float) : type_size(type)) >= kStreamed;
  p.b = work;
  if (!share.wide) {
    const uint32_t planes = planes_of(type, p.dz32);
    const int status = USE == kRows ? launch_prepare<false>(work, p.w, type, planes, p.N, p.K, p.N, stream)
                                    : launch_prepare<true>(work, p.w, type, planes, p.N, p.K, p.K, stream);
    if (status) return status;
  } else if (USE == kRows) {
    p.b_stride = p.K;
    hipLaunchKernelGGL(dense_turn_kernel, dim3(ceil_div(p.N, 64), ceil_div(p.K, 64)), dim3(256), 0, stream, static_cast<uint16_t *>(work),
                       static_cast<const uint16_t *>(p.w), p.K, p.N);
    NTS_LAUNCH_CHECK("dense_turn_kernel");
  } else {
    p.b = p.w, p.b_stride = p.K;
  }
  if (type == NTS_F32) launch_product_of<float, USE>(p, share, stream);
  else if (type == NTS_BF16) launch_product_of<Bf16, USE>(p, share, stream);
  else launch_product_of<F16, USE>(p, share, stream);
  NTS_LAUNCH_CHECK("dense_rows_kernel");
  return NTS_OK;
}
template <typename T, bool PAIRS>
void launch_weight_of(const DenseArgs &p, const dim3 &grid, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.dz32) {
      hipLaunchKernelGGL((dense_weight_kernel<T, PAIRS, kInWords>), grid, dim3(256), 0, stream, p);
      return;
    }
  }
  if (p.y) hipLaunchKernelGGL((dense_weight_kernel<T, PAIRS, kMasked>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((dense_weight_kernel<T, PAIRS, kPlain>), grid, dim3(256), 0, stream, p);
}
template <typename T>
void launch_weight(const DenseArgs &p, const dim3 &grid, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.M % 2 == 0 && p.N % 2 == 0) return launch_weight_of<T, true>(p, grid, stream);
  }
  launch_weight_of<T, false>(p, grid, stream);
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

size_t nts_dense_work_bytes(int type, uint32_t n, uint32_t N, uint32_t F) {
  return bad_shapes(type, N, F, 0, nullptr) || n <= kFewRows ? 0 : weight_bytes(type, n, N, F, false);
}

int nts_dense(void *y, const void *x, const void *w, const void *bias, const void *residual, int type, uint32_t n, uint32_t N,
              uint32_t F, int activation, const nts_dropout_t *dropout, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_dense");
  if (const char *why = bad_shapes(type, N, F, activation, dropout)) return fail_in("nts_dense", why);
  if (n == 0) return NTS_OK;
  if (!y || !x || !w) return fail_in("nts_dense", "null pointer");
  for (const void *at : {static_cast<const void *>(y), x, w, bias, residual})
    if (!aligned_to(at, type_size(type))) return fail_in("nts_dense", "a value's alignment");
  DenseArgs p{};
  p.a = x, p.w = w, p.M = n, p.N = N, p.K = F, p.a_stride = F, p.out = y, p.bias = bias, p.more = residual;
  p.act = activation, p.drop = drop_args(dropout);
  if (n <= kFewRows) {
    if (type == NTS_F32) launch_few<float>(p, stream);
    else if (type == NTS_BF16) launch_few<Bf16>(p, stream);
    else launch_few<F16>(p, stream);
    NTS_LAUNCH_CHECK("nts_dense");
    return NTS_OK;
  }
  if (!work || !aligned_to(work, 16)) return fail_in("nts_dense", "needs nts_dense_work_bytes of 16-byte-aligned work");
  return launch_product<kLayer>(p, type, work, stream);
}

size_t nts_dense_grad_work_bytes(int type, uint32_t n, uint32_t N, uint32_t F, int activation, int with_dropout, int with_y, int with_rows,
                                 int with_weight, int with_bias) {
  if (bad_shapes(type, N, F, activation, nullptr)) return 0;
  return grad_work(type, n, N, F, activation, with_dropout != 0, with_y != 0, with_rows != 0, with_weight != 0, with_bias != 0).bytes;
}

int nts_dense_grad(void *gx, void *gw, void *gb, const void *g, const void *x, const void *w, const void *bias, const void *y, int type,
                   uint32_t n, uint32_t N, uint32_t F, int activation, const nts_dropout_t *dropout, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_dense_grad");
  const char *const name = "nts_dense_grad";
  if (const char *why = bad_shapes(type, N, F, activation, dropout)) return fail_in(name, why);
  if ((n == 0 || !gx) && !gw && !gb) return NTS_OK;
  const Work layout = grad_work(type, n, N, F, activation, dropout != nullptr, y != nullptr, gx != nullptr, gw != nullptr, gb != nullptr);
  if (n && (!g || ((gw || layout.again) && !x) || ((gx || layout.again) && !w))) return fail_in(name, "null pointer");
  for (const void *at : {static_cast<const void *>(gx), static_cast<const void *>(gw), static_cast<const void *>(gb), g, x, w, bias, y})
    if (!aligned_to(at, type_size(type))) return fail_in(name, "a value's alignment");
  if (layout.bytes && (!work || !aligned_to(work, 16))) return fail_in(name, "needs nts_dense_grad_work_bytes of 16-byte-aligned work");
  char *const base = static_cast<char *>(work);
  void *const prepared = base + layout.weight_at;
  uint32_t sum_rows = n || layout.beside ? layout.sums : 0u;
  float *const sums = gb ? reinterpret_cast<float *>(base + layout.sums_at) : nullptr;
  const void *dz = g;
  DenseArgs p{};
  p.drop = drop_args(dropout), p.act = activation, p.w = w, p.mask_scale = 1.0f;
  p.drop.step_kept = nullptr;
  if (n && (layout.stored || (gb && !layout.beside))) {
    DenseArgs q = p;
    q.more = g, q.M = n, q.N = N, q.sums = sums;
    if (layout.stored) dz = q.out = work;
    if (layout.from_y) q.y = y, q.mask_scale = p.drop.scale;
    if (layout.again) {
      q.a = x, q.K = F, q.a_stride = F, q.bias = bias;
      sum_rows = share_for<kSlope>(q, type).workers;
      if (const int status = launch_product<kSlope>(q, type, prepared, stream)) return status;
    } else {
      const dim3 grid(ceil_div(N, kWave), layout.sums);
      if (type == NTS_F32) hipLaunchKernelGGL(dense_columns_kernel<float>, grid, dim3(256), 0, stream, q);
      else if (type == NTS_BF16) hipLaunchKernelGGL(dense_columns_kernel<Bf16>, grid, dim3(256), 0, stream, q);
      else hipLaunchKernelGGL(dense_columns_kernel<F16>, grid, dim3(256), 0, stream, q);
      NTS_LAUNCH_CHECK("dense_columns_kernel");
    }
  }
  if (layout.masked) p.y = y, p.mask_scale = p.drop.scale;
  p.after = layout.masked || (layout.stored && !layout.again) ? p.drop.scale : 1.0f;
  p.dz32 = layout.dz32;
  if (gx && n) {
    DenseArgs q = p;
    q.a = dz, q.M = n, q.N = F, q.K = N, q.a_stride = N, q.out = gx;
    if (const int status = launch_product<kRows>(q, type, prepared, stream)) return status;
  }
  if (gw) {
    DenseArgs q = p;
    q.a = dz, q.b = x, q.M = N, q.N = F, q.K = n, q.a_stride = N, q.b_stride = F, q.out = gw, q.part_terms = layout.parts.terms;
    q.tiles_m = ceil_div(N, kTile), q.tiles_n = ceil_div(F, kTile);
    if (layout.beside) q.column_sums = sums;
    const uint32_t parts = layout.parts.count;
    q.sums = parts > 1 ? reinterpret_cast<float *>(base + layout.parts_at) : nullptr;
    const dim3 grid(q.tiles_m * q.tiles_n, 1, parts);
    if (type == NTS_F32) launch_weight<float>(q, grid, stream);
    else if (type == NTS_BF16) launch_weight<Bf16>(q, grid, stream);
    else launch_weight<F16>(q, grid, stream);
    NTS_LAUNCH_CHECK("dense_weight_kernel");
    if (parts > 1)
      if (const int status = launch_sum(gw, type, q.sums, static_cast<uint64_t>(N) * F, parts, stream)) return status;
  }
  if (gb)
    if (const int status = launch_sum(gb, type, sums, N, sum_rows, stream)) return status;
  return NTS_OK;
}

}  // extern "C"
