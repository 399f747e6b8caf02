// Number formats of the vertex tables that are held in few bits.
//   e8m0   a scale byte b: 2^(b - 127), 255 = NaN
//   e2m1   4 bits: sign, and 0, 0.5, 1, 1.5, 2, 3, 4, 6
//   e4m3   8 bits: sign, 4 bits of exponent, 3 of fraction; at most 448; 0x7F / 0xFF = NaN, no infinity
#pragma once

#include "common.hpp"

namespace nts {

constexpr uint32_t kMxBlock = 32;  // values that share a scale in a 4-bit row
inline __host__ __device__ uint32_t mx_blocks(uint32_t F) { return F / kMxBlock + (F % kMxBlock != 0); }
// Scale bytes are kept in rows of whole words, so that four blocks' scales are one aligned load.
inline __host__ __device__ uint32_t mx_scale_stride(uint32_t F) { return (mx_blocks(F) + 3) / 4 * 4; }
constexpr uint32_t kMostWidth = 1u << 17;  // columns (and outputs) of a row: the tiles of any product fit one launch
// Columns of a row that the cache of 8-bit keys and values keeps: whole 16-byte loads.
inline __host__ __device__ uint32_t kv8_row_width(uint32_t D) { return (D + 15) / 16 * 16; }

// An output from this size on is more than the L2s hold (8 of 4 MB) and is written past the caches.  Its reader does not seem to miss
// it there: twelve batches of a Products-shaped epoch, whose 94 MB of gathered features the aggregation reads next, take 11.4 ms
// with this bound and 11.5 with one of 256 MB, which nothing in them reaches.
constexpr uint64_t kStreamedBytes = 32ull << 20;

#if defined(__HIPCC__)
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// Four floats at an address that is a multiple of four bytes only: global memory takes a 16-byte access there.
typedef float FloatQuad __attribute__((ext_vector_type(4), aligned(4)));
// Stores them, past the caches if `streamed`.  The empty statements keep the compiler from making one plain store of the two.
__device__ __forceinline__ void store_quad(float *to, FloatQuad v, bool streamed) {
  if (streamed) {
    asm volatile("");
    __builtin_nontemporal_store(v, reinterpret_cast<FloatQuad *>(to));
    asm volatile("");
  } else {
    *reinterpret_cast<FloatQuad *>(to) = v;
  }
}

__device__ __forceinline__ float e8m0_value(uint32_t b) {
  return b == 0u ? __uint_as_float(0x00400000u) : b == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(b << 23);
}
// 2^-(b - 127) for the bytes that the quantisers write (0 .. 252): a normal float.
__device__ __forceinline__ float e8m0_inverse(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// The four e2m1 values of the lower half of a word, lowest four bits first, times `scale`.
__device__ __forceinline__ void e2m1_decode4(uint32_t word, float scale, float *v) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 1);
  v[0] = a.x * scale, v[1] = a.y * scale, v[2] = b.x * scale, v[3] = b.y * scale;
}
// The eight e2m1 values of a word, lowest four bits first, times `scale`.
__device__ __forceinline__ void e2m1_decode8(uint32_t word, float scale, float *v) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 1),
              c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 3);
  v[0] = a.x * scale, v[1] = a.y * scale, v[2] = b.x * scale, v[3] = b.y * scale;
  v[4] = c.x * scale, v[5] = c.y * scale, v[6] = d.x * scale, v[7] = d.y * scale;
}

// Nearest e2m1 code (ties to the even code, magnitudes above 6 become 6) of y = x * inverse, finite.
__device__ __forceinline__ uint32_t e2m1_encode(float x, float inverse) {
  const float y = fabsf(x) * inverse;
  const uint32_t bits = __float_as_uint(y);
  // from 1 up the code is the exponent and the first bit of the fraction; below it a count of halves
  const uint32_t large = ((bits + 0x1FFFFFu + ((bits >> 22) & 1u)) >> 22) - 252u;
  const uint32_t small = static_cast<uint32_t>(__builtin_rintf(y * 2.0f));
  const uint32_t code = y < 1.0f ? small : (large < 7u ? large : 7u);
  return code | ((__float_as_uint(x) >> 28) & 8u);
}

// Four e4m3 values of a word.
__device__ __forceinline__ void e4m3_decode4(uint32_t word, float *v) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), true);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
// Four floats of at most 448 as e4m3, ties to even; what is not finite becomes NaN.
__device__ __forceinline__ uint32_t e4m3_encode4(const float *v) {
  float u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = fabsf(v[i]) <= 448.0f ? v[i] : __uint_as_float(0x7FC00000u);
  int word = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], 0, false);
  word = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], word, true);
  return static_cast<uint32_t>(word);
}
#endif

}  // namespace nts
