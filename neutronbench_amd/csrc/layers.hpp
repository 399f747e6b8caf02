// What the operators of a layer in training share: values of 32 and 16 bits, the numbers that dropout draws.
#pragma once

#include "common.hpp"

namespace nts {

constexpr uint32_t kMostColumns = 1u << 17;  // columns (and outputs) of a row

inline bool known_type(int type) { return type == NTS_F32 || type == NTS_BF16 || type == NTS_F16; }
inline size_t type_size(int type) { return type == NTS_F32 ? 4 : 2; }

// Dropout as the kernels take it.  A value is dropped where its 16-bit number is below `threshold` (0: nothing is; 65,536: all).
struct DropArgs {
  uint32_t threshold, key0, key1, step;
  float scale;
  const uint32_t *step_device;  // the step is read there, and `step` is 0
  uint32_t *step_kept;          // and written here
};
inline const char *bad_dropout(const nts_dropout_t *d) {
  if (d && !(d->p >= 0.0f && d->p <= 1.0f)) return "dropout's p is not within 0 .. 1";
  return nullptr;
}
inline DropArgs drop_args(const nts_dropout_t *d) {
  DropArgs a{};
  a.scale = 1.0f;
  if (!d) return a;
  // p is a 32-bit value: its product with 2^16 is exact, and half way between two whole numbers goes to the even one
  a.threshold = static_cast<uint32_t>(__builtin_rint(static_cast<double>(d->p) * 65536.0));
  a.scale = a.threshold < 65536u ? static_cast<float>(65536.0 / (65536.0 - a.threshold)) : 0.0f;
  a.key0 = static_cast<uint32_t>(d->seed), a.key1 = static_cast<uint32_t>(d->seed >> 32);
  a.step = d->step_device ? 0u : d->step, a.step_device = d->step_device, a.step_kept = d->step_kept;
  return a;
}

#if defined(__HIPCC__)
// Values of 16 bits are raw words: their arithmetic is in 32 bits.
struct Bf16 {
  uint16_t bits;
};
struct F16 {
  uint16_t bits;
};
template <typename T>
struct ValueOf;
template <>
struct ValueOf<float> {
  typedef float raw;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct ValueOf<Bf16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
  static __device__ __forceinline__ uint16_t put(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }
};
template <>
struct ValueOf<F16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(uint16_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
  static __device__ __forceinline__ uint16_t put(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
};
template <typename T>
__device__ __forceinline__ float get_value(const T *at) { return ValueOf<T>::get(*reinterpret_cast<const typename ValueOf<T>::raw *>(at)); }
template <typename T>
__device__ __forceinline__ void put_value(T *at, float v) { *reinterpret_cast<typename ValueOf<T>::raw *>(at) = ValueOf<T>::put(v); }

// N neighbouring values at any address that is a multiple of a value's size: global memory takes accesses of 16 bytes there.
template <typename T, int N>
struct Pack {
  typedef typename ValueOf<T>::raw raw;
  typedef raw type __attribute__((ext_vector_type(N), aligned(sizeof(raw))));
};
template <int N, typename T>
__device__ __forceinline__ void get_values(const T *at, float *v) {
  const typename Pack<T, N>::type p = *reinterpret_cast<const typename Pack<T, N>::type *>(at);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = ValueOf<T>::get(p[i]);
}
// Past the caches if `streamed`: what the L2s do not hold.  The empty statements keep the compiler from making one plain store of the two.
template <int N, typename T>
__device__ __forceinline__ void put_values(T *at, const float *v, bool streamed = false) {
  typename Pack<T, N>::type p;
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = ValueOf<T>::put(v[i]);
  if (streamed) {
    asm volatile("");
    __builtin_nontemporal_store(p, reinterpret_cast<typename Pack<T, N>::type *>(at));
    asm volatile("");
  } else {
    *reinterpret_cast<typename Pack<T, N>::type *>(at) = p;
  }
}

// Philox-4x32 with ten rounds (J. Salmon et al., Parallel random numbers: as easy as 1, 2, 3, 2011): 128 bits of counter and 64 of
// key to 128 bits.  Number i of the eight is half i % 2 of word i / 2.
__device__ __forceinline__ uint4 philox(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c.x) * 0xD2511F53u, b = static_cast<uint64_t>(c.z) * 0xCD9E8D57u;
    c = make_uint4(static_cast<uint32_t>(b >> 32) ^ c.y ^ k0, static_cast<uint32_t>(b), static_cast<uint32_t>(a >> 32) ^ c.w ^ k1,
                   static_cast<uint32_t>(a));
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return c;
}
__device__ __forceinline__ uint32_t drop_step(const DropArgs &d) { return d.step + (d.step_device ? *d.step_device : 0u); }
__device__ __forceinline__ uint32_t half_of(const uint4 &n, int i) {
  const uint32_t w = i / 2 == 0 ? n.x : i / 2 == 1 ? n.y : i / 2 == 2 ? n.z : n.w;
  return i & 1 ? w >> 16 : w & 0xFFFFu;
}
// Bit i set: number i says keep.
__device__ __forceinline__ uint32_t keep_bits(const uint4 &n, uint32_t threshold) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) bits |= half_of(n, i) >= threshold ? 1u << i : 0u;
  return bits;
}
// Columns 8 * group .. 8 * group + 7 of a row.
__device__ __forceinline__ uint4 row_numbers(const DropArgs &d, uint32_t step, uint32_t row, uint32_t group) {
  return philox(make_uint4(group, row, step, 0u), d.key0, d.key1);
}
// Query heads 8 * group .. 8 * group + 7 of the edge from `src` to `dst`.
__device__ __forceinline__ uint4 edge_numbers(const DropArgs &d, uint32_t step, uint32_t src, uint32_t dst, uint32_t group) {
  return philox(make_uint4(src, dst, step, 1u + group), d.key0, d.key1);
}
#endif

}  // namespace nts
