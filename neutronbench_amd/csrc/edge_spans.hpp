// How attention over neighbours shares rows of edges out among walkers (aligned groups of lanes of a wavefront), and sums inside one.
#pragma once

#include "common.hpp"

namespace nts {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kRowCost = 8;  // 2.48 M edges in 169 K rows, 4 heads of 32 in 8 bits: 194 us when chosen (201 now); 4: 209, 16: 192, 1: 230

inline uint32_t next_power(uint32_t v) {
  uint32_t p = 1;
  while (p < v) p <<= 1;
  return p;
}
inline uint32_t shift_of(uint32_t power) { return static_cast<uint32_t>(__builtin_ctz(power)); }

#if defined(__HIPCC__)
// Sum over an aligned group of ND lanes, the same in all of them; the exchanges are part of the additions.
template <int CTRL>
__device__ __forceinline__ float add_lane(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int ND>
__device__ __forceinline__ float lanes_sum(float v) {
  if (ND > 1) v = add_lane<0xB1>(v);   // neighbours in pairs
  if (ND > 2) v = add_lane<0x4E>(v);   // pairs in fours
  if (ND > 4) v = add_lane<0x141>(v);  // fours, mirrored within eight
  if (ND > 8) v = add_lane<0x140>(v);  // eights, mirrored within sixteen
  if (ND > 16) {                       // the other sixteen
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(both[0]) + __uint_as_float(both[1]);
  }
  return v;
}

// Long rows are shared out and short ones bundled without a look at the degrees on the host: rows and edges are
// lined up -- row r takes kRowCost positions from r * kRowCost + offsets[r] - offsets[0] on, which is what beginning and writing a
// row costs in edges, and its edges the positions behind them -- and every walker takes the rows that begin within its
// span of positions.  A row of more edges than a span has positions is cut at the spans' ends: every span that it reaches into
// sums its part into a record (1: the row begins in this span, 0: in an earlier one) and a second launch adds the
// parts in order.  No atomics: the same bits on every call.
__device__ __forceinline__ uint64_t position_of(const uint32_t *co, uint32_t co0, uint64_t r) { return r * kRowCost + (co[r] - co0); }

// The last row at or before position x: a candidate for every lane of the walker a step.
__device__ __forceinline__ uint32_t destination_at(const uint32_t *co, uint32_t co0, uint32_t Vd, uint64_t x, uint32_t walker_shift) {
  const uint32_t lanes = 1u << walker_shift, lane = threadIdx.x & (lanes - 1u);
  const uint64_t group = lanes == 64u ? ~0ull : ((1ull << lanes) - 1ull) << ((threadIdx.x & 63u) & ~(lanes - 1u));
  uint32_t lo = 0, hi = Vd;  // position_of(lo) <= x, the answer is in [lo, hi)
  while (hi - lo > 1) {
    const uint32_t step = lanes == 1u ? (hi - lo) / 2u : (hi - lo - 1u) / lanes + 1u;
    const uint64_t r = static_cast<uint64_t>(lo) + static_cast<uint64_t>(lanes == 1u ? 1u : lane) * step;
    const bool before = r < hi && position_of(co, co0, r) <= x;
    if (lanes == 1u) {
      if (before) lo += step; else hi = lo + step;
      continue;
    }
    const uint32_t count = __popcll(__ballot(before) & group);  // lane 0 always counts
    const uint32_t next = lo + (count - 1u) * step;
    hi = hi - next > step ? next + step : hi;
    lo = next;
  }
  return lo;
}
#endif

}  // namespace nts
