// Kernels of attention over neighbours' float rows (dot_args.hpp: what is computed), for one type of values to a source file.
#pragma once

#include <algorithm>

#include "dot_args.hpp"
#include "edge_spans.hpp"
#include "launch_size.hpp"

namespace nts {
namespace {

// How the rows that edges name are read.  By buffer descriptors and 32-bit offsets, where an edge without a row and a lane without a
// piece get an offset behind the end: tables of up to 1.5 GB and 2^24 rows, whose rows begin at multiples of 4 bytes and have a piece at
// least; heads of whole lanes (16 columns times a power of two) need no look at single pieces.  The others go by address.
enum Reach { kWhole, kPieces, kFar };
// A walker per row, walkers that take spans, and those that are wavefronts.
enum Form { kPerRow, kNarrow, kWide };

// Wavefronts to a SIMD that the registers allow, and edges of a slot that are requested together.  2.48 M edges, 8 heads of 64 in bf16 with
// gradients: 2,390 us; two edges and wavefronts in place of four and four, three, two: 2,420 with 6, 3, 2, 2,350 with 5, 4, 3, with which 360,000
// edges of 4 heads of 32 in 32 bits take 464 instead of 350.  Of walkers per row, 410,000 edges of 8 heads of 32 in 16 bits take 64 us forward
// with three and 69 with four, which spill; 1,020,000 of 8 query heads of 64 that share 2 heads 113 and 106.
template <typename T, int KIND, int REACH, int FORM>
constexpr int kWavesOf = KIND == kForward         ? (REACH == kWhole && FORM == kWide && sizeof(T) == 2            ? 4
                                                     : (REACH != kWhole && FORM == kNarrow) || (REACH == kFar && FORM == kPerRow) ? 2
                                                                                                                                  : 3)
                         : KIND == kByDestination && REACH == kWhole && FORM == kWide ? 3
                                                                                      : 2;
template <typename T>
constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;

// sum: of p c, norm: of p.  Where no p counts, nothing does.
__device__ __forceinline__ Ends ends_of(float base2, float sum, float norm) {
  return norm == 0.0f ? Ends{base2, 0.0f, 0.0f} : Ends{base2, sum / norm, 1.0f / norm};
}

// What an edge without a row reads.
__device__ __attribute__((aligned(16))) float zero_row[256];
// Offsets behind the end of every buffer, which read zeros: of an edge without a row, also with a row's bytes added, and of a piece that a
// lane does not have, with any edge's offset added.
constexpr uint32_t kNowhere = 0x80000000u, kNoPiece = static_cast<uint32_t>(kMostNear);  // their sum is one, too

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void *p, uint64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, static_cast<uint32_t>(bytes), 0x00027000);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 Loaded __attribute__((aligned(2)));  // global memory takes 16 bytes at any value's address
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// c plus the products of a piece's values, in 32 bits.  Products of 16-bit values are exact.
template <typename T>
__device__ __forceinline__ float dot_piece(u32x4 a, u32x4 b, float c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = fmaf(__uint_as_float(a[i]), __uint_as_float(b[i]), c);
  return c;
}
template <>
__device__ __forceinline__ float dot_piece<Bf16>(u32x4 a, u32x4 b, float c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = a[i], y = b[i];  // an element itself cannot be cast: its bits are taken from where the vector begins
    c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), __builtin_bit_cast(bf16x2, y), c, false);
  }
  return c;
}
template <>
__device__ __forceinline__ float dot_piece<F16>(u32x4 a, u32x4 b, float c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = a[i], y = b[i];
    c = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), __builtin_bit_cast(f16x2, y), c, false);
  }
  return c;
}
template <typename T>
__device__ __forceinline__ float value_of(u32x4 a, int i) {
  if (sizeof(T) == 4) return __uint_as_float(a[i]);
  return ValueOf<T>::get(static_cast<uint16_t>(i & 1 ? a[i / 2] >> 16 : a[i / 2] & 0xFFFFu));
}
template <>
__device__ __forceinline__ float value_of<Bf16>(u32x4 a, int i) {
  return __uint_as_float(i & 1 ? a[i / 2] & 0xFFFF0000u : a[i / 2] << 16);
}

// WIDE: a walker is a wavefront, whose row, edges and loops are then in scalar registers.
template <typename T, int ND, int KIND, int REACH, bool WIDE>
struct Walk {
  static constexpr bool NEAR = REACH != kFar;
  static constexpr int C = 16, CH = 16 / sizeof(T), NC = C / CH;
  typedef typename ValueOf<T>::raw raw;
  const DotArgs &p;
  uint32_t dl, unit, first_head, heads_of_pass, slot, slot_lanes, rounds, lanes_base, step_now;
  bool live;
  uint32_t col[NC], skip[NC], piece_at[NC];  // a piece's first column (and byte), and how many of its values belong to the piece before it (CH: no piece)
  uint32_t row_bytes, lane_at;  // of the rows that edges name; the lane's first byte there
  uint32_t own_at;              // the lane's head in the row that is walked over
  __amdgpu_buffer_rsrc_t rx, ry, rends;
  uint32_t row;
  // forward: a = q, s = sum of w v.  By destination: a = q, b = g, s = sum of p c k, t = sum of p k.  By source: a = k, b = v, s = gk, t = gv.
  u32x4 a[NC], b[NC];
  float s[C], t[C], top, sum, norm, base2;  // norm: by destination, sum of p
  uint32_t at;  // the lane's first column (of 16) after join()

  __device__ __forceinline__ Walk(const DotArgs &args, uint32_t pass) : p(args) {
    constexpr uint32_t kShift = ND == 1 ? 0 : ND == 2 ? 1 : ND == 4 ? 2 : ND == 8 ? 3 : 4;
    const uint32_t lane = threadIdx.x & (kWave - 1), l = WIDE ? lane : lane & ((1u << p.walker_shift) - 1u);
    lanes_base = lane - l;
    dl = l & (ND - 1);
    unit = (pass << p.hw_shift) + ((l >> kShift) & ((1u << p.hw_shift) - 1u));
    heads_of_pass = (1u << p.hw_shift) * (KIND == kBySource ? min(p.share, 32u) : 1u);
    first_head = (pass << p.hw_shift) * (KIND == kBySource ? p.share : 1u);
    rounds = (WIDE ? 6u : p.walker_shift) - p.hw_shift - kShift;
    slot_lanes = ND << p.hw_shift;
    slot = l >> (kShift + p.hw_shift);
    live = unit < p.units;
    if (!live) unit = 0;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const uint32_t c = j * ND + dl;
      col[j] = c < p.chunks ? c * CH : 0u;
      skip[j] = c < p.chunks ? 0u : CH;
      if (c < p.chunks && col[j] + CH > p.D && !p.narrow) {
        skip[j] = CH - p.D % CH;
        col[j] = p.D - CH;
      }
      piece_at[j] = c < p.chunks ? col[j] * static_cast<uint32_t>(sizeof(T)) : kNoPiece;
    }
    const uint32_t width = KIND == kBySource ? p.q_heads : p.heads;
    row_bytes = width * p.D * sizeof(T);
    own_at = unit * p.D;
    lane_at = (KIND == kBySource ? unit * p.share : unit / p.share) * p.D * sizeof(T) + (REACH == kWhole ? dl * 16u : 0u);
    if (NEAR) {
      const uint64_t bytes = static_cast<uint64_t>(p.others) * row_bytes;
      rx = buffer_of(KIND == kBySource ? p.q : p.k, bytes);
      ry = buffer_of(KIND == kBySource ? p.g : p.v, bytes);
      if (KIND == kBySource) rends = buffer_of(p.ends, static_cast<uint64_t>(p.others) * p.q_heads * sizeof(Ends));
    }
    step_now = p.drop.threshold ? drop_step(p.drop) : 0u;
  }

  // Values that are another piece's, or none, are 0.
  __device__ __forceinline__ void clear_skipped(u32x4 *v) const {
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        if (sizeof(T) == 4) v[j][i] = i >= skip[j] ? v[j][i] : 0u;
        else v[j][i] &= (2u * i >= skip[j] ? 0xFFFFu : 0u) | (2u * i + 1u >= skip[j] ? 0xFFFF0000u : 0u);
      }
  }
  // A head's columns by address.
  __device__ __forceinline__ void get(const T *row_at, uint32_t head_at, u32x4 *v) const {
    const T *const from = row_at + head_at;
    if (!NEAR && p.narrow) {
      raw part[CH] = {};
#pragma unroll
      for (uint32_t i = 0; i < CH - 1; ++i)
        if (i < p.D) part[i] = *reinterpret_cast<const raw *>(from + i);
      v[0] = __builtin_bit_cast(u32x4, part);
#pragma unroll
      for (int j = 1; j < NC; ++j) v[j] = u32x4{0, 0, 0, 0};
      if (dl) v[0] = u32x4{0, 0, 0, 0};
      return;
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) v[j] = *reinterpret_cast<const Loaded *>(row_at + (head_at + col[j]));
    if (REACH != kWhole) clear_skipped(v);
  }
  // The same `from` bytes into the buffer.
  __device__ __forceinline__ void get(__amdgpu_buffer_rsrc_t buffer, uint32_t from, u32x4 *v) const {
#pragma unroll
    for (int j = 0; j < NC; ++j) v[j] = __builtin_amdgcn_raw_buffer_load_b128(buffer, REACH == kWhole ? from + j * ND * 16 : from + piece_at[j], 0, 0);
    if (REACH == kPieces && p.partial_piece) clear_skipped(v);
  }
  __device__ __forceinline__ float dot(const u32x4 *x, const u32x4 *y) const {
    float d = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j) d = dot_piece<T>(x[j], y[j], d);
    return lanes_sum<ND>(d);
  }

  // `some`: the row has edges.
  __device__ __forceinline__ void begin(uint32_t r, bool some) {
    row = r;
#pragma unroll
    for (int i = 0; i < C; ++i) s[i] = t[i] = 0.0f;
    sum = norm = 0.0f;
    top = -INFINITY;
    base2 = INFINITY;
    if (KIND == kBySource && !some) return;  // elsewhere few rows have none, and the load need not wait for the offsets
    const uint64_t first = static_cast<uint64_t>(r) * (KIND == kBySource ? p.heads : p.q_heads) * p.D;
    if (KIND == kBySource) {
      get(static_cast<const T *>(p.k) + first, own_at, a);
      get(static_cast<const T *>(p.v) + first, own_at, b);
    } else {
      get(static_cast<const T *>(p.q) + first, own_at, a);
      if (KIND == kByDestination) {
        get(static_cast<const T *>(p.g) + first, own_at, b);
        const float l = (p.lse + static_cast<uint64_t>(r) * p.q_heads)[unit];
        if (l != -INFINITY) base2 = l * kLog2e;  // otherwise no score counts: every p is 0
      }
    }
  }

  // Bits of the dropout for up to 32 heads from `from` on, of the edge between the row and `id`.
  __device__ __forceinline__ uint32_t drop_word(uint32_t id, uint32_t from) const {
    uint32_t word = 0;
    for (uint32_t g = from >> 3; g <= (from + heads_of_pass - 1u) >> 3; ++g) {
      const uint32_t bits = keep_bits(edge_numbers(p.drop, step_now, KIND == kBySource ? row : id, KIND == kBySource ? id : row, g), p.drop.threshold);
      const int shift = static_cast<int>(g * 8u) - static_cast<int>(from);
      word |= shift >= 0 ? bits << shift : bits >> -shift;
    }
    return word;
  }
  __device__ __forceinline__ float drop_factor(uint32_t word, uint32_t bit) const {
    return !p.drop.threshold ? 1.0f : word >> (bit & 31u) & 1u ? p.drop.scale : 0.0f;  // lanes without a unit have a bit that no word has
  }

  // Rows of U edges, requested together.  where[u]: NEAR the offset of the edge's row, kNowhere for none; else its id, kNoSlot for none.
  template <int U>
  __device__ __forceinline__ void request(const uint32_t *where, uint32_t more, u32x4 (*x)[NC], u32x4 (*y)[NC]) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (NEAR) {
        get(rx, where[u] + lane_at + more, x[u]);
        get(ry, where[u] + lane_at + more, y[u]);
      } else {
        const bool there = where[u] != kNoSlot;
        const T *const none = reinterpret_cast<const T *>(zero_row);
        const uint64_t from = (static_cast<uint64_t>(where[u]) * row_bytes + lane_at + more) / sizeof(T);
        get(there ? static_cast<const T *>(KIND == kBySource ? p.q : p.k) + from : none, 0u, x[u]);
        get(there ? static_cast<const T *>(KIND == kBySource ? p.g : p.v) + from : none, 0u, y[u]);
      }
    }
  }
  static __device__ __forceinline__ bool there(uint32_t where) { return NEAR ? where < kNowhere : where != kNoSlot; }

  // In the gradients an edge whose score is -infinity has no part, whatever its rows hold: 0 times their infinities would be NaN.
  static __device__ __forceinline__ void leave_out(bool out, u32x4 *x, u32x4 *y, float *gv, float *mean) {
#pragma unroll
    for (int j = 0; j < NC; ++j) x[j] = out ? u32x4{0, 0, 0, 0} : x[j], y[j] = out ? u32x4{0, 0, 0, 0} : y[j];
    *gv = out ? 0.0f : *gv, *mean = out ? 0.0f : *mean;
  }

  template <int U>
  __device__ __forceinline__ void step(const uint32_t *where, const uint32_t *ids, const uint32_t *words, uint32_t from) {
    const float scale2 = p.score_scale * kLog2e;
    if (KIND == kBySource) {
      const uint32_t h0 = unit * p.share + from, h1 = min(h0 + 32u, unit * p.share + p.share);
      for (uint32_t h = h0; h < h1; ++h) {
        u32x4 x[U][NC], y[U][NC];
        Ends e[U];
        request<U>(where, (h - unit * p.share) * p.D * static_cast<uint32_t>(sizeof(T)), x, y);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (NEAR) {
            const auto got = __builtin_amdgcn_raw_buffer_load_b96(rends, there(where[u]) ? (__umul24(ids[u], p.q_heads) + h) * static_cast<uint32_t>(sizeof(Ends)) : kNowhere, 0, 0);
            e[u] = Ends{__uint_as_float(got[0]), __uint_as_float(got[1]), __uint_as_float(got[2])};
          } else {
            e[u] = *(there(where[u]) ? p.ends + static_cast<uint64_t>(ids[u]) * p.q_heads + h : reinterpret_cast<const Ends *>(zero_row));
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float qk = dot(x[u], a);
          float gv = dot(y[u], b);
          const float z = fmaf(qk, scale2, -e[u].base2);
          const float w = there(where[u]) ? __builtin_amdgcn_exp2f(z) * e[u].share : 0.0f;
          if (__any(z == -INFINITY)) leave_out(z == -INFINITY, x[u], y[u], &gv, &e[u].mean);
          const float m = drop_factor(words[u], h - first_head - from);
          const float c = m == 0.0f ? 0.0f : gv * m;
          const float ds = w * (c - e[u].mean) * p.score_scale, wm = w * m;
#pragma unroll
          for (int i = 0; i < C; ++i)
            s[i] = fmaf(ds, value_of<T>(x[u][i / CH], i % CH), s[i]), t[i] = fmaf(wm, value_of<T>(y[u][i / CH], i % CH), t[i]);
        }
      }
      return;
    }
    u32x4 x[U][NC], y[U][NC];
    request<U>(where, 0u, x, y);
    if (KIND == kByDestination) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float qk = dot(a, x[u]), z = fmaf(qk, scale2, -base2);
        float gv = dot(b, y[u]), none;
        const float w = there(where[u]) ? __builtin_amdgcn_exp2f(z) : 0.0f;
        if (__any(z == -INFINITY)) leave_out(z == -INFINITY, x[u], y[u], &gv, &none);
        const float m = drop_factor(words[u], unit - first_head), wc = m == 0.0f ? 0.0f : w * (gv * m);
        sum += wc, norm += w;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float k = value_of<T>(x[u][i / CH], i % CH);
          s[i] = fmaf(wc, k, s[i]), t[i] = fmaf(w, k, t[i]);
        }
      }
      return;
    }
    float z[U], now = top;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float d = dot(a, x[u]) * scale2;
      z[u] = there(where[u]) ? d : -INFINITY;
      now = fmaxf(now, z[u]);
    }
    const float base = now == -INFINITY ? 0.0f : now, keep = __builtin_amdgcn_exp2f(top - base);
    top = now;
    sum *= keep;
#pragma unroll
    for (int i = 0; i < C; ++i) s[i] *= keep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = __builtin_amdgcn_exp2f(z[u] - base);
      sum += w;
      const float wm = w * drop_factor(words[u], unit - first_head);
#pragma unroll
      for (int i = 0; i < C; ++i) s[i] = fmaf(wm, value_of<T>(y[u][i / CH], i % CH), s[i]);
    }
  }

  // Edges [j0, j1) of the row whose edges begin at `first`: the walker's lanes look up one edge each, and the next ones ahead.
  __device__ __forceinline__ void edges(uint32_t first, uint32_t j0, uint32_t j1) {
    if (j0 >= j1) return;
    const uint32_t *ids = p.ids + first;
    const uint32_t width = WIDE ? 64u : 1u << p.walker_shift, l = (threadIdx.x & (kWave - 1)) - lanes_base, slots = 1u << rounds;
    uint32_t next = j0 + l < j1 ? ids[j0 + l] : kNoSlot;
    for (uint32_t base = j0; base < j1;) {
      const uint32_t id = next < p.others ? next : kNoSlot;
      const uint32_t where = !NEAR ? id : id != kNoSlot ? __umul24(id, row_bytes) : kNowhere;
      const uint32_t count = min(width, j1 - base);
      next = base + width < j1 && base + width + l < j1 ? ids[base + width + l] : kNoSlot;
      base += count;
      // by source, heads that share their keys in turns of 32 (in one, unless there are more)
      for (uint32_t from = 0; from < (KIND == kBySource ? p.share : 1u); from += 32u) {
        const uint32_t word = p.drop.threshold ? drop_word(id, first_head + from) : 0u;
        uint32_t i = 0;
        auto take = [&](auto u_) __attribute__((always_inline)) {
          constexpr int U = decltype(u_)::value;
          uint32_t places[U], mine[U], words[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint32_t j = i + u * slots + slot;
            const int lane = static_cast<int>((lanes_base + (j & (width - 1u))) * 4u);
            places[u] = __builtin_amdgcn_ds_bpermute(lane, where);
            mine[u] = KIND == kBySource && NEAR ? __builtin_amdgcn_ds_bpermute(lane, id) : places[u];
            words[u] = p.drop.threshold ? __builtin_amdgcn_ds_bpermute(lane, word) : 0u;
            if (j >= count) places[u] = NEAR ? kNowhere : kNoSlot;
          }
          step<U>(places, mine, words, from);
          i += U * slots;
        };
        while (i < count) {
          if (kAhead<T> > 2 && count - i > 2u * slots) take(std::integral_constant<int, kAhead<T>>());
          else if (count - i > slots) take(std::integral_constant<int, 2>());
          else take(std::integral_constant<int, 1>());
        }
      }
      if (count < width) break;  // the last edges (base would not pass 2^32)
    }
  }

  // The value of the lane whose number differs in bit M alone.
  template <int M>
  static __device__ __forceinline__ float across(float v) {
    const int x = __float_as_int(v);
    if (M == 8) return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x128, 0xF, 0xF, true));  // eight further round the row of sixteen
    return __int_as_float(__builtin_amdgcn_ds_swizzle(x, (M << 10) | 0x1F));
  }
  // The values of the lane with bit M clear and of the one with it set, in both: of `low` on the one side, of `high` on the other.
  template <int M>
  static __device__ __forceinline__ float2 both_sides(float low, float high, bool upper) {
    if (M >= 16) {
      const auto pair = M == 32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(low), __float_as_uint(high), false, false)
                                : __builtin_amdgcn_permlane16_swap(__float_as_uint(low), __float_as_uint(high), false, false);
      return make_float2(__uint_as_float(pair[0]), __uint_as_float(pair[1]));
    }
    // The empty statement keeps the compiler from choosing between the values' places instead, which would put the arrays into memory.
    asm("" : "+v"(low), "+v"(high));
    const float keep = upper ? high : low, other = across<M>(upper ? low : high);
    return make_float2(upper ? other : keep, upper ? keep : other);
  }
  // A round of join(): HALF of the lane's columns go to the other lane, the part of the others comes from there.
  template <int M, int HALF>
  __device__ __forceinline__ void join_round() {
    const bool upper = (threadIdx.x & M) != 0;
    if (HALF && upper) at += HALF;
    float f = 1.0f, o = 1.0f;
    if (KIND == kForward) {
      const float2 tops = both_sides<M>(top, top, upper);
      top = fmaxf(tops.x, tops.y);
      const float base = top == -INFINITY ? 0.0f : top;
      f = __builtin_amdgcn_exp2f(tops.x - base), o = __builtin_amdgcn_exp2f(tops.y - base);
    }
    // both sides add in the same order
    auto joined = [&](float low, float high) {
      const float2 v = both_sides<M>(low, high, upper);
      return KIND == kForward ? fmaf(v.y, o, v.x * f) : v.x + v.y;
    };
    if (KIND != kBySource) sum = joined(sum, sum);
    if (KIND == kByDestination) norm = joined(norm, norm);
#pragma unroll
    for (int i = 0; i < (HALF ? HALF : 1); ++i) {
      s[i] = joined(s[i], s[i + HALF]);
      if (KIND != kForward) t[i] = joined(t[i], t[i + HALF]);
    }
  }
  // Joins the slots, the furthest lanes first.  Each round halves a lane's columns: 16 columns and 2^r slots take 8 + 4 + .. exchanges
  // instead of 16 a round.
  template <int M, int HALF>
  __device__ __forceinline__ void join_from() {
    if constexpr (M >= ND) {
      if (M < slot_lanes) return;
      join_round<M, HALF>();
      join_from<M / 2, HALF / 2>();
    }
  }
  __device__ __forceinline__ void join() {
    at = 0;
    if (WIDE || p.walker_shift == 6) return join_from<32, 8>();
    if (p.walker_shift == 5) return join_from<16, 8>();
    if (p.walker_shift == 4) return join_from<8, 8>();
    if (p.walker_shift == 3) return join_from<4, 8>();
    if (p.walker_shift == 2) return join_from<2, 8>();
    if (p.walker_shift == 1) return join_from<1, 8>();
  }

  // The lane's values after join() to a head's columns.
  template <typename U>
  __device__ __forceinline__ void store(U *row_at, uint32_t head_at, const float *v) const {
    if (rounds > 4u && (slot & ((1u << (rounds - 4u)) - 1u))) return;  // the slots of the last rounds hold the same column
    const uint32_t count = rounds < 4 ? 16u >> rounds : 1u;
    if (REACH != kWhole) {
      U *const to = row_at + head_at;
#pragma unroll
      for (uint32_t i = 0; i < C; ++i) {
        const uint32_t c = at + i, w = c % CH;
        uint32_t place = col[0], none = skip[0];
#pragma unroll
        for (int j = 1; j < NC; ++j)
          if (c / CH == static_cast<uint32_t>(j)) place = col[j], none = skip[j];
        if (i < count && w >= none && place + w < p.D) put_value(to + place + w, v[i]);
      }
      return;
    }
    // whole pieces: number j begins ND lanes behind number j - 1
    const uint32_t first = head_at + dl * CH + at / CH * (ND * CH) + at % CH;
    if (count == 16) {
#pragma unroll
      for (int j = 0; j < NC; ++j) put_values<CH>(row_at + (first + j * ND * CH), v + j * CH);
    } else if (count == 8) {
#pragma unroll
      for (int j = 0; j < NC / 2; ++j) put_values<CH>(row_at + (first + j * ND * CH), v + j * CH);
    } else if (count == 4) {
      put_values<4>(row_at + first, v);
    } else if (count == 2) {
      put_values<2>(row_at + first, v);
    } else {
      put_value(row_at + first, v[0]);
    }
  }

  __device__ __forceinline__ void write() {
    if (!live) return;
    const uint64_t first = static_cast<uint64_t>(row) * (KIND == kBySource ? p.heads : p.q_heads) * p.D;
    if (KIND == kBySource) {
      store(static_cast<T *>(p.out) + first, own_at, s);
      store(static_cast<T *>(p.out2) + first, own_at, t);
      return;
    }
    const uint64_t head = static_cast<uint64_t>(row) * p.q_heads;
    if (KIND == kForward) {
      // the reciprocal is within one step of 32 bits, and its product another half
      const float f = sum == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum);
#pragma unroll
      for (int i = 0; i < C; ++i) s[i] = sum == 0.0f ? 0.0f : s[i] * f;
      if (dl == 0 && slot == 0) (p.lse + head)[unit] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
      const Ends e = ends_of(base2, sum, norm);
#pragma unroll
      for (int i = 0; i < C; ++i) s[i] = fmaf(-e.mean, t[i], s[i]) * (p.score_scale * e.share);
      if (dl == 0 && slot == 0) (p.ends + head)[unit] = e;
    }
    store(static_cast<T *>(p.out) + first, own_at, s);
  }

  // A part of a row's edges, for join_dot_spans_kernel.
  __device__ __forceinline__ void write_partial(uint64_t record) const {
    if (!live) return;
    float *const to = p.partial + record * record_size<KIND>(p.q_heads, p.heads, p.D);
    const uint32_t columns = (KIND == kBySource ? p.heads : p.q_heads) * p.D;
    store(to, own_at, s);
    if (KIND != kForward) store(to, columns + own_at, t);
    if (dl == 0 && slot == 0) {
      if (KIND == kForward) to[columns + unit] = top, to[columns + p.q_heads + unit] = sum;
      if (KIND == kByDestination) to[2u * columns + unit] = sum, to[2u * columns + p.q_heads + unit] = norm;
    }
  }
};

__device__ __forceinline__ uint64_t walker_of_grid(const DotArgs &p, bool wide, uint32_t *pass) {
  const uint32_t block = blockIdx.x / p.passes;
  *pass = blockIdx.x - block * p.passes;
  return wide ? block * 4ull + wave_of_block() : (static_cast<uint64_t>(block) * 256u + threadIdx.x) >> p.walker_shift;
}
// An offset by the scalar cache: offsets are only read.
__device__ __forceinline__ uint32_t offset_at(const uint32_t *offsets, uint64_t row) {
  return *reinterpret_cast<const __attribute__((address_space(4))) uint32_t *>(reinterpret_cast<uintptr_t>(offsets + row));
}
__device__ __forceinline__ void keep_step(const DotArgs &p) {
  if (p.drop.step_kept && blockIdx.x == 0 && threadIdx.x == 0) *p.drop.step_kept = drop_step(p.drop);
}

// A walker per row.  40,000 rows of 9 edges, 4 heads of 32 in 32 bits: 68 us, 5.4 TB/s of keys and values, and 65 by destination.
template <typename T, int ND, int KIND, int REACH>
__global__ __launch_bounds__(256, (kWavesOf<T, KIND, REACH, kPerRow>)) void dot_rows_kernel(DotArgs p) {
  keep_step(p);
  uint32_t pass;
  uint64_t row = walker_of_grid(p, false, &pass);
  Walk<T, ND, KIND, REACH, false> w(p, pass);
  const uint64_t walkers = static_cast<uint64_t>(gridDim.x / p.passes) * 256u >> p.walker_shift;
  for (; row < p.rows; row += walkers) {
    const uint32_t first = p.offsets[row], degree = p.offsets[row + 1] - first;
    w.begin(static_cast<uint32_t>(row), degree > 0);
    w.edges(first, 0, degree);
    w.join();
    w.write();
  }
}

// A block per destination, for few destinations of up to some thousand edges: its wavefronts share the edges and join through LDS, in
// one launch.  One of 300 edges, 4 heads of 32 in 32 bits: 8.4 us, three memory latencies and a launch.
constexpr uint32_t kBlockWaves = 16;
template <typename T, int ND, int REACH>
__global__ __launch_bounds__(kBlockWaves *kWave) void dot_block_kernel(DotArgs p) {
  __shared__ float tops[kBlockWaves][kWave], sums[kBlockWaves][kWave], accs[kBlockWaves][kWave * 16];  // of a pass's heads
  keep_step(p);
  const uint32_t row = blockIdx.x / p.passes, pass = blockIdx.x - row * p.passes, wave = wave_of_block();
  const uint32_t first = offset_at(p.offsets, row), degree = offset_at(p.offsets, row + 1u) - first;
  {
    Walk<T, ND, kForward, REACH, true> w(p, pass);
    const uint32_t share = (degree + kBlockWaves - 1u) / kBlockWaves, j0 = min(degree, wave * share), j1 = min(degree, j0 + share);
    w.begin(row, j0 < j1);
    w.edges(first, j0, j1);
    w.join();
    if (w.live) {
      const uint32_t unit = w.unit - (pass << p.hw_shift);
      w.store(accs[wave], unit * p.D, w.s);
      if (w.dl == 0 && w.slot == 0) tops[wave][unit] = w.top, sums[wave][unit] = w.sum;
    }
  }
  __syncthreads();
  const uint32_t units = min(1u << p.hw_shift, p.units - (pass << p.hw_shift));
  for (uint32_t i = threadIdx.x; i < units * p.D; i += kBlockWaves * kWave) {
    const uint32_t unit = i / p.D;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kBlockWaves; ++w) top = fmaxf(top, tops[w][unit]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (uint32_t w = 0; w < kBlockWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(tops[w][unit] - base);
      sum = fmaf(sums[w][unit], f, sum);
      acc = fmaf(accs[w][i], f, acc);
    }
    const uint64_t head = static_cast<uint64_t>(row) * p.q_heads + (pass << p.hw_shift);
    put_value(static_cast<T *>(p.out) + head * p.D + i, sum == 0.0f ? 0.0f : acc / sum);
    if (i == unit * p.D) p.lse[head + unit] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

// Walkers that take spans of rows and edges, however long the rows are.  2.48 M edges, 8 heads of 64 in bf16: 740 us forward, 760 by destination
// and 810 by source: 5.1 GB of rows at 6.3-6.9 TB/s from beyond the L2s, which hold few of them.  8 query heads on 2: 330 us, vector
// instructions for three quarters of the time.  (A chiplet to a head, whose rows its L2 holds more of: 1,030 us.)
template <typename T, int ND, int KIND, int REACH, bool WIDE>
__global__ __launch_bounds__(256, (kWavesOf<T, KIND, REACH, WIDE ? kWide : kNarrow>)) void dot_spans_kernel(DotArgs p) {
  keep_step(p);
  uint32_t pass;
  const uint64_t span = walker_of_grid(p, WIDE, &pass);
  if (span >= p.spans) return;
  Walk<T, ND, KIND, REACH, WIDE> w(p, pass);
  auto offset = [&](uint32_t row) { return WIDE ? offset_at(p.offsets, row) : p.offsets[row]; };
  const uint64_t begin = span * p.span, end = min(begin + p.span, p.positions);
  const uint32_t co0 = offset(0);
  uint32_t tail = kNoSlot;
  uint32_t row = destination_at(p.offsets, co0, p.rows, begin, WIDE ? 6u : p.walker_shift);
  if (WIDE) row = wave_first(row);
  uint32_t first = offset(row);
  for (; row < p.rows; ++row) {
    const uint32_t next = offset(row + 1), degree = next - first;
    const uint64_t at = static_cast<uint64_t>(row) * kRowCost + (first - co0), edges_at = at + kRowCost;
    if (at >= end) break;
    const bool cut = degree > p.span;
    const uint32_t mine = first;
    first = next;
    if (at < begin && !cut) continue;  // the earlier span has done it
    const uint32_t j0 = edges_at < begin ? static_cast<uint32_t>(min<uint64_t>(begin - edges_at, degree)) : 0u;
    const uint32_t j1 = !cut ? degree : edges_at < end ? static_cast<uint32_t>(min<uint64_t>(degree, end - edges_at)) : 0u;
    if (j0 >= j1 && at < begin) continue;
    w.begin(row, j0 < j1);
    w.edges(mine, j0, j1);
    w.join();
    if (!cut) {
      w.write();
      continue;
    }
    w.write_partial(span * 2u + (at < begin ? 0u : 1u));
    if (at >= begin) tail = row;
  }
  if (pass == 0 && (threadIdx.x & ((1u << p.walker_shift) - 1u)) == 0) p.tail_row[span] = tail;
}

// The rows that were cut: 64 columns of kJoinSpans spans' rows a block.  Every wavefront takes rows of few parts of its own; of longer ones
// all take every kJoinWaves-th part, and the first adds up what they have.  Parts in order, so the same bits on every call.  2.48 M edges of 8
// heads of 64: 20-30 us.
constexpr uint32_t kJoinWaves = 16, kJoinSpans = 32, kJoinAhead = 8, kJoinAlone = 16;
// What the parts of a column come to.  Forward: largest score, sum and weighted sum; by destination: the sums of p k, p c, p c k and p.
template <int KIND>
struct Joined {
  float top = KIND == kForward ? -INFINITY : 0.0f, sum = 0.0f, acc = 0.0f, norm = 0.0f;
  __device__ __forceinline__ void add(float t, float l, float v, float n) {
    if (KIND == kForward) {
      const float now = fmaxf(top, t), base = now == -INFINITY ? 0.0f : now;
      const float f = __builtin_amdgcn_exp2f(top - base), o = __builtin_amdgcn_exp2f(t - base);
      top = now;
      sum = sum * f + l * o;
      acc = acc * f + v * o;
    } else {
      top += t, sum += l, acc += v, norm += n;
    }
  }
};
template <typename T, int KIND>
__global__ __launch_bounds__(kJoinWaves *kWave) void join_dot_spans_kernel(DotArgs p) {
  __shared__ float tops[kJoinWaves][kWave], sums[kJoinWaves][kWave], accs[kJoinWaves][kWave], norms[KIND == kByDestination ? kJoinWaves : 1][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block(), of_norms = KIND == kByDestination ? wave : 0u;
  const uint32_t columns = (KIND == kBySource ? 2u * p.heads : p.q_heads) * p.D, c = blockIdx.y * kWave + lane, cc = min(c, columns - 1u), h = cc / p.D;
  const uint64_t size = record_size<KIND>(p.q_heads, p.heads, p.D);
  const uint64_t span0 = static_cast<uint64_t>(blockIdx.x) * kJoinSpans;
  const uint32_t rows = lane < kJoinSpans && span0 + lane < p.spans ? p.tail_row[span0 + lane] : kNoSlot;
  uint64_t cut = __ballot(rows != kNoSlot);  // the same in every wavefront
  // where a record has the other numbers of a column
  const uint64_t at_a = KIND == kForward ? columns + h : columns + cc, at_b = KIND == kForward ? columns + p.q_heads + h : 2ull * columns + h;
  const uint64_t at_c = 2ull * columns + p.q_heads + h;
  auto parts_of = [&](uint64_t first, uint64_t last, uint64_t from, uint64_t step) {
    Joined<KIND> j;
    for (uint64_t s = from; s <= last; s += kJoinAhead * step) {
      float t[kJoinAhead], l[kJoinAhead], v[kJoinAhead], n[kJoinAhead];
#pragma unroll
      for (uint32_t u = 0; u < kJoinAhead; ++u) {
        const uint64_t part = s + u * step;
        t[u] = KIND == kForward ? -INFINITY : 0.0f, l[u] = v[u] = n[u] = 0.0f;
        if (part <= last) {
          const float *const record = p.partial + (part * 2u + (part == first ? 1u : 0u)) * size;
          v[u] = record[cc];
          if (KIND != kBySource) t[u] = record[at_a], l[u] = record[at_b];
          if (KIND == kByDestination) n[u] = record[at_c];
        }
      }
#pragma unroll
      for (uint32_t u = 0; u < kJoinAhead; ++u) j.add(t[u], l[u], v[u], n[u]);
    }
    return j;
  };
  auto write = [&](uint32_t row, const Joined<KIND> &j) {
    if (c >= columns) return;
    const uint64_t head = static_cast<uint64_t>(row) * p.q_heads + h;
    if (KIND == kForward) {
      put_value(static_cast<T *>(p.out) + static_cast<uint64_t>(row) * columns + c, j.sum == 0.0f ? 0.0f : j.acc / j.sum);
      if (c == h * p.D) p.lse[head] = j.sum == 0.0f ? -INFINITY : (j.top + __builtin_amdgcn_logf(j.sum)) * kLn2;
    } else if (KIND == kByDestination) {
      const float l = p.lse[head];
      const Ends e = ends_of(l == -INFINITY ? INFINITY : l * kLog2e, j.sum, j.norm);
      put_value(static_cast<T *>(p.out) + static_cast<uint64_t>(row) * columns + c, fmaf(-e.mean, j.top, j.acc) * (p.score_scale * e.share));
      if (c == h * p.D) p.ends[head] = e;
    } else {
      const bool second = c >= columns / 2u;
      put_value(static_cast<T *>(second ? p.out2 : p.out) + static_cast<uint64_t>(row) * (columns / 2u) + (second ? c - columns / 2u : c), j.acc);
    }
  };
  auto last_part = [&](uint32_t row) {  // where its last edge lies
    const uint64_t at = static_cast<uint64_t>(row) * kRowCost + (kRowCost - 1u) + (offset_at(p.offsets, row + 1ull) - offset_at(p.offsets, 0));
    return min<uint64_t>(at / p.span, p.spans - 1u);
  };
  uint64_t together = 0;
  for (uint32_t taker = 0; cut; cut &= cut - 1, ++taker) {
    const uint32_t k = __builtin_ctzll(cut), row = wave_read(rows, k);
    const uint64_t first = span0 + k, last = last_part(row);
    if (last - first >= kJoinAlone) together |= 1ull << k;
    else if (taker % kJoinWaves == wave) write(row, parts_of(first, last, first, 1u));
  }
  for (; together; together &= together - 1) {
    const uint32_t k = __builtin_ctzll(together), row = wave_read(rows, k);
    const uint64_t first = span0 + k;
    Joined<KIND> j = parts_of(first, last_part(row), first + wave, kJoinWaves);
    tops[wave][lane] = j.top, sums[wave][lane] = j.sum, accs[wave][lane] = j.acc;
    if (KIND == kByDestination) norms[of_norms][lane] = j.norm;
    __syncthreads();
    if (wave == 0) {
      for (uint32_t w = 1; w < kJoinWaves; ++w) j.add(tops[w][lane], sums[w][lane], accs[w][lane], norms[KIND == kByDestination ? w : 0][lane]);
      write(row, j);
    }
    __syncthreads();
  }
}

template <typename T, int ND, int KIND, int REACH>
int launch(const DotArgs &p, hipStream_t stream) {
  if constexpr (KIND == kForward && REACH != kFar) {
    if (p.blocks) {
      hipLaunchKernelGGL((dot_block_kernel<T, ND, REACH>), dim3(p.rows * p.passes), dim3(kBlockWaves * kWave), 0, stream, p);
      NTS_LAUNCH_CHECK("dot_block_kernel");
      return NTS_OK;
    }
  }
  const uint32_t walkers = 256u >> p.walker_shift;  // a block's
  if (!p.span) {
    if (KIND == kBySource) return NTS_OK;  // always in spans
    const uint64_t blocks = std::min<uint64_t>(ceil_div(p.rows, walkers), kMostBlocks / p.passes) * p.passes;
    hipLaunchKernelGGL((dot_rows_kernel<T, ND, KIND == kBySource ? kForward : KIND, REACH>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream, p);
    NTS_LAUNCH_CHECK("dot_rows_kernel");
    return NTS_OK;
  }
  const dim3 grid(ceil_div(p.spans, walkers) * p.passes);
  if (REACH != kFar && p.walker_shift == 6)
    hipLaunchKernelGGL((dot_spans_kernel<T, ND, KIND, REACH, REACH != kFar>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((dot_spans_kernel<T, ND, KIND, REACH, false>), grid, dim3(256), 0, stream, p);
  NTS_LAUNCH_CHECK("dot_spans_kernel");
  if (p.spans > 1) {  // with one span no row has more edges than it has positions
    const uint64_t columns = static_cast<uint64_t>(KIND == kBySource ? 2 * p.heads : p.q_heads) * p.D;
    hipLaunchKernelGGL((join_dot_spans_kernel<T, KIND>), dim3(ceil_div(p.spans, kJoinSpans), ceil_div(columns, kWave)), dim3(kJoinWaves * kWave), 0,
                       stream, p);
    NTS_LAUNCH_CHECK("join_dot_spans_kernel");
  }
  return NTS_OK;
}
template <typename T, int KIND, int REACH>
int launch_nd(const DotArgs &p, uint32_t nd, hipStream_t stream) {
  switch (nd) {
    case 1: return launch<T, 1, KIND, REACH>(p, stream);
    case 2: return launch<T, 2, KIND, REACH>(p, stream);
    case 4: return launch<T, 4, KIND, REACH>(p, stream);
    case 8: return launch<T, 8, KIND, REACH>(p, stream);
    default: return launch<T, 16, KIND, REACH>(p, stream);
  }
}

template <typename T, int KIND>
int launch_reach(const DotArgs &p, uint32_t nd, bool near, hipStream_t stream) {
  if (!near) return launch_nd<T, KIND, kFar>(p, nd, stream);
  return p.ragged ? launch_nd<T, KIND, kPieces>(p, nd, stream) : launch_nd<T, KIND, kWhole>(p, nd, stream);
}

template <typename T>
int launch_kind(int kind, const DotArgs &p, uint32_t nd, bool near, hipStream_t stream) {
  if (kind == kForward) return launch_reach<T, kForward>(p, nd, near, stream);
  return kind == kByDestination ? launch_reach<T, kByDestination>(p, nd, near, stream) : launch_reach<T, kBySource>(p, nd, near, stream);
}

}  // namespace
}  // namespace nts
