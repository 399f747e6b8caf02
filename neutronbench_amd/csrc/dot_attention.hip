// Attention of destinations over the float rows of their edges' sources, and its gradients.
//   forward       s_e = scale <q[d], k[src e]>, p_e = exp(s_e) / sum, out[d] = sum_e m_e p_e v[src e]; lse = log of the sum
//   by destination (offsets, ids: the edges by destination)
//                 p_e again from lse; c_e = m_e <g[d], v[src e]>, mean = sum_e p_e c_e,
//                 gq[d] = scale sum_e p_e (c_e - mean) k[src e] = scale (sum_e p_e c_e k[src e] - mean sum_e p_e k[src e])
//   by source     (offsets, ids: the edges by source)
//                 gk[s] = scale sum_e p_e (c_e - mean[dst e]) q[dst e], gv[s] = sum_e m_e p_e g[dst e]
// per query head, which shares its keys and values with the other heads of its group; m is the dropout's 0 or 1 / (1 - p).
// Both sums of gq and the mean come from one pass over the edges, so neither `out` nor the scores are kept.
#include <algorithm>

#include "edge_spans.hpp"
#include "launch_size.hpp"
#include "layers.hpp"

namespace nts {
namespace {

enum Kind { kForward, kByDestination, kBySource };

// A lane holds 8 columns of one head ("unit": a query head, by source a head of keys), as one 16-byte piece of 16-bit
// values or two of 32-bit ones, ND lanes apart, so that neighbouring lanes read neighbouring 16 bytes.  ND lanes (a power of two) cover a
// unit, 2^hw_shift units lie side by side, and further edges of the row go to further such sets of lanes ("slots"), joined at
// the end.  All slots of a row are a walker; a wavefront is one walker or several.
struct DotArgs {
  void *out, *out2;  // out; gq; gk and gv
  float *lse;
  float2 *ends;  // [Vd, q_heads]: lse over log 2, mean
  const void *q, *k, *v, *g;
  const uint32_t *offsets, *ids;
  uint32_t rows, others;  // rows that are walked over; rows that ids may name
  uint32_t q_heads, heads, share, D, chunks;
  bool narrow, ragged;  // less than a piece; the last piece is not whole or some lanes have none
  float score_scale;
  DropArgs drop;
  uint32_t units, hw_shift, walker_shift, passes;
  uint32_t span, spans;  // edges in spans of positions (edge_spans.hpp)
  uint64_t positions;
  float *partial;
  uint32_t *tail_row;
};

// Wavefronts to a SIMD that the registers allow.
template <typename T, int KIND>
constexpr int kWavesOf = KIND == kForward && sizeof(T) == 2 ? 4 : KIND == kBySource ? 2 : 3;

// What an edge without a row reads.
__device__ __attribute__((aligned(16))) float zero_row[256];

// Floats of a span's record.
template <int KIND>
__host__ __device__ __forceinline__ uint64_t record_size(uint32_t q_heads, uint32_t heads, uint32_t D) {
  if (KIND == kForward) return static_cast<uint64_t>(q_heads) * (D + 2u);
  if (KIND == kByDestination) return static_cast<uint64_t>(q_heads) * (2u * D + 1u);
  return 2ull * heads * D;
}

template <typename T, int ND, int KIND>
struct Walk {
  static constexpr int CH = 16 / sizeof(T), NC = 8 / CH;
  typedef typename Pack<T, CH>::type Piece;
  const DotArgs &p;
  const T *const pq, *const pk, *const pv, *const pg;
  uint32_t dl, unit, first_head, heads_of_pass, slot, rounds, lanes_base, step_now;
  bool live;
  uint32_t col[NC], skip[NC];  // a piece's first column, and how many of its values belong to the piece before it (CH: no piece)
  uint32_t row;
  // forward: a = q, s = sum of w v.  By destination: a = q, b = g, s = sum of p c k, t = sum of p k.  By source: a = k, b = v, s = gk, t = gv.
  float a[8], b[8], s[8], t[8], top, sum, base2;
  uint32_t at;  // the lane's first column (of 8) after join()

  __device__ __forceinline__ Walk(const DotArgs &args, uint32_t pass)
      : p(args), pq(static_cast<const T *>(args.q)), pk(static_cast<const T *>(args.k)), pv(static_cast<const T *>(args.v)),
        pg(static_cast<const T *>(args.g)) {
    constexpr uint32_t kShift = ND == 1 ? 0 : ND == 2 ? 1 : ND == 4 ? 2 : ND == 8 ? 3 : ND == 16 ? 4 : 5;
    const uint32_t lane = threadIdx.x & (kWave - 1), l = lane & ((1u << p.walker_shift) - 1u);
    lanes_base = lane - l;
    dl = l & (ND - 1);
    unit = (pass << p.hw_shift) + ((l >> kShift) & ((1u << p.hw_shift) - 1u));
    heads_of_pass = (1u << p.hw_shift) * (KIND == kBySource ? min(p.share, 32u) : 1u);
    first_head = (pass << p.hw_shift) * (KIND == kBySource ? p.share : 1u);
    rounds = p.walker_shift - p.hw_shift - kShift;
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
    }
    step_now = p.drop.threshold ? drop_step(p.drop) : 0u;
  }

  __device__ __forceinline__ void get(const T *from, Piece *v) const {
    if (p.narrow) {
#pragma unroll
      for (int i = 0; i < CH; ++i) v[0][i] = 0;
#pragma unroll
      for (uint32_t i = 0; i < CH - 1; ++i)
        if (i < p.D) v[0][i] = *reinterpret_cast<const typename Pack<T, CH>::raw *>(from + i);
#pragma unroll
      for (int j = 1; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < CH; ++i) v[j][i] = 0;
      return;
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) v[j] = *reinterpret_cast<const Piece *>(from + col[j]);
  }
  __device__ __forceinline__ void floats(const Piece *v, float *f) const {
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < CH; ++i) f[j * CH + i] = ValueOf<T>::get(v[j][i]);
    if (p.ragged) {
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (uint32_t i = 0; i < CH; ++i) f[j * CH + i] = i >= skip[j] ? f[j * CH + i] : 0.0f;
    }
  }
  __device__ __forceinline__ void get_floats(const T *from, float *f) const {
    Piece v[NC];
    get(from, v);
    floats(v, f);
  }

  __device__ __forceinline__ void begin(uint32_t r) {
    row = r;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = t[i] = 0.0f;
    sum = 0.0f;
    top = -INFINITY;
    const uint64_t first = (static_cast<uint64_t>(r) * (KIND == kBySource ? p.heads : p.q_heads) + unit) * p.D;
    if (KIND == kBySource) {
      get_floats(pk + first, a);
      get_floats(pv + first, b);
    } else {
      get_floats(pq + first, a);
      if (KIND == kByDestination) {
        get_floats(pg + first, b);
        const float l = p.lse[static_cast<uint64_t>(r) * p.q_heads + unit];
        base2 = l == -INFINITY ? INFINITY : l * kLog2e;  // no score counts: every p is 0
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
    return !p.drop.threshold ? 1.0f : word >> bit & 1u ? p.drop.scale : 0.0f;
  }

  // U edges of the slot, ids[u] (kNoSlot: none); their rows are requested together.
  template <int U>
  __device__ __forceinline__ void step(const uint32_t *ids, const uint32_t *words, uint32_t from) {
    const float scale2 = p.score_scale * kLog2e;
    if (KIND == kBySource) {
      const uint32_t h0 = unit * p.share + from, h1 = min(h0 + 32u, unit * p.share + p.share);
      for (uint32_t h = h0; h < h1; ++h) {
        Piece x[U][NC], y[U][NC];
        float2 e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool there = ids[u] != kNoSlot;
          const uint64_t head = static_cast<uint64_t>(ids[u]) * p.q_heads + h;
          const T *const none = reinterpret_cast<const T *>(zero_row);
          get(there ? pq + head * p.D : none, x[u]);
          get(there ? pg + head * p.D : none, y[u]);
          e[u] = *(there ? p.ends + head : reinterpret_cast<const float2 *>(zero_row));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float q[8], g[8], qk = 0.0f, gv = 0.0f;
          floats(x[u], q);
          floats(y[u], g);
#pragma unroll
          for (int i = 0; i < 8; ++i) qk = fmaf(q[i], a[i], qk), gv = fmaf(g[i], b[i], gv);
          qk = lanes_sum<ND>(qk), gv = lanes_sum<ND>(gv);
          const float w = ids[u] != kNoSlot ? __builtin_amdgcn_exp2f(fmaf(qk, scale2, -e[u].x)) : 0.0f;
          const float m = drop_factor(words[u], h - first_head - from);
          const float c = m == 0.0f ? 0.0f : gv * m;
          const float ds = w * (c - e[u].y) * p.score_scale, wm = w * m;
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i] = fmaf(ds, q[i], s[i]), t[i] = fmaf(wm, g[i], t[i]);
          __builtin_amdgcn_sched_barrier(0);  // one edge's floats at a time: the registers do not hold all
        }
      }
      return;
    }
    Piece x[U][NC], y[U][NC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = ids[u] != kNoSlot;
      const uint64_t from = (static_cast<uint64_t>(ids[u]) * p.heads + unit / p.share) * p.D;
      const T *const none = reinterpret_cast<const T *>(zero_row);
      get(there ? pk + from : none, x[u]);
      get(there ? pv + from : none, y[u]);
    }
    if (KIND == kByDestination) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float k[8], v[8], qk = 0.0f, gv = 0.0f;
        floats(x[u], k);
        floats(y[u], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) qk = fmaf(a[i], k[i], qk), gv = fmaf(b[i], v[i], gv);
        qk = lanes_sum<ND>(qk), gv = lanes_sum<ND>(gv);
        const float w = ids[u] != kNoSlot ? __builtin_amdgcn_exp2f(fmaf(qk, scale2, -base2)) : 0.0f;
        const float m = drop_factor(words[u], unit - first_head), wc = m == 0.0f ? 0.0f : w * (gv * m);
        sum += wc;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = fmaf(wc, k[i], s[i]), t[i] = fmaf(w, k[i], t[i]);
        __builtin_amdgcn_sched_barrier(0);  // one edge's floats at a time: the registers do not hold all
      }
      return;
    }
    float z[U], now = top;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float k[8], dot = 0.0f;
      floats(x[u], k);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(a[i], k[i], dot);
      dot = lanes_sum<ND>(dot) * scale2;
      z[u] = ids[u] != kNoSlot ? dot : -INFINITY;
      now = fmaxf(now, z[u]);
    }
    const float base = now == -INFINITY ? 0.0f : now, keep = __builtin_amdgcn_exp2f(top - base);
    top = now;
    sum *= keep;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= keep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[8];
      floats(y[u], v);
      const float w = __builtin_amdgcn_exp2f(z[u] - base);
      sum += w;
      const float wm = w * drop_factor(words[u], unit - first_head);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = fmaf(wm, v[i], s[i]);
    }
  }

  // Edges [j0, j1) of the row whose edges begin at `first`: the walker's lanes look up one edge each, and the next ones ahead.
  __device__ __forceinline__ void edges(uint32_t first, uint32_t j0, uint32_t j1) {
    if (j0 >= j1) return;
    const uint32_t *ids = p.ids + first;
    const uint32_t width = 1u << p.walker_shift, l = (threadIdx.x & (kWave - 1)) - lanes_base, slots = 1u << rounds;
    uint32_t next = j0 + l < j1 ? ids[j0 + l] : kNoSlot;
    for (uint32_t base = j0; base < j1;) {
      const uint32_t id = next < p.others ? next : kNoSlot;
      const uint32_t count = min(width, j1 - base);
      next = base + width < j1 && base + width + l < j1 ? ids[base + width + l] : kNoSlot;
      base += count;
      // by source, heads that share their keys in turns of 32 (in one, unless there are more)
      for (uint32_t from = 0; from < (KIND == kBySource ? p.share : 1u); from += 32u) {
        const uint32_t word = p.drop.threshold ? drop_word(id, first_head + from) : 0u;
        uint32_t i = 0;
        auto take = [&](auto u_) __attribute__((always_inline)) {
          constexpr int U = decltype(u_)::value;
          uint32_t mine[U], words[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint32_t j = i + u * slots + slot;
            mine[u] = __shfl(id, lanes_base + (j & (width - 1u)), kWave);
            words[u] = p.drop.threshold ? __shfl(word, lanes_base + (j & (width - 1u)), kWave) : 0u;
            if (j >= count) mine[u] = kNoSlot;
          }
          step<U>(mine, words, from);
          i += U * slots;
        };
        while (i < count) {
          if (count - i > 2u * slots) take(std::integral_constant<int, 4>());
          else if (count - i > slots) take(std::integral_constant<int, 2>());
          else take(std::integral_constant<int, 1>());
        }
      }
      if (count < width) break;  // the last edges (base would not pass 2^32)
    }
  }

  // Joins the slots.  Each round halves a lane's columns: it hands one half to the lane of the other slot and takes in that one's
  // part of its own half.
  __device__ __forceinline__ void join() {
    at = 0;
    const uint32_t lanes = 1u << (p.walker_shift - rounds);
#pragma unroll
    for (uint32_t r = 0; r < 6; ++r) {
      if (r >= rounds) break;
      const uint32_t m = lanes << r;
      const int half = r < 3 ? 4 >> r : 0;
      const bool upper = (slot >> r) & 1u;
      if (half && upper) at += half;
      float f = 1.0f, o = 1.0f;
      const float more = KIND == kBySource ? 0.0f : __shfl_xor(sum, m, kWave);
      if (KIND == kForward) {
        const float other = __shfl_xor(top, m, kWave), now = fmaxf(top, other), base = now == -INFINITY ? 0.0f : now;
        f = __builtin_amdgcn_exp2f(top - base), o = __builtin_amdgcn_exp2f(other - base);
        top = now;
      }
      // both sides of the exchange add in the same order: the lower slot's part first
      sum = upper ? more * o + sum * f : sum * f + more * o;
      if (half) {
#pragma unroll
        for (int i = 0; i < (half ? half : 1); ++i) {
          const float mine = upper ? s[i + half] : s[i], give = upper ? s[i] : s[i + half];
          s[i] = mine * f + __shfl_xor(give, m, kWave) * o;
          if (KIND != kForward) {
            const float mine2 = upper ? t[i + half] : t[i], give2 = upper ? t[i] : t[i + half];
            t[i] = mine2 + __shfl_xor(give2, m, kWave);
          }
        }
      } else {
        s[0] = s[0] * f + __shfl_xor(s[0], m, kWave) * o;
        if (KIND != kForward) t[0] += __shfl_xor(t[0], m, kWave);
      }
    }
  }

  // The lane's values after join() to a head's columns.
  template <typename U>
  __device__ __forceinline__ void store(U *to, const float *v) const {
    if (slot >> 3) return;  // further slots hold the same columns
    const uint32_t count = rounds < 3 ? 8u >> rounds : 1u;
    if (p.narrow || p.ragged) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        if (i >= count) break;
        const uint32_t c = at + i, j = c / CH, w = c % CH;
        const uint32_t place = (NC > 1 && j ? col[NC - 1] : col[0]) + w, none = NC > 1 && j ? skip[NC - 1] : skip[0];
        if (w >= none && place < p.D) put_value(to + place, v[i]);
      }
    } else if (count == 8) {
#pragma unroll
      for (int j = 0; j < NC; ++j) put_values<CH>(to + col[j], v + j * CH);
    } else {
      to += (NC > 1 && at / CH ? col[NC - 1] : col[0]) + at % CH;
      if (count == 4) put_values<4>(to, v);
      else if (count == 2) put_values<2>(to, v);
      else put_value(to, v[0]);
    }
  }

  __device__ __forceinline__ void write() {
    if (!live) return;
    if (KIND == kBySource) {
      const uint64_t first = (static_cast<uint64_t>(row) * p.heads + unit) * p.D;
      store(static_cast<T *>(p.out) + first, s);
      store(static_cast<T *>(p.out2) + first, t);
      return;
    }
    const uint64_t head = static_cast<uint64_t>(row) * p.q_heads + unit;
    if (KIND == kForward) {
      const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = sum == 0.0f ? 0.0f : s[i] * f;
      if (dl == 0 && slot == 0) p.lse[head] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = fmaf(-sum, t[i], s[i]) * p.score_scale;
      if (dl == 0 && slot == 0) p.ends[head] = make_float2(base2, sum);
    }
    store(static_cast<T *>(p.out) + head * p.D, s);
  }

  // A part of a row's edges, for join_dot_spans_kernel.
  __device__ __forceinline__ void write_partial(uint64_t record) const {
    if (!live) return;
    float *const to = p.partial + record * record_size<KIND>(p.q_heads, p.heads, p.D);
    const uint64_t columns = static_cast<uint64_t>(KIND == kBySource ? p.heads : p.q_heads) * p.D;
    store(to + static_cast<uint64_t>(unit) * p.D, s);
    if (KIND != kForward) store(to + columns + static_cast<uint64_t>(unit) * p.D, t);
    if (dl == 0 && slot == 0) {
      if (KIND == kForward) to[columns + unit] = top, to[columns + p.q_heads + unit] = sum;
      if (KIND == kByDestination) to[2u * columns + unit] = sum;
    }
  }
};

__device__ __forceinline__ uint64_t walker_of_grid(const DotArgs &p, uint32_t *pass) {
  const uint64_t w = (static_cast<uint64_t>(blockIdx.x) * 256u + threadIdx.x) >> p.walker_shift;
  *pass = p.passes == 1 ? 0u : static_cast<uint32_t>(w % p.passes);
  return p.passes == 1 ? w : w / p.passes;
}
__device__ __forceinline__ void keep_step(const DotArgs &p) {
  if (p.drop.step_kept && blockIdx.x == 0 && threadIdx.x == 0) *p.drop.step_kept = drop_step(p.drop);
}

// A walker per row.
template <typename T, int ND, int KIND>
__global__ __launch_bounds__(256, (kWavesOf<T, KIND>)) void dot_rows_kernel(DotArgs p) {
  keep_step(p);
  uint32_t pass;
  uint64_t row = walker_of_grid(p, &pass);
  Walk<T, ND, KIND> w(p, pass);
  const uint64_t walkers = (static_cast<uint64_t>(gridDim.x) * 256u >> p.walker_shift) / p.passes;  // whole rounds of passes
  if (row >= walkers) return;
  for (; row < p.rows; row += walkers) {
    const uint32_t first = p.offsets[row], degree = p.offsets[row + 1] - first;
    w.begin(static_cast<uint32_t>(row));
    w.edges(first, 0, degree);
    w.join();
    w.write();
  }
}

template <typename T, int ND, int KIND>
__global__ __launch_bounds__(256, (kWavesOf<T, KIND>)) void dot_spans_kernel(DotArgs p) {
  keep_step(p);
  uint32_t pass;
  const uint64_t span = walker_of_grid(p, &pass);
  if (span >= p.spans) return;
  Walk<T, ND, KIND> w(p, pass);
  const uint64_t begin = span * p.span, end = min(begin + p.span, p.positions);
  const uint32_t co0 = p.offsets[0];
  uint32_t tail = kNoSlot;
  for (uint32_t row = destination_at(p.offsets, co0, p.rows, begin, p.walker_shift); row < p.rows; ++row) {
    const uint32_t first = p.offsets[row], degree = p.offsets[row + 1] - first;
    const uint64_t at = static_cast<uint64_t>(row) * kRowCost + (first - co0), edges_at = at + kRowCost;
    if (at >= end) break;
    const bool cut = degree > p.span;
    if (at < begin && !cut) continue;  // the earlier span has done it
    const uint32_t j0 = edges_at < begin ? static_cast<uint32_t>(min<uint64_t>(begin - edges_at, degree)) : 0u;
    const uint32_t j1 = !cut ? degree : edges_at < end ? static_cast<uint32_t>(min<uint64_t>(degree, end - edges_at)) : 0u;
    if (j0 >= j1 && at < begin) continue;
    w.begin(row);
    w.edges(first, j0, j1);
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

// The rows that were cut: 64 columns a block, its wavefronts take every kJoinWaves-th part, and the first adds up what they have, in
// order.
constexpr uint32_t kJoinWaves = 8, kJoinSpans = 32, kJoinAhead = 8;
template <typename T, int KIND>
__global__ __launch_bounds__(kJoinWaves *kWave) void join_dot_spans_kernel(DotArgs p) {
  __shared__ float tops[kJoinWaves][kWave], sums[kJoinWaves][kWave], accs[kJoinWaves][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block();
  const uint32_t columns = (KIND == kBySource ? 2u * p.heads : p.q_heads) * p.D, c = blockIdx.y * kWave + lane, cc = min(c, columns - 1u), h = cc / p.D;
  const uint64_t size = record_size<KIND>(p.q_heads, p.heads, p.D);
  const uint64_t span0 = static_cast<uint64_t>(blockIdx.x) * kJoinSpans;
  const uint32_t rows = lane < kJoinSpans && span0 + lane < p.spans ? p.tail_row[span0 + lane] : kNoSlot;
  if (__ballot(rows != kNoSlot) == 0) return;  // the same in every wavefront
  // where a record has the three numbers of a column: forward top, sum and weighted sum; by destination none, mean, both sums
  const uint64_t at_a = KIND == kForward ? columns + h : columns + cc, at_b = KIND == kForward ? columns + p.q_heads + h : 2ull * columns + h;
  for (uint32_t k = 0; k < kJoinSpans; ++k) {
    const uint64_t span = span0 + k;
    const uint32_t row = wave_read(rows, k);
    if (row == kNoSlot) continue;
    const uint64_t last_at = static_cast<uint64_t>(row) * kRowCost + (kRowCost - 1u) + (p.offsets[row + 1] - p.offsets[0]);  // its last edge's
    const uint64_t last = min<uint64_t>(last_at / p.span, p.spans - 1u);
    float top = KIND == kForward ? -INFINITY : 0.0f, sum = 0.0f, acc = 0.0f;
    for (uint64_t s = span + wave; s <= last; s += kJoinAhead * kJoinWaves) {
      float t[kJoinAhead], l[kJoinAhead], v[kJoinAhead];
#pragma unroll
      for (uint32_t u = 0; u < kJoinAhead; ++u) {
        const uint64_t part = s + u * kJoinWaves;
        t[u] = KIND == kForward ? -INFINITY : 0.0f, l[u] = v[u] = 0.0f;
        if (part <= last) {
          const float *const record = p.partial + (part * 2u + (part == span ? 1u : 0u)) * size;
          v[u] = record[cc];
          if (KIND != kBySource) t[u] = record[at_a], l[u] = record[at_b];
        }
      }
      if (KIND == kForward) {
        float now = top;
#pragma unroll
        for (uint32_t u = 0; u < kJoinAhead; ++u) now = fmaxf(now, t[u]);
        const float base = now == -INFINITY ? 0.0f : now, f = __builtin_amdgcn_exp2f(top - base);
        top = now;
        sum *= f;
        acc *= f;
#pragma unroll
        for (uint32_t u = 0; u < kJoinAhead; ++u) {
          const float o = __builtin_amdgcn_exp2f(t[u] - base);
          sum = fmaf(l[u], o, sum);
          acc = fmaf(v[u], o, acc);
        }
      } else {
#pragma unroll
        for (uint32_t u = 0; u < kJoinAhead; ++u) top += t[u], sum += l[u], acc += v[u];
      }
    }
    tops[wave][lane] = top, sums[wave][lane] = sum, accs[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < columns) {
      for (uint32_t w = 1; w < kJoinWaves; ++w) {
        if (KIND == kForward) {
          const float t = tops[w][lane], now = fmaxf(top, t), base = now == -INFINITY ? 0.0f : now;
          const float f = __builtin_amdgcn_exp2f(top - base), o = __builtin_amdgcn_exp2f(t - base);
          top = now;
          sum = sum * f + sums[w][lane] * o;
          acc = acc * f + accs[w][lane] * o;
        } else {
          top += tops[w][lane], sum += sums[w][lane], acc += accs[w][lane];
        }
      }
      const uint64_t head = static_cast<uint64_t>(row) * p.q_heads + h;
      if (KIND == kForward) {
        put_value(static_cast<T *>(p.out) + static_cast<uint64_t>(row) * columns + c, sum == 0.0f ? 0.0f : acc / sum);
        if (c == h * p.D) p.lse[head] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
      } else if (KIND == kByDestination) {
        put_value(static_cast<T *>(p.out) + static_cast<uint64_t>(row) * columns + c, fmaf(-sum, top, acc) * p.score_scale);
        if (c == h * p.D) {
          const float l = p.lse[head];
          p.ends[head] = make_float2(l == -INFINITY ? INFINITY : l * kLog2e, sum);
        }
      } else {
        const bool second = c >= columns / 2u;
        put_value(static_cast<T *>(second ? p.out2 : p.out) + static_cast<uint64_t>(row) * (columns / 2u) + (second ? c - columns / 2u : c), acc);
      }
    }
    __syncthreads();
  }
}

constexpr uint32_t kMostHeadWidth = 256, kMostHeads = 1024;
// Above this bound (or without one) a row may be long enough to keep one walker busy after the others are done.
constexpr uint32_t kMostRowEdges = 256;
bool by_spans(uint32_t max_degree) { return max_degree == 0 || max_degree > kMostRowEdges; }

// How the lanes are laid out.  `slot_edges`: edges of a row for each of its slots.
struct Lanes {
  uint32_t nd, hw_shift, walker_shift, passes;
};
Lanes lanes_for(uint32_t units, uint32_t share, uint32_t D, size_t size, uint64_t slot_edges) {
  Lanes l;
  const uint32_t piece = static_cast<uint32_t>(16 / size);
  l.nd = next_power(ceil_div(ceil_div(D, piece), 8 / piece));
  // the query heads of a pass fit a word of the dropout's bits
  uint32_t hw = std::min(kWave / l.nd, next_power(units));
  while (hw > 1 && hw * share > 32u) hw /= 2;
  l.hw_shift = shift_of(hw);
  const uint32_t slots = std::min<uint32_t>(kWave / (l.nd * hw), next_power(static_cast<uint32_t>(std::min<uint64_t>(slot_edges, 64))));
  l.walker_shift = shift_of(l.nd * hw * slots);
  l.passes = ceil_div(units, hw);
  return l;
}

// Positions of a span: 256, so that a part's record is little beside its edges, but spans for all wavefronts that the chip holds
// where there are few positions (none of fewer than 64), and no more spans than fill it four times over or have records of
// 256 MB, but up to 256 spans whatever theirs take.
struct Spans {
  uint64_t positions, count;
  uint32_t length;
  size_t bytes;
};
template <int KIND>
Spans spans_for(uint32_t rows, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t D) {
  Spans s;
  const uint64_t records = 2 * record_size<KIND>(q_heads, heads, D) * sizeof(float);
  s.positions = static_cast<uint64_t>(rows) * kRowCost + edges;
  const uint64_t most = std::max<uint64_t>(256, std::min<uint64_t>(16384, (256ull << 20) / records));
  const uint64_t wanted = std::min(most, std::max<uint64_t>(1024, s.positions / 256));
  s.length = static_cast<uint32_t>(std::max<uint64_t>((s.positions + wanted - 1) / wanted, 64));
  s.count = (s.positions + s.length - 1) / s.length;
  s.bytes = static_cast<size_t>(s.count * (records + sizeof(uint32_t)));
  return s;
}

template <typename T, int ND, int KIND>
int launch(const DotArgs &p, hipStream_t stream) {
  const uint32_t walkers = 256u >> p.walker_shift;  // a block's
  if (!p.span) {
    if (KIND == kBySource) return NTS_OK;  // always in spans
    const uint64_t blocks = std::min<uint64_t>((static_cast<uint64_t>(p.rows) * p.passes + walkers - 1) / walkers, kMostBlocks);
    hipLaunchKernelGGL((dot_rows_kernel<T, ND, KIND == kBySource ? kForward : KIND>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream, p);
    NTS_LAUNCH_CHECK("dot_rows_kernel");
    return NTS_OK;
  }
  hipLaunchKernelGGL((dot_spans_kernel<T, ND, KIND>), dim3(ceil_div(static_cast<uint64_t>(p.spans) * p.passes, walkers)), dim3(256), 0, stream, p);
  NTS_LAUNCH_CHECK("dot_spans_kernel");
  if (p.spans > 1) {  // with one span no row has more edges than it has positions
    const uint64_t columns = static_cast<uint64_t>(KIND == kBySource ? 2 * p.heads : p.q_heads) * p.D;
    hipLaunchKernelGGL((join_dot_spans_kernel<T, KIND>), dim3(ceil_div(p.spans, kJoinSpans), ceil_div(columns, kWave)), dim3(kJoinWaves * kWave), 0,
                       stream, p);
    NTS_LAUNCH_CHECK("join_dot_spans_kernel");
  }
  return NTS_OK;
}
template <typename T, int KIND>
int launch_nd(const DotArgs &p, uint32_t nd, hipStream_t stream) {
  switch (nd) {
    case 1: return launch<T, 1, KIND>(p, stream);
    case 2: return launch<T, 2, KIND>(p, stream);
    case 4: return launch<T, 4, KIND>(p, stream);
    case 8: return launch<T, 8, KIND>(p, stream);
    case 16: return launch<T, 16, KIND>(p, stream);
    default: return launch<T, 32, KIND>(p, stream);
  }
}

// Lays out lanes and spans for `p`, whose operands are set, and runs it.
template <int KIND>
int run(DotArgs p, int type, uint32_t edges, uint32_t max_degree, void *work, hipStream_t stream) {
  if (p.rows == 0) return NTS_OK;
  const size_t size = type_size(type);
  const uint32_t piece = static_cast<uint32_t>(16 / size);
  const bool spans = KIND == kBySource || by_spans(max_degree);
  p.units = KIND == kBySource ? p.heads : p.q_heads;
  const Lanes l = lanes_for(p.units, KIND == kBySource ? p.share : 1u, p.D, size, spans ? (static_cast<uint64_t>(edges) / p.rows + 4) / 4 : (max_degree + 15) / 16);
  p.hw_shift = l.hw_shift, p.walker_shift = l.walker_shift, p.passes = l.passes;
  p.chunks = ceil_div(p.D, piece);
  p.narrow = p.D < piece;
  p.ragged = p.D % piece != 0 || p.chunks != l.nd * (8 / piece);
  if (spans) {
    const Spans s = spans_for<KIND>(p.rows, edges, p.q_heads, p.heads, p.D);
    p.positions = s.positions, p.span = s.length, p.spans = static_cast<uint32_t>(s.count);
    p.partial = static_cast<float *>(work);
    p.tail_row = reinterpret_cast<uint32_t *>(p.partial + s.count * 2 * record_size<KIND>(p.q_heads, p.heads, p.D));
  }
  if (type == NTS_F32) return launch_nd<float, KIND>(p, l.nd, stream);
  return type == NTS_BF16 ? launch_nd<Bf16, KIND>(p, l.nd, stream) : launch_nd<F16, KIND>(p, l.nd, stream);
}

int fail_in(const char *call, const char *why) {
  char text[160];
  snprintf(text, sizeof(text), "%s: %s", call, why);
  return fail(NTS_ERR_INVALID, text);
}

const char *bad_shapes(int type, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t D, const nts_dropout_t *dropout) {
  if (!known_type(type)) return "unknown type";
  if (heads == 0 || q_heads == 0 || q_heads > kMostHeads || q_heads % heads) return "q_heads is no multiple of heads up to 1,024";
  if (D == 0 || D > kMostHeadWidth) return "width is 0 or above 256";
  if (edges > 0xFFFF0000u) return "more than 2^32 - 2^16 edges";
  return bad_dropout(dropout);
}

size_t forward_work(uint32_t Vd, uint32_t edges, uint32_t q_heads, uint32_t D, uint32_t max_degree) {
  return Vd && by_spans(max_degree) ? spans_for<kForward>(Vd, edges, q_heads, q_heads, D).bytes : 0;
}
size_t ends_bytes(uint32_t Vd, uint32_t q_heads) { return (static_cast<size_t>(Vd) * q_heads * sizeof(float2) + 15) / 16 * 16; }

}  // namespace
}  // namespace nts

using namespace nts;

extern "C" {

size_t nts_dot_attention_work_bytes(uint32_t Vd, uint32_t edges, uint32_t q_heads, uint32_t width, uint32_t max_degree) {
  if (q_heads == 0 || q_heads > kMostHeads || width == 0 || width > kMostHeadWidth) return 0;
  return forward_work(Vd, edges, q_heads, width, max_degree);
}

int nts_dot_attention(void *out, float *lse, const void *q, const void *k, const void *v, int type, const uint32_t *co,
                      const uint32_t *ri, uint32_t Vd, uint32_t Vs, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t width,
                      float score_scale, uint32_t max_degree, const nts_dropout_t *dropout, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_dot_attention");
  if (const char *why = bad_shapes(type, edges, q_heads, heads, width, dropout)) return fail_in("nts_dot_attention", why);
  if (Vd == 0) return NTS_OK;
  if (!out || !lse || !q || !co || (edges && !ri) || (edges && Vs && (!k || !v))) return fail_in("nts_dot_attention", "null pointer");
  const size_t size = type_size(type);
  if (!aligned_to(out, size) || !aligned_to(q, size) || !aligned_to(k, size) || !aligned_to(v, size))
    return fail_in("nts_dot_attention", "a value's alignment");
  if (forward_work(Vd, edges, q_heads, width, max_degree) && (!work || !aligned_to(work, 16)))
    return fail_in("nts_dot_attention", "needs nts_dot_attention_work_bytes of 16-byte-aligned work");
  DotArgs p{};
  p.out = out, p.lse = lse, p.q = q, p.k = k, p.v = v, p.offsets = co, p.ids = ri, p.rows = Vd, p.others = Vs;
  p.q_heads = q_heads, p.heads = heads, p.share = q_heads / heads, p.D = width, p.score_scale = score_scale, p.drop = drop_args(dropout);
  return run<kForward>(p, type, edges, max_degree, work, stream);
}

size_t nts_dot_attention_grad_work_bytes(uint32_t Vd, uint32_t Vs, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t width,
                                         uint32_t max_degree) {
  if (q_heads == 0 || q_heads > kMostHeads || heads == 0 || heads > q_heads || width == 0 || width > kMostHeadWidth) return 0;
  const size_t mine = Vd && by_spans(max_degree) ? spans_for<kByDestination>(Vd, edges, q_heads, heads, width).bytes : 0;
  const size_t theirs = Vs ? spans_for<kBySource>(Vs, edges, q_heads, heads, width).bytes : 0;
  return ends_bytes(Vd, q_heads) + std::max(mine, theirs);
}

int nts_dot_attention_grad(void *gq, void *gk, void *gv, const void *g, const void *q, const void *k, const void *v, const float *lse,
                           int type, const uint32_t *co, const uint32_t *ri, const uint32_t *ro, const uint32_t *ci, uint32_t Vd,
                           uint32_t Vs, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t width, float score_scale,
                           uint32_t max_degree, const nts_dropout_t *dropout, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_dot_attention_grad");
  if (const char *why = bad_shapes(type, edges, q_heads, heads, width, dropout)) return fail_in("nts_dot_attention_grad", why);
  if (Vd == 0 && Vs == 0) return NTS_OK;
  if ((Vd && (!gq || !g || !q || !lse || !co)) || (Vs && (!gk || !gv || !k || !v || !ro)) || (edges && Vd && !ri) || (edges && Vs && !ci))
    return fail_in("nts_dot_attention_grad", "null pointer");
  const size_t size = type_size(type);
  for (const void *at : {static_cast<const void *>(gq), static_cast<const void *>(gk), static_cast<const void *>(gv), g, q, k, v})
    if (!aligned_to(at, size)) return fail_in("nts_dot_attention_grad", "a value's alignment");
  if (!work || !aligned_to(work, 16)) return fail_in("nts_dot_attention_grad", "needs nts_dot_attention_grad_work_bytes of 16-byte-aligned work");
  DotArgs p{};
  p.lse = const_cast<float *>(lse), p.ends = static_cast<float2 *>(work), p.q = q, p.k = k, p.v = v, p.g = g;
  p.q_heads = q_heads, p.heads = heads, p.share = q_heads / heads, p.D = width, p.score_scale = score_scale, p.drop = drop_args(dropout);
  p.drop.step_kept = nullptr;
  void *const rest = static_cast<char *>(work) + ends_bytes(Vd, q_heads);
  p.out = gq, p.offsets = co, p.ids = ri, p.rows = Vd, p.others = Vs;
  if (const int status = run<kByDestination>(p, type, edges, max_degree, rest, stream)) return status;
  p.out = gk, p.out2 = gv, p.offsets = ro, p.ids = ci, p.rows = Vs, p.others = Vd;
  return run<kBySource>(p, type, edges, 0, rest, stream);
}

}  // extern "C"
