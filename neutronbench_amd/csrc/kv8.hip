// Keys and values of vertices in 8 bits (e4m3) with a scale (e8m0) for each block of vertices, each head and each of the
// two, and every destination's attention over its neighbours' rows of that cache.
//   cache   [capacity, 2, heads, row width] bytes, keys before values; the row width is the head's rounded up to 16
//   scales  [ceil(capacity / block_rows), 2, heads]
#include <algorithm>

#include "launch_size.hpp"
#include "lowbit.hpp"

namespace nts {
namespace {

// ---- writing rows -----------------------------------------------------------------------------------
// A wavefront takes one block of rows, one of keys and values and one head: the largest finite magnitude first, then the codes.
// The scale is the smallest power of two with max <= 448 * scale, so every value lies within e4m3's range.  Rows of the block
// that were there before `first` keep their place: the scale is at least theirs, and they are rounded once more where it grew
// (exactly, unless the value falls among e4m3's subnormals).
struct AppendArgs {
  uint8_t *cache;
  uint8_t *scales;
  const float *k, *v;
  uint32_t first, n, heads, D, quads;  // quads = row width / 4
  uint32_t block_rows, first_block;
  uint64_t units;
};

__device__ __forceinline__ void append_values(const AppendArgs &p, const float *src, const uint8_t *held, float held_scale,
                                              uint32_t row, uint32_t quad, float *v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = 0.0f;
  const uint32_t col = quad * 4u;
  if (row < p.first) {
    e4m3_decode4(*reinterpret_cast<const uint32_t *>(held + static_cast<uint64_t>(row) * 2u * p.heads * p.quads * 4u + col), v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= held_scale;
    return;
  }
  const float *at = src + static_cast<uint64_t>(row - p.first) * p.heads * p.D + col;
  if (col + 4u <= p.D) {
    const FloatQuad q = *reinterpret_cast<const FloatQuad *>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q[i];
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
      if (col + i < p.D) v[i] = at[i];
  }
}

// Bound by memory and by vector instructions, which are under way all of the time: 2.45 M rows of 4 heads of 32, blocks of 16, 563 us
// after other work, 5.6 TB/s of floats read and bytes written; 603 one after the other.  Read twice, the second time from the
// caches: 712.
// HELD: blocks of at most 64 * HELD quads, which the lanes hold between the passes; 0: of any size, read twice.
template <int HELD>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs p) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const uint64_t waves = static_cast<uint64_t>(gridDim.x) * (256 / kWave);
  for (uint64_t u = wave_of_grid(); u < p.units; u += waves) {
    const uint32_t head = static_cast<uint32_t>(u % p.heads), side = static_cast<uint32_t>(u / p.heads % 2u);
    const uint64_t block = p.first_block + u / (2u * p.heads);
    const uint64_t row0 = block * p.block_rows;
    const uint32_t rows = static_cast<uint32_t>(min(static_cast<uint64_t>(p.block_rows), static_cast<uint64_t>(p.first) + p.n - row0));
    const float *src = (side ? p.v : p.k) + head * p.D;
    uint8_t *held = p.cache + (side * p.heads + head) * p.quads * 4u;
    uint8_t *scale = p.scales + (block * 2u + side) * p.heads + head;
    const bool keeps = row0 < p.first;
    const uint32_t old = keeps ? *scale : 0u;
    const float held_scale = e8m0_value(old);
    const uint32_t total = rows * p.quads;
    uint32_t top = 0;
    auto largest = [&](const float *v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        if (b < 0x7F800000u) top = max(top, b);
      }
    };
    float kept[HELD ? HELD : 1][4];
    if (HELD) {
#pragma unroll
      for (uint32_t k = 0; k < HELD; ++k) {
        const uint32_t j = k * kWave + lane, r = j / p.quads;
#pragma unroll
        for (int i = 0; i < 4; ++i) kept[k][i] = 0.0f;
        if (j < total) append_values(p, src, held, held_scale, static_cast<uint32_t>(row0) + r, j - r * p.quads, kept[k]);
      }
#pragma unroll
      for (uint32_t k = 0; k < HELD; ++k) largest(kept[k]);
    } else {
      for (uint32_t j = lane; j < total; j += kWave) {
        const uint32_t r = j / p.quads;
        float v[4];
        append_values(p, src, held, held_scale, static_cast<uint32_t>(row0) + r, j - r * p.quads, v);
        largest(v);
      }
    }
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, kWave)));
    // 448 = 1.75 * 2^8
    const uint32_t up = (top >> 23) + ((top & 0x7FFFFFu) > 0x600000u ? 1u : 0u);
    const uint32_t byte = max(old, up > 8u ? up - 8u : 0u);
    // 2^-127 and 2^-128, which only rows from elsewhere can ask for, lie below the normal floats
    const float inverse = byte < 254u ? e8m0_inverse(byte) : __uint_as_float(0x00400000u >> (byte - 254u));
    auto put = [&](uint32_t j, float *v) {
      const uint32_t r = j / p.quads;
      const uint32_t row = static_cast<uint32_t>(row0) + r, quad = j - r * p.quads;
      if (row < p.first && byte == old) return;
      if (!HELD) append_values(p, src, held, held_scale, row, quad, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] *= inverse;
      *reinterpret_cast<uint32_t *>(held + static_cast<uint64_t>(row) * 2u * p.heads * p.quads * 4u + quad * 4u) = e4m3_encode4(v);
    };
    if (HELD) {
#pragma unroll
      for (uint32_t k = 0; k < HELD; ++k)
        if (k * kWave + lane < total) put(k * kWave + lane, kept[k]);
    } else {
      float v[4];
      for (uint32_t j = lane; j < total; j += kWave) put(j, v);
    }
    if (lane == 0) *scale = static_cast<uint8_t>(byte);
  }
}

// ---- attention --------------------------------------------------------------------------------------
//   s_e = score_scale * q[d, h] . K[src(e), h'],  p_e = exp(s_e - max s),  out[d, h, :] = sum_e p_e V[src(e), h'] / sum_e p_e
// for the edges e of destination d whose source is cached; h' = h / (q_heads / heads).  One pass: the running maximum, sum
// and weighted sum of values stay in registers and are rescaled when the maximum grows.
//
// A lane holds 16 columns of G query heads that share a head of the cache ("unit"): one 16-byte load of a key row and one of a
// value row serve them.  ND lanes (a power of two) cover a unit, 2^hw_shift units lie side by side, and further edges of the
// destination go to further such sets of lanes ("slots"), each with a running softmax of its own, joined at the end.  All slots of
// one destination are a walker; a wavefront is one walker or, where rows are short, several.
// 2.48 M edges of 169,343 destinations, 8 query heads on 2 of 64: 394 us after other work, of which some 29 in the join; that is 1.3 GB of
// rows, queries and results at 3.6 TB/s in the walkers.  Bound by vector instructions (64 % of the time; without reading rows 333 us when
// the whole took 392): 48 a lane and edge to convert and multiply 16 columns of a key and a value, about as many again to look up,
// scale, rescale, join and write.
struct AttendArgs {
  float *out, *lse;
  const float *q;
  const uint8_t *cache, *scales;
  const uint32_t *co, *ri, *mirror;
  uint32_t mirror_rows;  // entries of mirror: an id beyond them names no row
  uint32_t Vd, cache_rows, q_heads, heads, D, row_width, block_shift;
  uint32_t share;             // query heads per head of the cache
  uint32_t units, per_head;   // units in all and of a head
  uint32_t passes;            // over the edges, 2^hw_shift units each; neighbouring wavefronts take the passes of one walker
  uint32_t hw_shift, walker_shift;  // log2 of units side by side, of a walker's lanes
  float score_scale;
  bool blocks;  // a block per destination
  // edges cut into spans of `span` positions (see below)
  uint32_t span, spans;
  uint64_t positions;
  float *partial;
  uint32_t *tail_row;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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
  return v;
}

// What the registers allow, measured: with one query head to a lane four wavefronts to a SIMD (2.48 M edges, 8 query heads of 64: 468 us at
// the time; three 507, two edges at a time 600); with two, two wavefronts (500 K edges, 16 query heads of 128: 205 us; three and two
// edges at a time 227, one head to a lane 259; but 2.48 M ragged edges 1,355 against 1,330).  Four heads to a lane leave one.
template <int G>
constexpr int kWavesOf = G == 1 ? 4 : 2;

// NEAR: cache and scales of less than 4 GB each and of at most 2^24 rows are read through buffer descriptors: 32-bit offsets from
// 24-bit products, and a row that is not there gets an offset beyond the end, which reads zeros without a branch.
template <int ND, int G, bool NEAR, int AHEAD = 4>
struct Attend {
  const AttendArgs &p;
  uint32_t dl, kv_head, q_head0, slot, rounds;
  uint32_t lane_edge, edge_step;  // the lane's first edge of a destination, and how far its next one lies behind it
  bool live;  // this lane has a unit and columns
  uint32_t key_at, row_bytes, values_at;  // the lane's 16 bytes of a row's keys; from there to its values
  __amdgpu_buffer_rsrc_t keys, values, key_scales, value_scales;
  float q[G][16], acc[G][16], top[G], sum[G];
  uint32_t col;  // the first of the lane's columns; fewer than 16 of them after join()

  __device__ __forceinline__ Attend(const AttendArgs &args, uint32_t pass) : p(args) {
    constexpr uint32_t kShift = ND == 1 ? 0 : ND == 2 ? 1 : ND == 4 ? 2 : ND == 8 ? 3 : 4;
    const uint32_t l = threadIdx.x & ((1u << p.walker_shift) - 1u);
    dl = l & (ND - 1);
    const uint32_t unit = (pass << p.hw_shift) + ((l >> kShift) & ((1u << p.hw_shift) - 1u));
    rounds = p.walker_shift - p.hw_shift - kShift;
    slot = l >> (kShift + p.hw_shift);
    lane_edge = slot;
    edge_step = 1u << rounds;
    live = unit < p.units && dl * 16u < p.row_width;
    kv_head = unit / p.per_head;
    q_head0 = (unit - kv_head * p.per_head) * G;  // within the head's share
    row_bytes = 2u * p.heads * p.row_width;
    values_at = p.heads * p.row_width;
    key_at = kv_head * p.row_width + dl * 16u;
    if (NEAR) {
      const uint32_t blocks = p.cache_rows ? ((p.cache_rows - 1u) >> p.block_shift) + 1u : 0u;
      // one for keys and one for values, so that an offset is one register and one behind the end stays there
      uint8_t *const cache = const_cast<uint8_t *>(p.cache), *const scales = const_cast<uint8_t *>(p.scales);
      const uint32_t bytes = p.cache_rows * row_bytes, scales_bytes = blocks * 2u * p.heads;
      keys = __builtin_amdgcn_make_buffer_rsrc(cache, 0, bytes, 0x00027000);
      values = __builtin_amdgcn_make_buffer_rsrc(cache + values_at, 0, bytes ? bytes - values_at : 0u, 0x00027000);
      key_scales = __builtin_amdgcn_make_buffer_rsrc(scales, 0, scales_bytes, 0x00027000);
      value_scales = __builtin_amdgcn_make_buffer_rsrc(scales + p.heads, 0, scales_bytes ? scales_bytes - p.heads : 0u, 0x00027000);
    }
  }

  __device__ __forceinline__ void begin(uint32_t row) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      top[g] = -INFINITY;
      sum[g] = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[g][i] = q[g][i] = 0.0f;
      if (live && q_head0 + g < p.share) {
        const float *src = p.q + (static_cast<uint64_t>(row) * p.q_heads + kv_head * p.share + q_head0 + g) * p.D + dl * 16u;
        if (dl * 16u + 16u <= p.D) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const FloatQuad four = *reinterpret_cast<const FloatQuad *>(src + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) q[g][i + k] = four[k];
          }
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 15; ++i)
            if (dl * 16u + i < p.D) q[g][i] = src[i];
        }
      }
    }
  }

  // The cache row of edge j, or a row that no cache has for an edge behind the last.
  __device__ __forceinline__ uint32_t cache_row(const uint32_t *ids, uint32_t j, uint32_t j1) const {
    uint32_t r = ids[min(j, j1 - 1u)];
    bool there = j < j1;
    if (p.mirror) {
      // Without a branch: an id beyond the mirror reads its first entry (20,000 rows of 25 edges, 16 query heads on 4 of 128: 212 us;
      // with one 240, without a look at the length 208).
      there = there && r < p.mirror_rows;
      r = p.mirror[there ? r : 0u];
    }
    return there ? r : 0xFFFFFFFFu;
  }

  // Edges of a slot whose rows are requested together: AHEAD, 2 or 4.
  static constexpr int kAhead = AHEAD;
  template <int U>
  __device__ __forceinline__ void step(const uint32_t *row) {
    u32x4 kc[U], vc[U];
    uint32_t kb[U], vb[U];
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      there[u] = row[u] < p.cache_rows;
      if (NEAR) {
        const bool read = there[u] && live;
        const uint32_t at = read ? __umul24(row[u], row_bytes) + key_at : 0xFFFFFF00u;
        const uint32_t scale_at = read ? __umul24(row[u] >> p.block_shift, 2u * p.heads) + kv_head : 0xFFFFFF00u;
        kc[u] = __builtin_amdgcn_raw_buffer_load_b128(keys, at, 0, 0);
        vc[u] = __builtin_amdgcn_raw_buffer_load_b128(values, at, 0, 0);
        kb[u] = __builtin_amdgcn_raw_buffer_load_b8(key_scales, scale_at, 0, 0);
        vb[u] = __builtin_amdgcn_raw_buffer_load_b8(value_scales, scale_at, 0, 0);
      } else {
        kc[u] = vc[u] = u32x4{0, 0, 0, 0};
        kb[u] = vb[u] = 0;
        if (there[u] && live) {
          const uint8_t *at = p.cache + static_cast<uint64_t>(row[u]) * row_bytes + key_at;
          kc[u] = *reinterpret_cast<const u32x4 *>(at);
          vc[u] = *reinterpret_cast<const u32x4 *>(at + values_at);
          const uint8_t *s = p.scales + static_cast<uint64_t>(row[u] >> p.block_shift) * 2u * p.heads + kv_head;
          kb[u] = s[0];
          vb[u] = s[p.heads];
        }
      }
    }
    const float unit = p.score_scale * kLog2e;
    float s[G][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float k[16];
      e4m3_decode4(kc[u][0], k), e4m3_decode4(kc[u][1], k + 4), e4m3_decode4(kc[u][2], k + 8), e4m3_decode4(kc[u][3], k + 12);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) dot = fmaf(q[g][i], k[i], dot);
        dot = __builtin_amdgcn_ldexpf(lanes_sum<ND>(dot) * unit, static_cast<int>(kb[u]) - 127);
        s[g][u] = there[u] ? dot : -INFINITY;
      }
    }
    float base[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float now = top[g];
#pragma unroll
      for (int u = 0; u < U; ++u) now = fmaxf(now, s[g][u]);
      base[g] = now == -INFINITY ? 0.0f : now;
      const float keep = __builtin_amdgcn_exp2f(top[g] - base[g]);
      top[g] = now;
      sum[g] *= keep;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[g][i] *= keep;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[16];
      e4m3_decode4(vc[u][0], v), e4m3_decode4(vc[u][1], v + 4), e4m3_decode4(vc[u][2], v + 8), e4m3_decode4(vc[u][3], v + 12);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float w = __builtin_amdgcn_exp2f(s[g][u] - base[g]);
        sum[g] += w;
        const float wv = __builtin_amdgcn_ldexpf(w, static_cast<int>(vb[u]) - 127);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[g][i] = fmaf(wv, v[i], acc[g][i]);
      }
    }
  }

  // Edges [j0, j1) of the destination whose edges begin at `first`; the next step's rows are looked up ahead.
  __device__ __forceinline__ void edges(uint32_t first, uint32_t j0, uint32_t j1) {
    if (j0 >= j1) return;
    const uint32_t *ids = p.ri + first;
    uint32_t row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) row[u] = cache_row(ids, j0 + u * edge_step + lane_edge, j1);
    uint32_t j = j0;
    for (; j1 - j > kAhead * edge_step; j += kAhead * edge_step) {
      uint32_t next[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) next[u] = cache_row(ids, j + (kAhead + u) * edge_step + lane_edge, j1);
      step<kAhead>(row);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) row[u] = next[u];
    }
    if (j1 - j > kAhead / 2 * edge_step)
      step<kAhead>(row);
    else if (kAhead == 2 || j1 - j <= edge_step)
      step<1>(row);
    else
      step<2>(row);
  }

  // Joins the slots.  Each round halves a lane's columns: it hands one half to the lane of the other slot and takes in that one's
  // part of its own half, so 16 columns and 2^r slots take 8 + 4 + .. exchanges instead of 16 a round.
  __device__ __forceinline__ void join() {
    col = dl * 16u;
    const uint32_t lanes = 1u << (p.walker_shift - rounds);
#pragma unroll
    for (uint32_t r = 0; r < 6; ++r) {
      if (r >= rounds) break;
      const uint32_t m = lanes << r;
      const int half = r < 4 ? 8 >> r : 0;
      const bool upper = (slot >> r) & 1u;
      if (half && upper) col += half;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float other = __shfl_xor(top[g], m, kWave), more = __shfl_xor(sum[g], m, kWave);
        const float now = fmaxf(top[g], other), base = now == -INFINITY ? 0.0f : now;
        const float a = __builtin_amdgcn_exp2f(top[g] - base), b = __builtin_amdgcn_exp2f(other - base);
        top[g] = now;
        // both sides of the exchange add in the same order: the lower slot's part first
        sum[g] = upper ? more * b + sum[g] * a : sum[g] * a + more * b;
        if (half) {
#pragma unroll
          for (int i = 0; i < (half ? half : 1); ++i) {
            const float mine = upper ? acc[g][i + half] : acc[g][i], give = upper ? acc[g][i] : acc[g][i + half];
            acc[g][i] = mine * a + __shfl_xor(give, m, kWave) * b;
          }
        } else {
          acc[g][0] = acc[g][0] * a + __shfl_xor(acc[g][0], m, kWave) * b;
        }
      }
    }
  }

  // A lane's columns after join(), times `factor`, to a row of `columns`.
  __device__ __forceinline__ void store(float *dst, int g, float factor, uint32_t columns) const {
    const uint32_t count = rounds < 4 ? 16u >> rounds : 1u;
    if (slot >> 4) return;  // further slots hold the same columns
#pragma unroll
    for (uint32_t i = 0; i < 16; i += 4) {
      if (i >= count) break;
      if (count >= 4 && col + i + 4u <= columns) {
        *reinterpret_cast<FloatQuad *>(dst + col + i) = FloatQuad{acc[g][i] * factor, acc[g][i + 1] * factor, acc[g][i + 2] * factor, acc[g][i + 3] * factor};
      } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
          if (i + k < count && col + i + k < columns) dst[col + i + k] = acc[g][i + k] * factor;
      }
    }
  }

  __device__ __forceinline__ void write(uint32_t row) const {
    if (!live) return;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (q_head0 + g >= p.share) continue;
      const uint64_t at = static_cast<uint64_t>(row) * p.q_heads + kv_head * p.share + q_head0 + g;
      // the reciprocal is within one step of 32 bits, and its product another half; divided correctly 418 us instead of 415 (the
      // edges above, one call after the other)
      store(p.out + at * p.D, g, sum[g] == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum[g]), p.D);
      if (p.lse && dl == 0 && slot == 0) p.lse[at] = sum[g] == 0.0f ? -INFINITY : (top[g] + __builtin_amdgcn_logf(sum[g])) * kLn2;
    }
  }

  // A part of a destination's edges: top, sum and weighted sums of every query head, for join_spans_kernel.
  __device__ __forceinline__ void write_partial(uint64_t record) const {
    if (!live) return;
    float *dst = p.partial + record * p.q_heads * (p.D + 2u);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (q_head0 + g >= p.share) continue;
      const uint32_t h = kv_head * p.share + q_head0 + g;
      store(dst + static_cast<uint64_t>(h) * p.D, g, 1.0f, p.D);
      if (dl == 0 && slot == 0) {
        dst[static_cast<uint64_t>(p.q_heads) * p.D + h] = top[g];
        dst[static_cast<uint64_t>(p.q_heads) * (p.D + 1u) + h] = sum[g];
      }
    }
  }
};

__device__ __forceinline__ uint64_t walker_of_grid(const AttendArgs &p, uint32_t *pass) {
  const uint64_t w = (static_cast<uint64_t>(blockIdx.x) * 256u + threadIdx.x) >> p.walker_shift;
  *pass = p.passes == 1 ? 0u : static_cast<uint32_t>(w % p.passes);
  return p.passes == 1 ? w : w / p.passes;
}

// A walker per destination.
template <int ND, int G, bool NEAR>
__global__ __launch_bounds__(256, kWavesOf<G>) void kv8_attend_rows_kernel(AttendArgs p) {
  uint32_t pass;
  uint64_t row = walker_of_grid(p, &pass);
  Attend<ND, G, NEAR> a(p, pass);
  const uint64_t walkers = (static_cast<uint64_t>(gridDim.x) * 256u >> p.walker_shift) / p.passes;  // whole rounds of passes
  if (row >= walkers) return;
  for (; row < p.Vd; row += walkers) {
    const uint32_t first = p.co[row], degree = p.co[row + 1] - first;
    a.begin(static_cast<uint32_t>(row));
    a.edges(first, 0, degree);
    a.join();
    a.write(static_cast<uint32_t>(row));
  }
}

// A block per destination, for few destinations of up to some thousand edges: its wavefronts share the edges and join through
// LDS, in one launch (one vertex with 300 neighbours: 6 us on the device, where spans and their join take 13).
constexpr uint32_t kBlockWaves = 16;
template <int ND, int G, bool NEAR>
__global__ __launch_bounds__(kBlockWaves *kWave) void kv8_attend_block_kernel(AttendArgs p) {
  __shared__ float tops[kBlockWaves * kWave * G / ND], sums[kBlockWaves * kWave * G / ND], accs[kBlockWaves * kWave * 16 * G];
  const uint32_t row = blockIdx.x / p.passes, pass = blockIdx.x - row * p.passes, wave = wave_of_block();
  const uint32_t hw = 1u << p.hw_shift, first = p.co[row], degree = p.co[row + 1] - first;
  {
    Attend<ND, G, NEAR, G == 1 ? 4 : 2> a(p, pass);  // what 128 registers hold
    a.lane_edge += wave * a.edge_step;
    a.edge_step *= kBlockWaves;
    a.begin(row);
    a.edges(first, 0, degree);
    a.join();
    if (a.live) {
      const uint32_t unit = (threadIdx.x & (kWave - 1)) / ND % hw;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t at = (wave * hw + unit) * G + g;
        a.store(accs + at * (ND * 16u), g, 1.0f, ND * 16u);
        if (a.dl == 0 && a.slot == 0) {
          tops[at] = a.top[g];
          sums[at] = a.sum[g];
        }
      }
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < hw * G * ND * 16u; i += kBlockWaves * kWave) {
    const uint32_t at = i / (ND * 16u), c = i % (ND * 16u), unit = pass * hw + at / G;
    const uint32_t kv_head = unit / p.per_head, q_head = (unit - kv_head * p.per_head) * G + at % G;
    if (unit >= p.units || c >= p.D || q_head >= p.share) continue;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kBlockWaves; ++w) top = fmaxf(top, tops[w * hw * G + at]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (uint32_t w = 0; w < kBlockWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(tops[w * hw * G + at] - base);
      sum = fmaf(sums[w * hw * G + at], f, sum);
      acc = fmaf(accs[(w * hw * G + at) * (ND * 16u) + c], f, acc);
    }
    const uint64_t h = static_cast<uint64_t>(row) * p.q_heads + kv_head * p.share + q_head;
    p.out[h * p.D + c] = sum == 0.0f ? 0.0f : acc / sum;
    if (p.lse && c == 0) p.lse[h] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

// Long rows are shared out and short ones bundled without a look at the degrees on the host: destinations and edges are
// lined up -- destination r takes kRowCost positions from r * kRowCost + co[r] - co[0] on, which is what beginning and writing a
// row costs in edges, and its edges the positions behind them -- and every walker takes the destinations that begin within its
// span of `span` positions.  A destination of more than `span` edges is cut at the spans' ends: every span that it reaches into
// sums its part into a record (1: the destination begins in this span, 0: in an earlier one) and join_spans_kernel adds the
// parts in order.  No atomics: the same bits on every call.
constexpr uint32_t kRowCost = 8;  // 2.48 M edges in 169 K rows, 4 heads of 32: 194 us when chosen (201 now); 4: 209, 16: 192, 1: 230
__device__ __forceinline__ uint64_t position_of(const uint32_t *co, uint32_t co0, uint64_t r) { return r * kRowCost + (co[r] - co0); }

// The last destination at or before position x: a candidate for every lane of the walker a step.
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

template <int ND, int G, bool NEAR>
__global__ __launch_bounds__(256, kWavesOf<G>) void kv8_attend_spans_kernel(AttendArgs p) {
  uint32_t pass;
  const uint64_t span = walker_of_grid(p, &pass);
  if (span >= p.spans) return;
  Attend<ND, G, NEAR> a(p, pass);
  const uint64_t begin = span * p.span, end = min(begin + p.span, p.positions);
  const uint32_t co0 = p.co[0];
  uint32_t tail = kNoSlot;
  for (uint32_t row = destination_at(p.co, co0, p.Vd, begin, p.walker_shift); row < p.Vd; ++row) {
    const uint32_t first = p.co[row], degree = p.co[row + 1] - first;
    const uint64_t at = static_cast<uint64_t>(row) * kRowCost + (first - co0), edges_at = at + kRowCost;
    if (at >= end) break;
    const bool cut = degree > p.span;
    if (at < begin && !cut) continue;  // the earlier span has done it
    const uint32_t j0 = edges_at < begin ? static_cast<uint32_t>(min<uint64_t>(begin - edges_at, degree)) : 0u;
    const uint32_t j1 = !cut ? degree : edges_at < end ? static_cast<uint32_t>(min<uint64_t>(degree, end - edges_at)) : 0u;
    if (j0 >= j1 && at < begin) continue;
    a.begin(row);
    a.edges(first, j0, j1);
    a.join();
    if (!cut) {
      a.write(row);
      continue;
    }
    a.write_partial(span * 2u + (at < begin ? 0u : 1u));
    if (at >= begin) tail = row;
  }
  if (pass == 0 && (threadIdx.x & ((1u << p.walker_shift) - 1u)) == 0) p.tail_row[span] = tail;
}

// The destinations that were cut: 64 columns a block, its wavefronts take every kJoinWaves-th part, and the first adds up
// what they have, in order.
constexpr uint32_t kJoinWaves = 8, kJoinSpans = 32, kJoinAhead = 16;
__global__ __launch_bounds__(kJoinWaves *kWave) void join_spans_kernel(AttendArgs p) {
  __shared__ float tops[kJoinWaves][kWave], sums[kJoinWaves][kWave], accs[kJoinWaves][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block();
  const uint32_t columns = p.q_heads * p.D, c = blockIdx.y * kWave + lane, h = min(c, columns - 1u) / p.D;
  const uint64_t size = static_cast<uint64_t>(p.q_heads) * (p.D + 2u);
  const uint64_t span0 = static_cast<uint64_t>(blockIdx.x) * kJoinSpans;
  const uint32_t rows = lane < kJoinSpans && span0 + lane < p.spans ? p.tail_row[span0 + lane] : kNoSlot;
  if (__ballot(rows != kNoSlot) == 0) return;  // the same in every wavefront
  for (uint32_t k = 0; k < kJoinSpans; ++k) {
    const uint64_t span = span0 + k;
    const uint32_t row = wave_read(rows, k);
    if (row == kNoSlot) continue;
    const uint64_t last_at = static_cast<uint64_t>(row) * kRowCost + (kRowCost - 1u) + (p.co[row + 1] - p.co[0]);  // its last edge's
    const uint64_t last = min<uint64_t>(last_at / p.span, p.spans - 1u);
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
    const float *const from = p.partial + min(c, columns - 1u);
    for (uint64_t s = span + wave; s <= last; s += kJoinAhead * kJoinWaves) {
      float t[kJoinAhead], l[kJoinAhead], v[kJoinAhead];
#pragma unroll
      for (uint32_t u = 0; u < kJoinAhead; ++u) {
        const uint64_t at = s + u * kJoinWaves;
        t[u] = -INFINITY, l[u] = v[u] = 0.0f;
        if (at <= last) {
          const uint64_t record = (at * 2u + (at == span ? 1u : 0u)) * size;
          t[u] = p.partial[record + columns + h];
          l[u] = p.partial[record + columns + p.q_heads + h];
          v[u] = from[record];
        }
      }
      float now = top;
#pragma unroll
      for (uint32_t u = 0; u < kJoinAhead; ++u) now = fmaxf(now, t[u]);
      const float base = now == -INFINITY ? 0.0f : now, a = __builtin_amdgcn_exp2f(top - base);
      top = now;
      sum *= a;
      acc *= a;
#pragma unroll
      for (uint32_t u = 0; u < kJoinAhead; ++u) {
        const float b = __builtin_amdgcn_exp2f(t[u] - base);
        sum = fmaf(l[u], b, sum);
        acc = fmaf(v[u], b, acc);
      }
    }
    tops[wave][lane] = top, sums[wave][lane] = sum, accs[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < columns) {
      for (uint32_t w = 1; w < kJoinWaves; ++w) {
        const float t = tops[w][lane], now = fmaxf(top, t), base = now == -INFINITY ? 0.0f : now;
        const float a = __builtin_amdgcn_exp2f(top - base), b = __builtin_amdgcn_exp2f(t - base);
        top = now;
        sum = sum * a + sums[w][lane] * b;
        acc = acc * a + accs[w][lane] * b;
      }
      p.out[static_cast<uint64_t>(row) * columns + c] = sum == 0.0f ? 0.0f : acc / sum;
      if (p.lse && c == h * p.D)
        p.lse[static_cast<uint64_t>(row) * p.q_heads + h] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    }
    __syncthreads();
  }
}

constexpr uint32_t kMostHeadWidth = 256, kMostHeads = 1024, kMostBlockRows = 1024;
// Above this bound (or without one) a row may be long enough to keep one walker busy after the others are done.
constexpr uint32_t kMostRowEdges = 256;
// Up to so many destinations and edges a block takes a destination, whatever the degrees.
constexpr uint32_t kBlockRows = 64, kBlockEdges = 4096;
bool by_blocks(uint32_t Vd, uint32_t edges, uint32_t max_degree) {
  return Vd <= kBlockRows && edges <= kBlockEdges && (max_degree == 0 || max_degree > 16);
}
bool by_spans(uint32_t Vd, uint32_t edges, uint32_t max_degree) {
  return !by_blocks(Vd, edges, max_degree) && (max_degree == 0 || max_degree > kMostRowEdges);
}

uint32_t next_power(uint32_t v) {
  uint32_t p = 1;
  while (p < v) p <<= 1;
  return p;
}
uint32_t shift_of(uint32_t power) { return static_cast<uint32_t>(__builtin_ctz(power)); }

// How the lanes are laid out.  `slot_edges`: edges of a row for each of its slots.
struct Lanes {
  uint32_t nd, g, units, per_head, hw_shift, walker_shift;
};
Lanes lanes_for(uint32_t q_heads, uint32_t heads, uint32_t D, uint64_t slot_edges) {
  Lanes l;
  const uint32_t share = q_heads / heads;
  l.nd = next_power(kv8_row_width(D) / 16);
  // Query heads of a head side by side as long as all fit a wavefront (their loads of the same row meet in the L1, and few
  // registers leave many wavefronts); two to a lane where the edges would have to be walked more than once.
  l.g = share > 1 && l.nd * heads * share > static_cast<uint32_t>(kWave) ? 2 : 1;
  l.per_head = ceil_div(share, l.g);
  l.units = heads * l.per_head;
  const uint32_t hw = std::min(kWave / l.nd, next_power(l.units));
  l.hw_shift = shift_of(hw);
  const uint32_t slots = std::min<uint32_t>(kWave / (l.nd * hw), next_power(static_cast<uint32_t>(std::min<uint64_t>(slot_edges, 64))));
  l.walker_shift = shift_of(l.nd * hw * slots);
  return l;
}

// Bytes of a span's two records.
uint64_t records_bytes(uint32_t q_heads, uint32_t D) { return 2ull * q_heads * (D + 2u) * sizeof(float); }
// Positions of a span: 256, so that a part's record is little beside its edges, but spans for all wavefronts that the chip holds
// where there are few positions (none of fewer than 64), and no more spans than fill it four times over or have records of
// 256 MB, but up to 256 spans whatever theirs take (of 1,024 heads of 256: 516 MB).
uint32_t span_length(uint64_t positions, uint32_t q_heads, uint32_t D) {
  const uint64_t most = std::max<uint64_t>(256, std::min<uint64_t>(16384, (256ull << 20) / records_bytes(q_heads, D)));
  const uint64_t spans = std::min(most, std::max<uint64_t>(1024, positions / 256));
  const uint64_t wanted = (positions + spans - 1) / spans;
  return static_cast<uint32_t>(std::max<uint64_t>(wanted, 64));
}

template <int ND, int G, bool NEAR>
int launch_attend(const AttendArgs &p, hipStream_t stream) {
  if (p.blocks) {
    hipLaunchKernelGGL((kv8_attend_block_kernel<ND, G, NEAR>), dim3(p.Vd * p.passes), dim3(kBlockWaves * kWave), 0, stream, p);
    NTS_LAUNCH_CHECK("nts_kv8_attention");
    return NTS_OK;
  }
  const uint32_t walkers = 256u >> p.walker_shift;  // a block's
  if (!p.span) {
    const uint64_t blocks = std::min<uint64_t>((static_cast<uint64_t>(p.Vd) * p.passes + walkers - 1) / walkers, kMostBlocks);
    hipLaunchKernelGGL((kv8_attend_rows_kernel<ND, G, NEAR>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream, p);
    NTS_LAUNCH_CHECK("nts_kv8_attention");
    return NTS_OK;
  }
  hipLaunchKernelGGL((kv8_attend_spans_kernel<ND, G, NEAR>), dim3(ceil_div(static_cast<uint64_t>(p.spans) * p.passes, walkers)), dim3(256), 0, stream, p);
  NTS_LAUNCH_CHECK("nts_kv8_attention");
  if (p.spans > 1) {  // with one span no destination has more edges than it has positions
    hipLaunchKernelGGL(join_spans_kernel, dim3(ceil_div(p.spans, kJoinSpans), ceil_div(static_cast<uint64_t>(p.q_heads) * p.D, kWave)),
                       dim3(kJoinWaves * kWave), 0, stream, p);
    NTS_LAUNCH_CHECK("join_spans_kernel");
  }
  return NTS_OK;
}
template <int ND, bool NEAR>
int launch_attend_g(const AttendArgs &p, uint32_t g, hipStream_t stream) {
  return g == 1 ? launch_attend<ND, 1, NEAR>(p, stream) : launch_attend<ND, 2, NEAR>(p, stream);
}
template <bool NEAR>
int launch_attend_nd(const AttendArgs &p, const Lanes &l, hipStream_t stream) {
  switch (l.nd) {
    case 1: return launch_attend_g<1, NEAR>(p, l.g, stream);
    case 2: return launch_attend_g<2, NEAR>(p, l.g, stream);
    case 4: return launch_attend_g<4, NEAR>(p, l.g, stream);
    case 8: return launch_attend_g<8, NEAR>(p, l.g, stream);
    default: return launch_attend_g<16, NEAR>(p, l.g, stream);
  }
}

size_t attention_work_bytes(uint32_t Vd, uint32_t edges, uint32_t q_heads, uint32_t D, uint32_t max_degree) {
  if (!by_spans(Vd, edges, max_degree)) return 0;
  const uint64_t positions = static_cast<uint64_t>(Vd) * kRowCost + edges;
  const uint32_t span = span_length(positions, q_heads, D);
  const uint64_t spans = (positions + span - 1) / span;
  return static_cast<size_t>(spans * (records_bytes(q_heads, D) + sizeof(uint32_t)));
}

const char *bad_cache(const uint8_t *cache, uint32_t heads, uint32_t D, uint32_t block_rows) {
  if (heads == 0 || heads > kMostHeads) return "heads is 0 or above 1,024";
  if (D == 0 || D > kMostHeadWidth) return "width is 0 or above 256";
  if (!is_power_of_two(block_rows) || block_rows > kMostBlockRows) return "block_rows is no power of two up to 1,024";
  if (!aligned_to(cache, 16)) return "the cache needs 16-byte alignment";
  return nullptr;
}

int fail_in(const char *call, const char *why) {
  char text[160];
  snprintf(text, sizeof(text), "%s: %s", call, why);
  return fail(NTS_ERR_INVALID, text);
}

int attend(const char *call, float *out, float *lse, const float *q, const uint8_t *cache, const uint8_t *scales, const uint32_t *co,
           const uint32_t *ri, const uint32_t *mirror, uint32_t mirror_rows, uint32_t Vd, uint32_t edges, uint32_t cache_rows,
           uint32_t q_heads, uint32_t heads, uint32_t width, uint32_t block_rows, float score_scale, uint32_t max_degree, void *work,
           hipStream_t stream) {
  if (const char *why = bad_cache(cache, heads, width, block_rows)) return fail_in(call, why);
  if (q_heads == 0 || q_heads % heads || q_heads > kMostHeads) return fail_in(call, "q_heads is no multiple of heads up to 1,024");
  if (edges > 0xFFFF0000u) return fail_in(call, "more than 2^32 - 2^16 edges");
  if (Vd == 0) return NTS_OK;
  if (!out || !q || !co || (edges && !ri) || (edges && cache_rows && (!cache || !scales))) return fail_in(call, "null pointer");
  AttendArgs p{};
  p.out = out, p.lse = lse, p.q = q, p.cache = cache, p.scales = scales, p.co = co, p.ri = ri, p.mirror = mirror;
  p.mirror_rows = mirror_rows;
  p.Vd = Vd, p.cache_rows = cache_rows, p.q_heads = q_heads, p.heads = heads, p.D = width, p.row_width = kv8_row_width(width);
  p.block_shift = static_cast<uint32_t>(__builtin_ctz(block_rows));
  p.share = q_heads / heads;
  p.score_scale = score_scale;
  // Slots: where a bound is known most rows reach it, and a slot that works through 16 edges costs least (60,000 rows of 10
  // edges, 4 heads of 32: 37 us with one slot, 42 with two, 51 with four when chosen, 40 now); averages hide longer rows (2.48 M edges
  // in 169 K rows: 229 us with four slots for 15 edges on average, 264 with two, 572 with one when chosen, 201 now).
  const bool blocks = by_blocks(Vd, edges, max_degree), spans = by_spans(Vd, edges, max_degree);
  const Lanes l = lanes_for(q_heads, heads, width, blocks ? kWave : spans ? (static_cast<uint64_t>(edges) / Vd + 4) / 4 : (max_degree + 15) / 16);
  p.units = l.units, p.per_head = l.per_head, p.hw_shift = l.hw_shift, p.walker_shift = l.walker_shift;
  p.passes = ceil_div(l.units, 1u << l.hw_shift);
  p.blocks = blocks;
  if (spans) {
    if (!work || !aligned_to(work, 16)) return fail_in(call, "needs nts_kv8_attention_work_bytes of 16-byte-aligned work");
    p.positions = static_cast<uint64_t>(Vd) * kRowCost + edges;
    p.span = span_length(p.positions, q_heads, width);
    p.spans = static_cast<uint32_t>((p.positions + p.span - 1) / p.span);
    p.partial = static_cast<float *>(work);
    p.tail_row = reinterpret_cast<uint32_t *>(p.partial + static_cast<uint64_t>(p.spans) * 2u * q_heads * (width + 2u));
  }
  const uint64_t bytes = 2ull * heads * std::max(static_cast<uint64_t>(cache_rows) * p.row_width, static_cast<uint64_t>(cache_rows) / block_rows + 1);
  return bytes < 0xFFFF0000ull && cache_rows <= (1u << 24) ? launch_attend_nd<true>(p, l, stream) : launch_attend_nd<false>(p, l, stream);
}

}  // namespace
}  // namespace nts

using namespace nts;

extern "C" {

int nts_kv8_append(uint8_t *cache, uint8_t *scales, const float *k, const float *v, uint32_t first, uint32_t n,
                   uint32_t capacity, uint32_t heads, uint32_t width, uint32_t block_rows, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_kv8_append");
  if (const char *why = bad_cache(cache, heads, width, block_rows)) return fail_in("nts_kv8_append", why);
  if (first > capacity || n > capacity - first) return fail_in("nts_kv8_append", "rows beyond the capacity");
  if (n == 0) return NTS_OK;
  if (!cache || !scales || !k || !v) return fail_in("nts_kv8_append", "null pointer");
  const uint32_t first_block = first / block_rows;
  const uint64_t blocks = (static_cast<uint64_t>(first) + n + block_rows - 1) / block_rows - first_block;
  const AppendArgs p{cache, scales, k, v, first, n, heads, width, kv8_row_width(width) / 4, block_rows, first_block,
                     blocks * 2u * heads};
  const uint64_t grid = std::min<uint64_t>((p.units + 3) / 4, kMostBlocks);
  const uint32_t quads = block_rows * p.quads;
  const auto kernel = quads <= 2 * kWave ? kv8_append_kernel<2> : quads <= 8 * kWave ? kv8_append_kernel<8> : kv8_append_kernel<0>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(grid)), dim3(256), 0, stream, p);
  NTS_LAUNCH_CHECK("nts_kv8_append");
  return NTS_OK;
}

size_t nts_kv8_attention_work_bytes(uint32_t Vd, uint32_t edges, uint32_t q_heads, uint32_t width, uint32_t max_degree) {
  if (q_heads == 0 || q_heads > kMostHeads || width == 0 || width > kMostHeadWidth) return 0;
  return attention_work_bytes(Vd, edges, q_heads, width, max_degree);
}

int nts_kv8_attention(float *out, float *lse, const float *q, const uint8_t *cache, const uint8_t *scales, const uint32_t *co,
                      const uint32_t *ri, const uint32_t *mirror, uint32_t Vd, uint32_t edges, uint32_t cache_rows,
                      uint32_t q_heads, uint32_t heads, uint32_t width, uint32_t block_rows, float score_scale,
                      uint32_t max_degree, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_kv8_attention");
  return attend("nts_kv8_attention", out, lse, q, cache, scales, co, ri, mirror, 0xFFFFFFFFu, Vd, edges, cache_rows, q_heads, heads,
                width, block_rows, score_scale, max_degree, work, stream);
}

int nts_kv8_attention_local(float *out, float *lse, const float *q, const uint8_t *cache, const uint8_t *scales, const uint32_t *co,
                            const uint32_t *ri, const uint32_t *mirror, uint32_t mirror_rows, uint32_t Vd, uint32_t edges,
                            uint32_t cache_rows, uint32_t q_heads, uint32_t heads, uint32_t width, uint32_t block_rows,
                            float score_scale, uint32_t max_degree, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_kv8_attention_local");
  if (mirror_rows && !mirror) return fail_in("nts_kv8_attention_local", "null pointer");
  // a mirror without entries names no row of the cache, like a cache without rows
  return attend("nts_kv8_attention_local", out, lse, q, cache, scales, co, ri, mirror_rows ? mirror : nullptr, mirror_rows, Vd, edges,
                mirror_rows ? cache_rows : 0u, q_heads, heads, width, block_rows, score_scale, max_degree, work, stream);
}

}  // extern "C"
