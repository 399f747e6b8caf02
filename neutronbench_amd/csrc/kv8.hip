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
// (exactly, unless the value falls among e4m3's subnormals).  Both passes read through the caches the second time.
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
    const Quad q = *reinterpret_cast<const Quad *>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q.v[i];
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
      if (col + i < p.D) v[i] = at[i];
  }
}

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
    for (uint32_t j = lane; j < total; j += kWave) {
      const uint32_t r = j / p.quads;
      float v[4];
      append_values(p, src, held, held_scale, static_cast<uint32_t>(row0) + r, j - r * p.quads, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        if (b < 0x7F800000u) top = max(top, b);
      }
    }
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, kWave)));
    // 448 = 1.75 * 2^8
    const uint32_t up = (top >> 23) + ((top & 0x7FFFFFu) > 0x600000u ? 1u : 0u);
    const uint32_t byte = max(old, up > 8u ? up - 8u : 0u);
    const float inverse = e8m0_inverse(min(byte, 253u));
    for (uint32_t j = lane; j < total; j += kWave) {
      const uint32_t r = j / p.quads;
      const uint32_t row = static_cast<uint32_t>(row0) + r, quad = j - r * p.quads;
      if (row < p.first && byte == old) continue;
      float v[4];
      append_values(p, src, held, held_scale, row, quad, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] *= inverse;
      *reinterpret_cast<uint32_t *>(held + static_cast<uint64_t>(row) * 2u * p.heads * p.quads * 4u + quad * 4u) = e4m3_encode4(v);
    }
    if (lane == 0) *scale = static_cast<uint8_t>(byte);
  }
}

// ---- attention --------------------------------------------------------------------------------------
//   s_e = score_scale * q[d, h] . K[src(e), h'],  p_e = exp(s_e - max s),  out[d, h, :] = sum_e p_e V[src(e), h'] / sum_e p_e
// for the edges e of destination d whose source is cached; h' = h / (q_heads / heads).  One pass: the running maximum, sum
// and weighted sum of values stay in registers and are rescaled when the maximum grows.
//
// A lane holds 16 columns of one head: one 16-byte load of a key row and one of a value row.  ND lanes (a power of two) cover a
// head, `hw` heads lie side by side, and what is left of the wavefront takes further edges of the same destination ("slots"),
// each with a running softmax of its own, joined at the end.  G query heads that share the head's keys are computed from one
// load.
struct AttendArgs {
  float *out, *lse;
  const float *q;
  const uint8_t *cache, *scales;
  const uint32_t *co, *ri, *mirror;
  uint32_t Vd, cache_rows, q_heads, heads, D, row_width, block_shift;
  uint32_t share;                       // query heads per head
  uint32_t hw_shift;                    // log2 of heads side by side
  uint32_t head_chunks, share_chunks;   // passes over the edges: blockIdx.y = head chunk * share_chunks + share chunk
  float score_scale;
  // edges cut into spans of `span` positions (see below); 0: a wavefront per destination
  uint32_t span, spans;
  uint64_t positions;
  float *partial;
  uint32_t *tail_row;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int ND, int G>
struct Attend {
  const AttendArgs &p;
  uint32_t dl, kv_head, q_head0, slot, slots;
  bool live;  // this lane has a head and columns
  float q[G][16], acc[G][16], top[G], sum[G];

  __device__ __forceinline__ Attend(const AttendArgs &args) : p(args) {
    const uint32_t lane = threadIdx.x & (kWave - 1);
    dl = lane & (ND - 1);
    const uint32_t hc = blockIdx.y / p.share_chunks, sc = blockIdx.y - hc * p.share_chunks;
    kv_head = (hc << p.hw_shift) + ((lane / ND) & ((1u << p.hw_shift) - 1u));
    slot = lane / (static_cast<uint32_t>(ND) << p.hw_shift);
    slots = (kWave / ND) >> p.hw_shift;
    live = kv_head < p.heads && dl * 16u < p.row_width;
    q_head0 = sc * G;  // within the head's share
  }

  __device__ __forceinline__ void begin(uint32_t row) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      top[g] = -INFINITY;
      sum[g] = 0.0f;
      const bool there = live && q_head0 + g < p.share;
      const float *src = p.q + (static_cast<uint64_t>(row) * p.q_heads + kv_head * p.share + q_head0 + g) * p.D + dl * 16u;
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        acc[g][i] = 0.0f;
        q[g][i] = there && dl * 16u + i < p.D ? src[i] : 0.0f;
      }
    }
  }

  // Edges [j0, j1) of the destination whose edges begin at `first`.
  __device__ __forceinline__ void edges(uint32_t first, uint32_t j0, uint32_t j1) {
    const float unit = p.score_scale * kLog2e;
    for (uint32_t j = j0; j < j1; j += slots) {
      const bool mine = j + slot < j1;
      uint32_t g_row = 0xFFFFFFFFu;
      if (mine) {
        g_row = p.ri[static_cast<uint64_t>(first) + j + slot];
        if (p.mirror) g_row = p.mirror[g_row];
      }
      const bool there = g_row < p.cache_rows;
      float k[16], v[16];
      float ks = 0.0f, vs = 0.0f;
      uint4 kc = make_uint4(0, 0, 0, 0), vc = kc;
      if (there && live) {
        const uint8_t *row = p.cache + (static_cast<uint64_t>(g_row) * 2u * p.heads + kv_head) * p.row_width + dl * 16u;
        kc = *reinterpret_cast<const uint4 *>(row);
        vc = *reinterpret_cast<const uint4 *>(row + static_cast<uint64_t>(p.heads) * p.row_width);
        const uint8_t *s = p.scales + static_cast<uint64_t>(g_row >> p.block_shift) * 2u * p.heads + kv_head;
        ks = e8m0_value(s[0]);
        vs = e8m0_value(s[p.heads]);
      }
      e4m3_decode4(kc.x, k), e4m3_decode4(kc.y, k + 4), e4m3_decode4(kc.z, k + 8), e4m3_decode4(kc.w, k + 12);
      e4m3_decode4(vc.x, v), e4m3_decode4(vc.y, v + 4), e4m3_decode4(vc.z, v + 8), e4m3_decode4(vc.w, v + 12);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s = fmaf(q[g][i], k[i], s);
        s = group_sum<ND>(s) * ks * unit;
        if (there) add(g, s, vs, v);
      }
    }
  }

  __device__ __forceinline__ void add(int g, float s, float vs, const float *v) {
    const float now = fmaxf(top[g], s);
    const float base = now == -INFINITY ? 0.0f : now;
    const float keep = __builtin_amdgcn_exp2f(top[g] - base), w = __builtin_amdgcn_exp2f(s - base);
    top[g] = now;
    sum[g] = fmaf(sum[g], keep, w);
    const float wv = w * vs;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[g][i] = fmaf(wv, v[i], acc[g][i] * keep);
  }

  // Joins the slots: every slot ends up with the whole.
  __device__ __forceinline__ void join() {
    for (uint32_t m = static_cast<uint32_t>(ND) << p.hw_shift; m < static_cast<uint32_t>(kWave); m <<= 1) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float other = __shfl_xor(top[g], m, kWave), more = __shfl_xor(sum[g], m, kWave);
        const float now = fmaxf(top[g], other), base = now == -INFINITY ? 0.0f : now;
        const float a = __builtin_amdgcn_exp2f(top[g] - base), b = __builtin_amdgcn_exp2f(other - base);
        top[g] = now;
        sum[g] = sum[g] * a + more * b;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[g][i] = acc[g][i] * a + __shfl_xor(acc[g][i], m, kWave) * b;
      }
    }
  }

  __device__ __forceinline__ void write(uint32_t row) {
    if (slot != 0 || !live) return;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (q_head0 + g >= p.share) continue;
      const uint64_t at = static_cast<uint64_t>(row) * p.q_heads + kv_head * p.share + q_head0 + g;
      float *dst = p.out + at * p.D + dl * 16u;
      const float inv = sum[g] == 0.0f ? 0.0f : 1.0f / sum[g];
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (dl * 16u + i < p.D) dst[i] = acc[g][i] * inv;
      if (p.lse && dl == 0) p.lse[at] = sum[g] == 0.0f ? -INFINITY : (top[g] + __builtin_amdgcn_logf(sum[g])) * kLn2;
    }
  }

  // A part of a destination's edges: top, sum and weighted sums of every query head, for join_spans_kernel.
  __device__ __forceinline__ void write_partial(uint32_t record) {
    if (slot != 0 || !live) return;
    const uint64_t size = static_cast<uint64_t>(p.q_heads) * (p.D + 2u);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (q_head0 + g >= p.share) continue;
      float *dst = p.partial + record * size;
      const uint32_t h = kv_head * p.share + q_head0 + g;
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (dl * 16u + i < p.D) dst[static_cast<uint64_t>(h) * p.D + dl * 16u + i] = acc[g][i];
      if (dl == 0) {
        dst[static_cast<uint64_t>(p.q_heads) * p.D + h] = top[g];
        dst[static_cast<uint64_t>(p.q_heads) * (p.D + 1u) + h] = sum[g];
      }
    }
  }
};

// A wavefront per destination.
template <int ND, int G>
__global__ __launch_bounds__(256) void kv8_attend_rows_kernel(AttendArgs p) {
  Attend<ND, G> a(p);
  const uint64_t waves = static_cast<uint64_t>(gridDim.x) * (256 / kWave);
  for (uint64_t row = wave_of_grid(); row < p.Vd; row += waves) {
    const uint32_t first = p.co[row], degree = p.co[row + 1] - first;
    a.begin(static_cast<uint32_t>(row));
    a.edges(first, 0, degree);
    a.join();
    a.write(static_cast<uint32_t>(row));
  }
}

// Long rows are shared out and short ones bundled without a look at the degrees on the host: destinations and edges are
// lined up -- destination r takes position r + co[r] - co[0], its edges the positions behind it -- and every wavefront walks
// one span of `span` positions.  Destinations that lie within the span are written at once; a part of one that reaches over
// the span's end or its beginning goes to the span's two records (0: began in an earlier span, 1: goes on in the next), and
// join_spans_kernel adds the parts in order.  No atomics: the same bits on every call.
__device__ __forceinline__ uint64_t position_of(const uint32_t *co, uint32_t co0, uint64_t r) { return r + (co[r] - co0); }

// The last destination at or before position x: 64 candidates a step.
__device__ __forceinline__ uint32_t destination_at(const uint32_t *co, uint32_t co0, uint32_t Vd, uint64_t x) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  uint32_t lo = 0, hi = Vd;  // position_of(lo) <= x, the answer is in [lo, hi)
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + kWave - 1) / kWave;
    const uint64_t r = static_cast<uint64_t>(lo) + static_cast<uint64_t>(lane) * step;
    const bool before = r < hi && position_of(co, co0, r) <= x;
    const uint32_t count = __popcll(__ballot(before));  // the first lane always counts
    const uint32_t next = lo + (count - 1) * step;
    hi = hi - next > step ? next + step : hi;
    lo = next;
  }
  return lo;
}

template <int ND, int G>
__global__ __launch_bounds__(256) void kv8_attend_spans_kernel(AttendArgs p) {
  const uint32_t span = static_cast<uint32_t>(wave_of_grid());
  if (span >= p.spans) return;
  Attend<ND, G> a(p);
  const uint64_t begin = static_cast<uint64_t>(span) * p.span, end = min(begin + p.span, p.positions);
  const uint32_t co0 = p.co[0];
  uint32_t row = wave_first(destination_at(p.co, co0, p.Vd, begin));
  uint32_t tail = kNoSlot;
  for (; row < p.Vd; ++row) {
    const uint32_t first = p.co[row], degree = p.co[row + 1] - first;
    const uint64_t at = static_cast<uint64_t>(row) + (first - co0);  // the destination's own position, its edges behind it
    if (at >= end) break;
    const uint32_t j0 = at + 1 < begin ? static_cast<uint32_t>(min<uint64_t>(begin - at - 1, degree)) : 0u;
    const uint32_t j1 = static_cast<uint32_t>(min<uint64_t>(degree, end - at - 1));
    a.begin(row);
    a.edges(first, j0, j1);
    a.join();
    const bool goes_on = j1 < degree;
    if (at < begin) {
      if (degree && j0 < degree) a.write_partial(span * 2u);
    } else if (goes_on) {
      a.write_partial(span * 2u + 1u);
      tail = row;
    } else {
      a.write(row);
    }
    if (goes_on) break;
  }
  if (blockIdx.y == 0 && (threadIdx.x & (kWave - 1)) == 0) p.tail_row[span] = tail;
}

// The destinations that reach over a span's end: a block each, columns in parallel, parts in order.
__global__ __launch_bounds__(256) void join_spans_kernel(AttendArgs p) {
  const uint32_t span = blockIdx.x, row = p.tail_row[span];
  if (row == kNoSlot) return;
  const uint64_t last_at = static_cast<uint64_t>(row) + (p.co[row + 1] - p.co[0]);  // position of its last edge
  const uint32_t last = static_cast<uint32_t>(min<uint64_t>(last_at / p.span, p.spans - 1u));
  const uint64_t size = static_cast<uint64_t>(p.q_heads) * (p.D + 2u);
  const uint32_t columns = p.q_heads * p.D;
  for (uint32_t c = threadIdx.x; c < columns; c += 256) {
    const uint32_t h = c / p.D;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
    for (uint32_t s = span; s <= last; ++s) {
      const float *from = p.partial + (static_cast<uint64_t>(s) * 2u + (s == span ? 1u : 0u)) * size;
      const float t = from[columns + h], l = from[columns + p.q_heads + h], v = from[c];
      const float now = fmaxf(top, t), base = now == -INFINITY ? 0.0f : now;
      const float a = __builtin_amdgcn_exp2f(top - base), b = __builtin_amdgcn_exp2f(t - base);
      top = now;
      sum = sum * a + l * b;
      acc = acc * a + v * b;
    }
    const uint64_t at = static_cast<uint64_t>(row) * p.q_heads + h;
    p.out[static_cast<uint64_t>(row) * columns + c] = sum == 0.0f ? 0.0f : acc / sum;
    if (p.lse && c == h * p.D) p.lse[at] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

constexpr uint32_t kMostHeadWidth = 256, kMostHeads = 1024, kMostBlockRows = 1024;
// Above this bound (or without one) a row may be long enough to keep one wavefront busy after the others are done.
constexpr uint32_t kMostRowEdges = 256;

// Bytes of a span's two records.
uint64_t records_bytes(uint32_t q_heads, uint32_t D) { return 2ull * q_heads * (D + 2u) * sizeof(float); }
// Positions of a span, for `positions` of them: 8,192 spans fill the chip (fewer where their records would take more than
// 256 MB), none of fewer than 64 positions.
uint32_t span_length(uint64_t positions, uint32_t q_heads, uint32_t D) {
  const uint64_t spans = std::max<uint64_t>(256, std::min<uint64_t>(8192, (256ull << 20) / records_bytes(q_heads, D)));
  const uint64_t wanted = (positions + spans - 1) / spans;
  return static_cast<uint32_t>(std::max<uint64_t>(wanted, 64));
}
bool by_spans(uint32_t max_degree) { return max_degree == 0 || max_degree > kMostRowEdges; }

template <int ND, int G>
int launch_attend(const AttendArgs &p, hipStream_t stream) {
  const uint32_t passes = p.head_chunks * p.share_chunks;
  if (!p.span) {
    const uint64_t blocks = std::min<uint64_t>((static_cast<uint64_t>(p.Vd) + 3) / 4, kMostBlocks / passes);
    hipLaunchKernelGGL((kv8_attend_rows_kernel<ND, G>), dim3(static_cast<uint32_t>(blocks), passes), dim3(256), 0, stream, p);
    NTS_LAUNCH_CHECK("nts_kv8_attention");
    return NTS_OK;
  }
  hipLaunchKernelGGL((kv8_attend_spans_kernel<ND, G>), dim3((p.spans + 3) / 4, passes), dim3(256), 0, stream, p);
  NTS_LAUNCH_CHECK("nts_kv8_attention");
  if (p.spans > 1) {
    hipLaunchKernelGGL(join_spans_kernel, dim3(p.spans), dim3(256), 0, stream, p);
    NTS_LAUNCH_CHECK("join_spans_kernel");
  }
  return NTS_OK;
}
template <int ND>
int launch_attend_g(const AttendArgs &p, uint32_t g, hipStream_t stream) {
  return g == 1 ? launch_attend<ND, 1>(p, stream) : g == 2 ? launch_attend<ND, 2>(p, stream) : launch_attend<ND, 4>(p, stream);
}

uint32_t next_power(uint32_t v) {
  uint32_t p = 1;
  while (p < v) p <<= 1;
  return p;
}

size_t attention_work_bytes(uint32_t Vd, uint32_t edges, uint32_t q_heads, uint32_t D, uint32_t max_degree) {
  if (!by_spans(max_degree)) return 0;
  const uint64_t positions = static_cast<uint64_t>(Vd) + edges;
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
  hipLaunchKernelGGL(kv8_append_kernel, dim3(static_cast<uint32_t>(grid)), dim3(256), 0, stream, p);
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
  const char *const call = "nts_kv8_attention";
  NTS_TRACE_RANGE("nts_kv8_attention");
  if (const char *why = bad_cache(cache, heads, width, block_rows)) return fail_in(call, why);
  if (q_heads == 0 || q_heads % heads || q_heads > kMostHeads) return fail_in(call, "q_heads is no multiple of heads up to 1,024");
  if (edges > 0xFFFF0000u) return fail_in(call, "more than 2^32 - 2^16 edges");
  if (Vd == 0) return NTS_OK;
  if (!out || !q || !co || (edges && !ri) || (edges && cache_rows && (!cache || !scales))) return fail_in(call, "null pointer");
  AttendArgs p{};
  p.out = out, p.lse = lse, p.q = q, p.cache = cache, p.scales = scales, p.co = co, p.ri = ri, p.mirror = mirror;
  p.Vd = Vd, p.cache_rows = cache_rows, p.q_heads = q_heads, p.heads = heads, p.D = width, p.row_width = kv8_row_width(width);
  p.block_shift = static_cast<uint32_t>(__builtin_ctz(block_rows));
  p.share = q_heads / heads;
  p.score_scale = score_scale;
  const uint32_t nd = next_power(p.row_width / 16);
  const uint32_t hw = std::min(kWave / nd, next_power(heads));
  p.hw_shift = static_cast<uint32_t>(__builtin_ctz(hw));
  const uint32_t g = p.share >= 3 ? 4 : p.share;
  p.head_chunks = ceil_div(heads, hw);
  p.share_chunks = ceil_div(p.share, g);
  if (by_spans(max_degree)) {
    if (!work || !aligned_to(work, 16)) return fail_in(call, "needs nts_kv8_attention_work_bytes of 16-byte-aligned work");
    p.positions = static_cast<uint64_t>(Vd) + edges;
    p.span = span_length(p.positions, q_heads, width);
    p.spans = static_cast<uint32_t>((p.positions + p.span - 1) / p.span);
    p.partial = static_cast<float *>(work);
    p.tail_row = reinterpret_cast<uint32_t *>(p.partial + static_cast<uint64_t>(p.spans) * 2u * q_heads * (width + 2u));
  }
  switch (nd) {
    case 1: return launch_attend_g<1>(p, g, stream);
    case 2: return launch_attend_g<2>(p, g, stream);
    case 4: return launch_attend_g<4>(p, g, stream);
    case 8: return launch_attend_g<8>(p, g, stream);
    default: return launch_attend_g<16>(p, g, stream);
  }
}

}  // extern "C"
