// Rows of 4-bit values (e2m1, 32 of them to an e8m0 scale) and products on them: the rounding of feature rows, a dense layer
// on rows gathered by vertex id, and its two gradients.  Reading such rows back as floats is in gather.hip.
#include <algorithm>

#include "launch_size.hpp"
#include "lowbit.hpp"

namespace nts {
namespace {

// ---- rounding ---------------------------------------------------------------------------------------
// Per block of 32 values of a row: e = floor(log2 max|x|) - 2, so that the largest value lies in [4, 8) of the code's range
// 0 .. 6 (7 and more become 6), then every x 2^-e to the nearest code.  Eight lanes take a block, four floats each; the
// maximum is one of integers, since the bits of |x| order as the values do and infinities and NaN lie above them.
// Blocks of a lane group that are requested together (2.45 M rows of 100: 282 us with four, 325 with one, 291 with two; 295 under a
// kernel trace, 3.9 TB/s).
constexpr uint32_t kQuantizeAhead = 4;
__global__ __launch_bounds__(256) void mx_quantize_kernel(uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                          const float *__restrict__ x, uint32_t n_blocks, uint32_t F,
                                                          uint32_t row_blocks, uint32_t scale_stride) {
  const uint32_t sub = threadIdx.x & 7u;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * (32u * kQuantizeAhead);
  for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * (32u * kQuantizeAhead) + threadIdx.x / 8u; first < n_blocks; first += step) {
    float v[kQuantizeAhead][4];
    uint64_t row[kQuantizeAhead];
    uint32_t kb[kQuantizeAhead];
#pragma unroll
    for (uint32_t u = 0; u < kQuantizeAhead; ++u) {
      const uint64_t b = first + u * 32u;
      const uint32_t r = static_cast<uint32_t>(b) / row_blocks;
      kb[u] = static_cast<uint32_t>(b) - r * row_blocks;
      row[u] = r;
      const uint32_t col = kb[u] * kMxBlock + sub * 4u;
      const float *src = x + row[u] * F + col;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = 0.0f;
      if (b >= n_blocks) continue;
      if (col + 4u <= F) {
        const FloatQuad q = *reinterpret_cast<const FloatQuad *>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[u][i] = q[i];
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i)
          if (col + i < F) v[u][i] = src[i];
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < kQuantizeAhead; ++u) {
      const uint64_t b = first + u * 32u;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[u][i]) & 0x7FFFFFFFu);
#pragma unroll
      for (int m = 1; m < 8; m <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, kWave)));
      if (b >= n_blocks) continue;
      const uint32_t exponent = top >> 23;
      const bool fine = exponent < 255u;
      const uint32_t byte = !fine ? 255u : (exponent > 2u ? exponent - 2u : 0u);
      const float inverse = e8m0_inverse(fine ? byte : 0u);
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) word |= e2m1_encode(v[u][i], inverse) << (4 * i);
      reinterpret_cast<uint16_t *>(codes)[b * 8u + sub] = static_cast<uint16_t>(fine ? word : 0u);
      // the block's scale, and the bytes that fill the last block's row up to whole words
      const uint32_t at = kb[u] + sub;
      if (sub == 0 || (kb[u] + 1 == row_blocks && at < scale_stride))
        scales[row[u] * scale_stride + at] = static_cast<uint8_t>(sub == 0 ? byte : 0u);
    }
  }
}

// ---- product ----------------------------------------------------------------------------------------
//   out[i, j] (+)= sum_f A[row_ids[i], f] W[j, f]
// v_mfma_scale_f32_16x16x128 takes 16 rows of each operand, 128 values deep: lane l holds row l % 16, the 32 values of block
// l / 16, which are 16 consecutive bytes of the row, and that block's scale.  So the operands go from memory to registers as
// they lie.  W is the first operand: a lane then ends up with four neighbouring columns of one output row.

// Blocks are handed to the eight chiplets, each with an L2 of its own, in turn.  Where there are kXcdTiles tiles of rows or more, a
// chiplet takes `group` of them at a time, every column of tiles for all of the group before the next: blocks that run together share
// rows and columns.  With fewer, tiles in turn fill the chip more evenly.  Product of 232,965 rows of 602 by 256: 79.5 -> 65.5 us, the
// rows' gradient of 169,343 by 640 by 640: 607 -> 489.
constexpr uint32_t kXcdTiles = 64;
__device__ __forceinline__ void tile_of(uint32_t tiles_n, bool by_xcd, uint32_t group, uint32_t *tm, uint32_t *tn) {
  if (by_xcd) {
    const uint32_t x = blockIdx.x / 8u, of = group * tiles_n, within = x % of;
    *tm = (x / of * group + within % group) * 8u + blockIdx.x % 8u;
    *tn = within / group;
  } else {
    *tm = blockIdx.x / tiles_n;
    *tn = blockIdx.x % tiles_n;
  }
}
uint32_t tile_blocks(uint32_t tiles_m, uint32_t tiles_n, uint32_t group) {
  return (tiles_m >= kXcdTiles ? ceil_div(tiles_m, 8 * group) * 8u * group : tiles_m) * tiles_n;
}

struct MxRows {
  const uint8_t *codes;
  const uint8_t *scales;
};

struct ProductArgs {
  float *out;
  MxRows a;
  uint32_t table_rows;
  const uint32_t *row_ids;  // null: row i
  uint32_t n;
  MxRows w;
  uint32_t N, row_blocks, scale_stride;
  int accumulate;
  bool streamed;  // the output goes past the caches
};

__device__ __forceinline__ i32x8 operand(i32x4 c) { return i32x8{c.x, c.y, c.z, c.w, 0, 0, 0, 0}; }

// Four neighbouring columns of an output row.
__device__ __forceinline__ void write_columns(const ProductArgs &p, uint64_t i, uint64_t c, f32x4 v) {
  float *dst = p.out + i * p.N + c;
  if (c + 4u <= p.N) {
    if (p.accumulate) {
      const FloatQuad old = *reinterpret_cast<const FloatQuad *>(dst);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += old[k];
    }
    store_quad(dst, FloatQuad{v.x, v.y, v.z, v.w}, p.streamed);
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (c + k < p.N) dst[k] = p.accumulate ? dst[k] + v[k] : v[k];
  }
}

// 16 rows by 16 columns; the scales are bytes `wb` of `sw` and `ab` of `sa`, constants once inlined.
__device__ __forceinline__ f32x4 multiply_16(i32x4 w, i32x4 a, f32x4 c, int wb, uint32_t sw, int ab, uint32_t sa) {
#define NTS_MX_MFMA(WB, AB) \
  __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(a), c, 4, 4, WB, static_cast<int>(sw), AB, static_cast<int>(sa))
#define NTS_MX_MFMA_A(WB) (ab == 0 ? NTS_MX_MFMA(WB, 0) : ab == 1 ? NTS_MX_MFMA(WB, 1) : ab == 2 ? NTS_MX_MFMA(WB, 2) : NTS_MX_MFMA(WB, 3))
  return wb == 0 ? NTS_MX_MFMA_A(0) : wb == 1 ? NTS_MX_MFMA_A(1) : wb == 2 ? NTS_MX_MFMA_A(2) : NTS_MX_MFMA_A(3);
#undef NTS_MX_MFMA_A
#undef NTS_MX_MFMA
}

// Few rows (a prediction for one vertex or some): the weight is what has to be read, once, and its latency is what counts.  A
// block takes 16 columns and 16 * MT rows; its wavefronts take every kFewWaves-th 128 values of the rows, two at a time, and the
// first adds up what they have, in order.
constexpr uint32_t kFewWaves = 8;
template <int MT>
__global__ __launch_bounds__(kFewWaves *kWave) void mx_product_few_kernel(ProductArgs p) {
  __shared__ f32x4 sums[kFewWaves - 1][MT][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block(), r = lane & 15u, part = lane >> 4;
  const uint64_t col = blockIdx.x * 16ull + r;
  uint64_t row[MT];
  bool there[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint64_t i = (blockIdx.y * MT + m) * 16ull + r;
    row[m] = 0;
    there[m] = i < p.n;
    if (there[m]) row[m] = p.row_ids ? p.row_ids[i] : i;
    there[m] = there[m] && row[m] < p.table_rows;
  }
  f32x4 acc[MT] = {};
  // a lane's part of 128 values of a row; zeros (and a scale that is none's) where there is no such block or row
  auto load = [&](const MxRows &t, uint64_t row, bool there, uint32_t block, i32x4 *codes, uint32_t *scale) {
    *codes = i32x4{0, 0, 0, 0};
    *scale = 127u;
    if (there && block < p.row_blocks) {
      *codes = *reinterpret_cast<const i32x4 *>(t.codes + (row * p.row_blocks + block) * 16u);
      *scale = t.scales[row * p.scale_stride + block];
    }
  };
  for (uint32_t base = wave * 4u; base < p.row_blocks; base += kFewWaves * 8u) {
    i32x4 w[2], a[2][MT];
    uint32_t sw[2], sa[2][MT];
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t block = base + u * kFewWaves * 4u + part;
      load(p.w, col, col < p.N, block, &w[u], &sw[u]);
#pragma unroll
      for (int m = 0; m < MT; ++m) load(p.a, row[m], there[m], block, &a[u][m], &sa[u][m]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = multiply_16(w[u], a[u][m], acc[m], 0, sw[u], 0, sa[u][m]);
  }
  if (wave) {
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave - 1][m][lane] = acc[m];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (uint32_t k = 0; k < kFewWaves - 1; ++k) acc[m] += sums[k][m][lane];
    const uint64_t i = (blockIdx.y * MT + m) * 16ull + r;
    if (i < p.n) write_columns(p, i, blockIdx.x * 16ull + part * 4u, acc[m]);
  }
}

// Many rows: a block of WM x WN wavefronts takes BM rows by BN columns through LDS, a stage of 32 * PARTS values at a time: 64
// or 128 bytes a row.  The loads write a stage to LDS themselves (no registers between) while the one before it is
// multiplied.  Part c of row r lies at c ^ (r * PARTS / 16) % PARTS, so that the 16 lanes that read one part of 16 rows meet all
// banks once.
// Measured (65,536 rows of 4,096 values by 4,096 columns): 700 us, 3.1 PFLOP/s (684 .. 715 from card to card), where a library's bf16
// product of that size takes 1,580 and its rate times four would take 394.  The matrix units are busy for 34 % of the time.  When the
// whole took 684: 411 without loads and stores, 493 with the stores, 686 with the loads: bound by the loads of codes into LDS and the
// waits for them.  Steps: registers in place of loads into LDS 1,170; stores past the caches 1,043 -> 900; operands asked for a step
// ahead 893 -> 785; results turned in LDS and stored as whole lines 785 -> 693.  128 x 128 with stages of 64 bytes takes 912.
typedef __attribute__((address_space(3))) void *LdsPointer;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t *p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, bytes, 0x00027000);
}
// 16 bytes a lane from `from` + offset + at to 1,024 consecutive bytes of LDS.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, uint8_t *to, uint32_t offset, uint32_t at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (LdsPointer)to, 16, offset, at, 0, 0);
}
__device__ __forceinline__ void load_to_lds(const uint8_t *from, uint8_t *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (LdsPointer)to, 16, 0, 0);
}
// An offset behind the end of any buffer, which reads zeros: also with a stage's 16 bytes times kMostWidth / 32 blocks added, of
// which the last begins within any table that has a row.
constexpr uint32_t kNowhere = 0xFFFF0000u;
static_assert(kNowhere + (kMostWidth / kMxBlock - 1) * 16u > kNowhere, "the sum fits 32 bits");
__device__ __attribute__((aligned(16))) uint8_t zero_part[16];  // zeros for the loads that go by address

// Waits for the wavefront's loads and LDS accesses, then for the block.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr uint32_t kRowGroup = 8;  // 65,536 x 4,096 by 4,096, one after the other: 718 us; groups of 4 737, of 2 752, tiles in turn 737
// NEAR: both tables' codes are less than 4 GB and are read through buffer descriptors, by 32-bit offsets.
template <int BM, int BN, int WM, int WN, int PARTS, bool NEAR>
__global__ __launch_bounds__(WM *WN *kWave, 2) void mx_product_tiled_kernel(ProductArgs p, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr int kThreads = WM * WN * kWave, kWaves = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int kRows = BM + BN, kBytes = PARTS * 16, kLoadRows = kWave / PARTS, kLoads = kRows / kLoadRows / kWaves;
  constexpr int kScaleRows = (kRows + kThreads - 1) / kThreads, kSpread = 16 / PARTS;
  static_assert(PARTS == 4 || PARTS == 8, "a row's part of a stage");
  static_assert(kLoads * kLoadRows * kWaves == kRows && BM % (kLoadRows * kWaves) == 0, "a load's rows are all of A or all of W");
  static_assert(kLoadRows * kWaves / kSpread % PARTS == 0, "rows of a wavefront's loads are alike in their parts");
  static_assert(BM % (WM * 64) == 0 && BN % (WN * 64) == 0, "whole words of scales");
  __shared__ __attribute__((aligned(16))) uint8_t tile0[kRows * kBytes], tile1[kRows * kBytes];
  __shared__ __attribute__((aligned(16))) uint8_t tile_scales[2][kRows * PARTS];
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = wave_of_block(), r = lane & 15u, part = lane >> 4;
  uint32_t tile_m, tn;
  tile_of(tiles_n, tiles_m >= kXcdTiles, kRowGroup, &tile_m, &tn);
  if (tile_m >= tiles_m) return;
  const uint64_t tm = tile_m;
  // the row of A's or W's table that row `row` of a stage holds; false: none
  auto table_row = [&](uint32_t row, uint64_t *g) {
    if (row < BM) {
      const uint64_t at = tm * BM + row;
      if (at >= p.n) return false;
      *g = p.row_ids ? p.row_ids[at] : at;
      return *g < p.table_rows;
    }
    *g = static_cast<uint64_t>(tn) * BN + row - BM;
    return *g < p.N;
  };
  // A wavefront's load writes 1,024 consecutive bytes of LDS, 16 a lane: kLoadRows rows of a stage.  Which part of its row a lane
  // fetches is what places the parts as the reads want them.
  const auto a_codes = buffer_of(p.a.codes, p.table_rows * p.row_blocks * 16u), w_codes = buffer_of(p.w.codes, p.N * p.row_blocks * 16u);
  uint32_t src[kLoads];
  const uint8_t *far[kLoads];
  const uint32_t chunk = (lane ^ ((wave * kLoadRows + lane / PARTS) / kSpread)) % PARTS;  // the same in all of the lane's rows
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t row = (i * kWaves + wave) * kLoadRows + lane / PARTS;
    uint64_t g = 0;
    const bool there = table_row(row, &g);
    src[i] = there ? (static_cast<uint32_t>(g) * p.row_blocks + chunk) * 16u : kNowhere;
    far[i] = there ? (row < BM ? p.a.codes : p.w.codes) + (g * p.row_blocks + chunk) * 16u : nullptr;
  }
  auto request = [&](uint8_t *tile, uint32_t base) {  // blocks base .. base + PARTS - 1
    const bool inside = base + chunk < p.row_blocks;
    // never behind the end of a table: the hardware may compare an offset with the table's length less this
    const uint32_t at = min(base, p.row_blocks - 1u) * 16u, a_at = p.table_rows ? at : 0u;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint8_t *to = tile + (i * kWaves + wave) * 1024u;
      const bool of_a = (i + 1) * kLoadRows * kWaves <= BM;
      if (NEAR)
        load_to_lds(of_a ? a_codes : w_codes, to, inside ? src[i] : kNowhere, of_a ? a_at : at);
      else
        load_to_lds(inside && far[i] ? far[i] + base * 16ull : zero_part, to);
    }
  };
  // Scales: 16 of a row at a time into registers, PARTS of them to LDS with each stage, as words that hold those of one block of
  // four rows that are 16 apart: four products take theirs from one word.
  const uint8_t *scale_src[kScaleRows];
  bool has_scales[kScaleRows];
  u32x4 words[kScaleRows];
#pragma unroll
  for (int i = 0; i < kScaleRows; ++i) {
    const uint32_t row = t + i * kThreads;
    uint64_t g = 0;
    has_scales[i] = row < kRows && table_row(row, &g);
    scale_src[i] = has_scales[i] ? (row < BM ? p.a.scales : p.w.scales) + g * p.scale_stride : p.w.scales;
  }
  auto request_scales = [&](uint32_t base) {  // behind a row's end: any bytes of it
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i) {
      if (base + 16u <= p.scale_stride) {
        struct __attribute__((packed, aligned(4))) Words {
          u32x4 v;
        };
        words[i] = reinterpret_cast<const Words *>(scale_src[i] + base)->v;
      } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
          words[i][k] = *reinterpret_cast<const uint32_t *>(scale_src[i] + min(base + k * 4u, p.scale_stride - 4u));
      }
    }
  };
  auto keep_scales = [&](uint32_t half, uint32_t s, uint32_t base) {
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i) {
      const uint32_t row = t + i * kThreads;
      if (row >= kRows) continue;
      uint8_t *to = &tile_scales[half][(row / 64u * 16u + row % 16u) * 4u + row / 16u % 4u];
#pragma unroll
      for (uint32_t k = 0; k < PARTS; k += 4) {
        // scales of a row that is not there and behind the last block are 0, whatever the table has
        uint32_t word = has_scales[i] ? words[i][(s % 16u + k) / 4u] : 0u;
        if (base + k + 4u > p.row_blocks) word &= base + k < p.row_blocks ? (1u << (8u * (p.row_blocks - base - k))) - 1u : 0u;
        to[k * kRows] = static_cast<uint8_t>(word);
        to[(k + 1u) * kRows] = static_cast<uint8_t>(word >> 8);
        to[(k + 2u) * kRows] = static_cast<uint8_t>(word >> 16);
        to[(k + 3u) * kRows] = static_cast<uint8_t>(word >> 24);
      }
    }
  };
  const uint32_t m0 = wave / WN * (BM / WM), n0 = BM + wave % WN * (BN / WN);
  f32x4 acc[MT][NT] = {};
  // Each step of NT products asks for the next one's operands first; the fences keep the compiler from asking for all at once,
  // which the registers do not hold, and from putting the products off behind the barrier.
  auto multiply = [&](const uint8_t *tile, uint32_t half) {
    const uint32_t at = r * kBytes + ((part ^ (r / kSpread)) % PARTS) * 16u;
    const uint8_t *words_at = &tile_scales[half][part * kRows + r * 4u];
    constexpr int kDeep = PARTS / 4;
    i32x4 w[2][NT], a[2];
    uint32_t sw[2][NT / 4], sa[2][MT / 4];
    auto columns = [&](int k) {
#pragma unroll
      for (int j = 0; j < NT; ++j) w[k & 1][j] = *reinterpret_cast<const i32x4 *>(&tile[(n0 + j * 16u) * kBytes + (at ^ (k * 64u))]);
#pragma unroll
      for (int j = 0; j < NT; j += 4)
        sw[k & 1][j / 4] = *reinterpret_cast<const uint32_t *>(words_at + k * 4 * kRows + (n0 / 16u + j) * 16u);
#pragma unroll
      for (int m = 0; m < MT; m += 4)
        sa[k & 1][m / 4] = *reinterpret_cast<const uint32_t *>(words_at + k * 4 * kRows + (m0 / 16u + m) * 16u);
    };
    auto rows = [&](int k, int m) { a[m & 1] = *reinterpret_cast<const i32x4 *>(&tile[(m0 + m * 16u) * kBytes + (at ^ (k * 64u))]); };
    columns(0);
    rows(0, 0);
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m + 1 < MT) rows(k, m + 1);
        if (m + 2 == MT && k + 1 < kDeep) columns(k + 1);
        if (m + 1 == MT && k + 1 < kDeep) rows(k + 1, 0);
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[m][j] = multiply_16(w[k & 1][j], a[m & 1], acc[m][j], j % 4, sw[k & 1][j / 4], m % 4, sa[k & 1][m / 4]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(acc[m][j]));
  };
  request_scales(0);
  request(tile0, 0);
  keep_scales(0, 0, 0);
  // two stages a turn, so that the halves are constants; one behind the last block is zeros that no memory is read for
  for (uint32_t base = 0; base < p.row_blocks; base += 2 * PARTS) {
#pragma unroll
    for (uint32_t s = 0; s < 2 * PARTS; s += PARTS) {
      const uint32_t half = s / PARTS, next = base + s + PARTS;
      stage_barrier();
      if (next % 16u == 0) request_scales(next);
      request(half ? tile0 : tile1, next);
      multiply(half ? tile1 : tile0, half);
      keep_scales(half ^ 1u, next % 16u, next);
    }
  }
  stage_barrier();  // no load may reach the LDS any more
  // A lane has four columns of 16 rows: stores of 64 bytes a row.  Through LDS, 16 rows at a time, they become 256 bytes a row (part c
  // of row r at c ^ r).
  f32x4 *const mine = reinterpret_cast<f32x4 *>(tile0) + wave * 256u;
  static_assert(NT == 4 && kWaves * 4096 <= kRows * kBytes, "64 columns, and room for 16 rows of every wavefront");
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < NT; ++j) mine[r * 16u + ((j * 4u + part) ^ r)] = acc[m][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t row = k * 4u + lane / 16u;
      const uint64_t i = tm * BM + m0 + m * 16u + row;
      const f32x4 v = mine[row * 16u + ((lane & 15u) ^ row)];
      if (i < p.n) write_columns(p, i, static_cast<uint64_t>(tn) * BN + (n0 - BM) + (lane & 15u) * 4u, v);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int BM, int BN, int WM, int WN, int PARTS, bool NEAR>
void launch_tiled(const ProductArgs &p, hipStream_t stream) {
  // rows in turns of at most 2^22 tiles, far below what a launch may have
  const uint32_t tiles_n = ceil_div(p.N, BN), turn = std::max(1u, (1u << 22) / tiles_n) * BM;
  for (uint64_t first = 0; first < p.n; first += turn) {
    ProductArgs q = p;
    q.out = p.out + first * p.N;
    q.n = static_cast<uint32_t>(std::min<uint64_t>(turn, p.n - first));
    if (p.row_ids) {
      q.row_ids = p.row_ids + first;
    } else {
      q.a.codes = p.a.codes + first * p.row_blocks * 16u;
      q.a.scales = p.a.scales + first * p.scale_stride;
      q.table_rows = p.table_rows > first ? static_cast<uint32_t>(p.table_rows - first) : 0u;
    }
    const uint32_t tiles_m = ceil_div(q.n, BM);
    hipLaunchKernelGGL((mx_product_tiled_kernel<BM, BN, WM, WN, PARTS, NEAR>), dim3(tile_blocks(tiles_m, tiles_n, kRowGroup)), dim3(WM * WN * kWave), 0,
                       stream, q, tiles_m, tiles_n);
  }
}

void launch_product(const ProductArgs &p, hipStream_t stream) {
  if (p.n <= 64) {
    const uint32_t mt = p.n <= 16 ? 1 : p.n <= 32 ? 2 : 4;
    const dim3 grid(ceil_div(p.N, 16), ceil_div(p.n, 16 * mt)), block(kFewWaves * kWave);
    if (mt == 1) hipLaunchKernelGGL(mx_product_few_kernel<1>, grid, block, 0, stream, p);
    else if (mt == 2) hipLaunchKernelGGL(mx_product_few_kernel<2>, grid, block, 0, stream, p);
    else hipLaunchKernelGGL(mx_product_few_kernel<4>, grid, block, 0, stream, p);
    return;
  }
  const uint64_t row_bytes = p.row_blocks * 16ull;
  if (std::max(p.table_rows, p.N) * row_bytes >= 0xFFFF0000ull) return launch_tiled<128, 128, 2, 2, 4, false>(p, stream);
  // The larger tile where there are enough of them to fill the chip twice and rows are long: 65,536 rows of 4,096 by 4,096 columns
  // 715 us against 912; 8,192 of 2,048 by 4,096: 61.5 against 64; but 65,536 of 1,024 by 1,024: 81 against 75; 232,965 of 602 by
  // 256: 86 against 66.
  if (p.row_blocks >= 64 && static_cast<uint64_t>(ceil_div(p.n, 256)) * ceil_div(p.N, 256) >= 512)
    return launch_tiled<256, 256, 2, 4, 8, true>(p, stream);
  launch_tiled<128, 128, 2, 2, 4, true>(p, stream);
}

// ---- gradients --------------------------------------------------------------------------------------
//   rows:    gx[i, f] (+)= sum_j g[i, j] W[j, f]                 P = g,   Q = W,          R = N terms
//   weight:  gw[j, f] (+)= sum_i g[i, j] A[row_ids[i], f]        P = g^T, Q = A by id,    R = n terms
// Q's 4-bit values times their scales are exact in bf16 (one bit of fraction, eight of exponent).  g is split into three bf16
// terms of eight bits of fraction each by cutting off bits, which is exact and cannot overflow, so three bf16 products summed
// in 32 bits keep the accuracy of a 32-bit product.  A block of four wavefronts takes 128 rows of the result by 128
// columns, 32 terms at a time through LDS, where both operands lie with the terms of a row or column side by side; the next
// terms are on their way into registers meanwhile.  What that costs is the waits for them, vector instructions and LDS: over
// 169,343 rows of 128 by 128 vector instructions are under way for 29 % of the time and the matrix units busy for 15 (rows) and 17
// (weight); of 640 by 640 for 54 and 38 (rows), 44 and 31 (weight).
// The weight's gradient has few results and many terms: blockIdx.z takes its part of the terms, the parts' sums are added in
// order by a second launch, so results do not depend on scheduling.
constexpr uint32_t kGradTile = 128, kGradTerms = 32;
// Where 8 of a row's 32 terms lie: as in the product, so that the 16 lanes that read one part of 16 rows meet all banks once.
constexpr uint32_t kGradQ = kGradTile * kGradTerms + kGradTile;
// Q's rows are written 8 apart by neighbouring lanes: 16 bytes more behind every eighth spread those over the banks as well.
__device__ __forceinline__ uint32_t grad_q_at(uint32_t row, uint32_t part) {
  return row * kGradTerms + ((row >> 3) + ((part + (row >> 2) - (row >> 3)) & 3u)) * 8u;
}
__device__ __forceinline__ uint32_t grad_at(uint32_t row, uint32_t part) { return row * kGradTerms + ((part ^ (row >> 2)) & 3u) * 8u; }

struct GradArgs {
  float *out;        // [M, F], or the parts' sums [parts, M, F]
  const float *g;    // [n, N]
  MxRows q;
  uint32_t q_rows;   // rows of Q's table: an id beyond them names a row of zeros
  const uint32_t *row_ids;
  uint32_t M, R, F, g_stride, row_blocks, scale_stride;
  uint32_t part_terms;        // terms a part sums (a multiple of kGradTerms)
  uint32_t tiles_m, tiles_f;  // of the rows' gradient
  int accumulate;
  bool streamed;  // the output goes past the caches
};

// x = hi + mid + lo, each the upper half of its word, exactly for finite x; an infinity or NaN goes to hi alone.
__device__ __forceinline__ void split3(float x, bool finite, uint32_t *hi, uint32_t *mid, uint32_t *lo) {
  const uint32_t b = __float_as_uint(x);
  const bool fine = finite || (b & 0x7F800000u) != 0x7F800000u;
  const float rest = fine ? x - __uint_as_float(b & 0xFFFF0000u) : 0.0f;
  const float m = __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
  *hi = b | (!finite && (b & 0x7FFFFFFFu) > 0x7F800000u ? 0x400000u : 0u);  // a NaN whose upper bits are an infinity's
  *mid = __float_as_uint(m);
  *lo = __float_as_uint(rest - m);
}
// The upper halves of two words.
__device__ __forceinline__ uint32_t upper_halves(uint32_t first, uint32_t second) { return __builtin_amdgcn_perm(second, first, 0x07060302u); }

// Whole stages load without branches, so that a wait is for the oldest loads alone: rows and columns of the tile that the result does
// not have read some other of it, ids that the table does not have read its first row and count as zeros.  What is left of the
// terms is loaded one by one.
// Weight: two stages of loads are on their way while a third is multiplied (640 by 640 over 169,343 rows: 832 -> 624 us, with the
// parts' sum, 128 by 128: 41 -> 33); it has blocks for two on a compute unit anyway.  Rows: one stage, and the registers for three
// blocks, are better (169,343 by 128 by 128: 38 us against 46).
template <bool WEIGHT, bool IDS>
__global__ __launch_bounds__(256, WEIGHT ? 2 : 3) void mx_grad_kernel(GradArgs p) {
  __shared__ __attribute__((aligned(16))) uint16_t sp0[3][kGradTile * kGradTerms], sp1[3][kGradTile * kGradTerms], sq0[kGradQ], sq1[kGradQ];
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = wave_of_block(), r = lane & 15u, part = lane >> 4;
  uint32_t tm = blockIdx.x, tf = blockIdx.y;
  if (!WEIGHT) {
    tile_of(p.tiles_f, p.tiles_m >= kXcdTiles, 1, &tm, &tf);
    if (tm >= p.tiles_m) return;
  }
  const uint64_t m0 = static_cast<uint64_t>(tm) * kGradTile;
  const uint32_t f0 = tf * kGradTile;
  const uint64_t begin = static_cast<uint64_t>(blockIdx.z) * p.part_terms;
  const uint64_t end = min(static_cast<uint64_t>(p.R), begin + p.part_terms);
  // P: a thread takes 16 terms of one row: neighbouring threads have neighbouring rows where those are g's columns, otherwise two
  // threads share a row.  Q: four columns of four terms.
  const uint32_t pm = WEIGHT ? (wave & 1u) * kWave + lane : t >> 1, pk = WEIGHT ? (wave >> 1) * 16u : (t & 1u) * 16u;
  const uint32_t qf = (t & 31u) * 4u, qk = (t >> 5) * 4u;
  const uint32_t m = static_cast<uint32_t>(min(m0 + pm, p.M - 1ull)), col = f0 + qf < p.F ? f0 + qf : 0u;
  float g[2][16];
  uint32_t code[2][4], scale[2][4], absent[2], id[4];
  auto look_up = [&](uint32_t stage, uint32_t *ids) __attribute__((always_inline)) {
    const uint64_t k0 = begin + static_cast<uint64_t>(stage) * kGradTerms;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) ids[i] = IDS ? (p.row_ids + k0)[qk + i] : static_cast<uint32_t>(k0) + qk + i;
  };
  auto request = [&](uint32_t stage, const uint32_t *ids, int u) __attribute__((always_inline)) {
    const uint64_t k0 = begin + static_cast<uint64_t>(stage) * kGradTerms;
    if (WEIGHT) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) g[u][i] = (p.g + (k0 + pk + i) * p.g_stride)[m];
    } else {
      const float *src = p.g + static_cast<uint64_t>(m) * p.g_stride + k0 + pk;
#pragma unroll
      for (uint32_t i = 0; i < 16; i += 4) {
        const FloatQuad q = *reinterpret_cast<const FloatQuad *>(src + i);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) g[u][i + k] = q[k];
      }
    }
    absent[u] = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t row = ids[i] < p.q_rows ? ids[i] : 0u;
      if (ids[i] >= p.q_rows) absent[u] |= 1u << i;
      code[u][i] = *reinterpret_cast<const uint16_t *>(p.q.codes + static_cast<uint64_t>(row) * (p.row_blocks * 16u) + col / 2u);
      scale[u][i] = p.q.scales[static_cast<uint64_t>(row) * p.scale_stride + col / kMxBlock];
    }
  };
  auto request_some = [&](uint64_t k0) {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const uint64_t k = k0 + pk + i;
      g[0][i] = k < end ? p.g[WEIGHT ? k * p.g_stride + m : static_cast<uint64_t>(m) * p.g_stride + k] : 0.0f;
    }
    absent[0] = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint64_t k = k0 + qk + i;
      uint32_t row = kNoSlot;
      if (k < end) row = IDS ? p.row_ids[k] : static_cast<uint32_t>(k);
      code[0][i] = scale[0][i] = 0;
      if (row < p.q_rows) {
        code[0][i] = *reinterpret_cast<const uint16_t *>(p.q.codes + static_cast<uint64_t>(row) * (p.row_blocks * 16u) + col / 2u);
        scale[0][i] = p.q.scales[static_cast<uint64_t>(row) * p.scale_stride + col / kMxBlock];
      }
    }
  };
  auto keep_g = [&](int u, uint16_t (*sp)[kGradTile * kGradTerms], bool finite) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < 16; i += 8) {
      uint32_t s[3][8];
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) split3(g[u][i + k], finite, &s[0][k], &s[1][k], &s[2][k]);
#pragma unroll
      for (int c = 0; c < 3; ++c)
        *reinterpret_cast<u32x4 *>(&sp[c][grad_at(pm, (pk + i) / 8u)]) = u32x4{upper_halves(s[c][0], s[c][1]), upper_halves(s[c][2], s[c][3]),
                                                               upper_halves(s[c][4], s[c][5]), upper_halves(s[c][6], s[c][7])};
    }
  };
  auto keep = [&](int u) __attribute__((always_inline)) {
    uint16_t(*const sp)[kGradTile * kGradTerms] = u ? sp1 : sp0;
    uint16_t *const sq = u ? sq1 : sq0;
    float probe = 0.0f;  // NaN where one of them is an infinity or NaN
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) probe = fmaf(g[u][i], 0.0f, probe);
    if (probe == 0.0f)
      keep_g(u, sp, true);
    else
      keep_g(u, sp, false);
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool there = !(absent[u] >> i & 1u);
      e2m1_decode4(there ? code[u][i] : 0u, there ? e8m0_value(scale[u][i]) : 0.0f, v[i]);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f)
      *reinterpret_cast<uint2 *>(&sq[grad_q_at(qf + f, qk / 8u) + qk % 8u]) =
          make_uint2(upper_halves(__float_as_uint(v[0][f]), __float_as_uint(v[1][f])), upper_halves(__float_as_uint(v[2][f]), __float_as_uint(v[3][f])));
  };
  const uint32_t wm = wave / 2u * 64u, wf = wave % 2u * 64u;
  f32x4 acc[4][4] = {};
  auto multiply = [&](int u) __attribute__((always_inline)) {
    uint16_t(*const sp)[kGradTile * kGradTerms] = u ? sp1 : sp0;
    const uint16_t *const sq = u ? sq1 : sq0;
    bf16x8 q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const bf16x8 *>(&sq[grad_q_at(wf + j * 16 + r, part)]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        const bf16x8 a = *reinterpret_cast<const bf16x8 *>(&sp[s][grad_at(wm + i * 16 + r, part)]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q[j], a, acc[i][j], 0, 0, 0);
      }
  };
  // Stages take the halves of LDS in turn, so one barrier a stage is enough: who writes a half has passed the barrier behind its last reads.
  const uint32_t full = p.q_rows && end > begin ? static_cast<uint32_t>((end - begin) / kGradTerms) : 0u;
  if (!WEIGHT && full) {
    uint32_t ids[4];
    look_up(0, ids);
    request(0, ids, 0);
    for (uint32_t s = 0; s < full; ++s) {
      keep(0);
      __syncthreads();
      if (s + 1u < full) {
        look_up(s + 1u, ids);
        request(s + 1u, ids, 0);
      }
      multiply(0);
      __syncthreads();
    }
  } else if (full) {
    const uint32_t last = full - 1u;
    uint32_t id0[4], id1[4];
    look_up(0, id0);
    look_up(min(1u, last), id1);
    look_up(min(2u, last), id);
    request(0, id0, 0);
    request(min(1u, last), id1, 1);
    uint32_t s = 0;
    auto stage = [&](int u, bool ahead) __attribute__((always_inline)) {
      keep(u);
      __syncthreads();
      if (ahead) {
        uint32_t next[4];
        look_up(min(s + 3u, last), next);
        request(s + 2u, id, u);
#pragma unroll
        for (int i = 0; i < 4; ++i) id[i] = next[i];
      }
      multiply(u);
      ++s;
    };
    while (s + 3u < full) {
      stage(0, true);
      stage(1, true);
    }
    if (s + 2u < full) {  // three left, two or one
      stage(0, true);
      stage(1, false);
      stage(0, false);
    } else {
      stage(0, false);
      if (s < full) stage(1, false);
    }
  }
  for (uint64_t k0 = begin + static_cast<uint64_t>(full) * kGradTerms; k0 < end; k0 += kGradTerms) {
    request_some(k0);
    __syncthreads();
    keep(0);
    __syncthreads();
    multiply(0);
  }
  __syncthreads();
  // rows of 64 columns through LDS, as the product's
  f32x4 *const mine = reinterpret_cast<f32x4 *>(&sp0[0][0]) + wave * 256u;
  static_assert(sizeof(sp0) >= 4 * 256 * sizeof(f32x4), "room for 16 rows of every wavefront");
#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[r * 16u + ((j * 4u + part) ^ r)] = acc[m][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t row = k * 4u + lane / 16u, f = f0 + wf + (lane & 15u) * 4u;
      const uint64_t i = m0 + wm + m * 16u + row;
      f32x4 v = mine[row * 16u + ((lane & 15u) ^ row)];
      if (i >= p.M) continue;
      float *dst = p.out + (static_cast<uint64_t>(blockIdx.z) * p.M + i) * p.F + f;
      if (f + 4u <= p.F) {
        if (p.accumulate) {
          const FloatQuad old = *reinterpret_cast<const FloatQuad *>(dst);
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] += old[c];
        }
        store_quad(dst, FloatQuad{v.x, v.y, v.z, v.w}, p.streamed);
      } else {
#pragma unroll
        for (uint32_t c = 0; c < 3; ++c)
          if (f + c < p.F) dst[c] = p.accumulate ? dst[c] + v[c] : v[c];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// out (+)= the sum of `parts` arrays of `count` floats, in order: four wavefronts take every fourth part of 64 values, eight
// loads at a time, and the first adds up what they have.
__global__ __launch_bounds__(256) void sum_parts_kernel(float *__restrict__ out, const float *__restrict__ from, uint64_t count,
                                                        uint32_t parts, int accumulate) {
  __shared__ float sums[3][kWave];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = wave_of_block();
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * kWave + lane;
  float sum = 0.0f;
  if (i < count) {
#pragma unroll 8
    for (uint32_t k = wave; k < parts; k += 4) sum += from[k * count + i];
  }
  if (wave) sums[wave - 1][lane] = sum;
  __syncthreads();
  if (wave || i >= count) return;
  sum += sums[0][lane];
  sum += sums[1][lane];
  sum += sums[2][lane];
  out[i] = accumulate ? out[i] + sum : sum;
}

struct Parts {
  uint32_t count, terms;
};
// Parts of the weight's gradient: 512 blocks, two for a compute unit, and none of fewer than 256 terms (169,343 rows of 640 by 640:
// 0.62 ms with 512; when that took 1.0, 256 took 2.0 and 1,024 took 1.0).
Parts weight_parts(uint32_t n, uint32_t N, uint32_t F) {
  const uint64_t tiles = static_cast<uint64_t>(ceil_div(N, kGradTile)) * ceil_div(F, kGradTile);
  const uint64_t want = std::max<uint64_t>(1, std::min<uint64_t>(512 / tiles, n / 256));
  const uint64_t terms = (n + want - 1) / want;
  Parts p;
  p.terms = static_cast<uint32_t>(std::min<uint64_t>((terms + kGradTerms - 1) / kGradTerms * kGradTerms, 0xFFFFFFE0u));
  p.count = std::max(1u, ceil_div(n, std::max(p.terms, 1u)));
  return p;
}

bool table_aligned(const uint8_t *codes, const uint8_t *scales) { return aligned_to(codes, 16) && aligned_to(scales, 4); }

}  // namespace
}  // namespace nts

using namespace nts;

extern "C" {

int nts_mxfp4_quantize(uint8_t *codes, uint8_t *scales, const float *x, uint32_t n, uint32_t F, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_mxfp4_quantize");
  if (F == 0 || F > kMostWidth) return fail(NTS_ERR_INVALID, "nts_mxfp4_quantize: F is 0 or above 2^17");
  if (n == 0) return NTS_OK;
  if (!codes || !scales || !x) return fail(NTS_ERR_INVALID, "nts_mxfp4_quantize: null pointer");
  if (!table_aligned(codes, scales)) return fail(NTS_ERR_INVALID, "nts_mxfp4_quantize: codes need 16-byte, scales 4-byte alignment");
  const uint32_t row_blocks = mx_blocks(F);
  const uint64_t blocks = static_cast<uint64_t>(n) * row_blocks;
  if (blocks > 0xFFFFFFFFull) return fail(NTS_ERR_INVALID, "nts_mxfp4_quantize: 2^32 blocks of 32 values or more");
  const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>((blocks + 32 * kQuantizeAhead - 1) / (32 * kQuantizeAhead), kMostBlocks)));
  hipLaunchKernelGGL(mx_quantize_kernel, grid, dim3(256), 0, stream, codes, scales, x, static_cast<uint32_t>(blocks), F, row_blocks,
                     mx_scale_stride(F));
  NTS_LAUNCH_CHECK("nts_mxfp4_quantize");
  return NTS_OK;
}

int nts_mxfp4_product(float *out, const uint8_t *codes, const uint8_t *scales, uint32_t table_rows, const uint32_t *row_ids,
                      uint32_t n, const uint8_t *w_codes, const uint8_t *w_scales, uint32_t N, uint32_t F, int accumulate,
                      nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_mxfp4_product");
  if (F == 0 || F > kMostWidth || N == 0 || N > kMostWidth)
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product: N or F is 0 or above 2^17");
  if (n == 0) return NTS_OK;
  if (!out || !w_codes || !w_scales || (table_rows && (!codes || !scales)))
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product: null pointer");
  if (!table_aligned(codes, scales) || !table_aligned(w_codes, w_scales))
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product: codes need 16-byte, scales 4-byte alignment");
  const ProductArgs p{out, {codes, scales}, table_rows, row_ids, n, {w_codes, w_scales}, N, mx_blocks(F), mx_scale_stride(F), accumulate,
                      static_cast<uint64_t>(n) * N * sizeof(float) >= kStreamedBytes};
  launch_product(p, stream);
  NTS_LAUNCH_CHECK("nts_mxfp4_product");
  return NTS_OK;
}

int nts_mxfp4_product_grad_rows(float *gx, const float *gout, const uint8_t *w_codes, const uint8_t *w_scales, uint32_t n,
                                uint32_t N, uint32_t F, int accumulate, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_mxfp4_product_grad_rows");
  if (F == 0 || F > kMostWidth || N == 0 || N > kMostWidth)
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product_grad_rows: N or F is 0 or above 2^17");
  if (n == 0) return NTS_OK;
  if (!gx || !gout || !w_codes || !w_scales) return fail(NTS_ERR_INVALID, "nts_mxfp4_product_grad_rows: null pointer");
  if (!table_aligned(w_codes, w_scales))
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product_grad_rows: codes need 16-byte, scales 4-byte alignment");
  const uint32_t terms = ceil_div(N, kGradTerms) * kGradTerms, cols = ceil_div(F, kGradTile);
  const GradArgs p{gx, gout, {w_codes, w_scales}, N, nullptr, n, N, F, N, mx_blocks(F), mx_scale_stride(F), terms, 0u, cols, accumulate,
                   static_cast<uint64_t>(n) * F * sizeof(float) >= kStreamedBytes};
  // launches of at most 2^24 - 1 blocks: rows of the result in turns
  const uint32_t turn = (kMostBlocks / cols - kXcdTiles) * kGradTile;
  for (uint64_t first = 0; first < n; first += turn) {
    GradArgs q = p;
    q.out = gx + first * F, q.g = gout + first * N;
    q.M = static_cast<uint32_t>(std::min<uint64_t>(turn, n - first));
    q.tiles_m = ceil_div(q.M, kGradTile);
    hipLaunchKernelGGL((mx_grad_kernel<false, false>), dim3(tile_blocks(q.tiles_m, cols, 1)), dim3(256), 0, stream, q);
    NTS_LAUNCH_CHECK("nts_mxfp4_product_grad_rows");
  }
  return NTS_OK;
}

size_t nts_mxfp4_product_grad_weight_work_bytes(uint32_t n, uint32_t N, uint32_t F) {
  if (N == 0 || F == 0 || N > kMostWidth || F > kMostWidth) return 0;
  const Parts parts = weight_parts(n, N, F);
  return parts.count > 1 ? static_cast<size_t>(parts.count) * N * F * sizeof(float) : 0;
}

int nts_mxfp4_product_grad_weight(float *gw, const float *gout, const uint8_t *codes, const uint8_t *scales,
                                  uint32_t table_rows, const uint32_t *row_ids, uint32_t n, uint32_t N, uint32_t F,
                                  int accumulate, void *work, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_mxfp4_product_grad_weight");
  if (F == 0 || F > kMostWidth || N == 0 || N > kMostWidth)
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product_grad_weight: N or F is 0 or above 2^17");
  if (!gw || (n && !gout) || (n && table_rows && (!codes || !scales)))
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product_grad_weight: null pointer");
  if (!table_aligned(codes, scales))
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product_grad_weight: codes need 16-byte, scales 4-byte alignment");
  const Parts parts = weight_parts(n, N, F);
  if (parts.count > 1 && (!work || !aligned_to(work, 16)))
    return fail(NTS_ERR_INVALID, "nts_mxfp4_product_grad_weight: needs nts_mxfp4_product_grad_weight_work_bytes of 16-byte-aligned work");
  GradArgs p{gw, gout, {codes, scales}, table_rows, row_ids, N, n, F, N, mx_blocks(F), mx_scale_stride(F), parts.terms, 0u, 0u, accumulate, false};
  if (parts.count > 1) p.out = static_cast<float *>(work), p.accumulate = 0;
  hipLaunchKernelGGL((row_ids ? mx_grad_kernel<true, true> : mx_grad_kernel<true, false>),
                     dim3(ceil_div(N, kGradTile), ceil_div(F, kGradTile), parts.count), dim3(256), 0, stream, p);
  NTS_LAUNCH_CHECK("nts_mxfp4_product_grad_weight");
  if (parts.count > 1) {
    const uint64_t count = static_cast<uint64_t>(N) * F;
    hipLaunchKernelGGL(sum_parts_kernel, dim3(ceil_div(count, kWave)), dim3(256), 0, stream, gw, static_cast<const float *>(work), count, parts.count, accumulate);
    NTS_LAUNCH_CHECK("sum_parts_kernel");
  }
  return NTS_OK;
}

}  // extern "C"
