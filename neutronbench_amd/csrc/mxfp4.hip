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
template <typename Index>
__global__ __launch_bounds__(256) void mx_quantize_kernel(uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                          const float *__restrict__ x, uint64_t n_blocks, uint32_t F,
                                                          uint32_t row_blocks, uint32_t scale_stride) {
  const uint32_t sub = threadIdx.x & 7u;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * 32u;
  for (uint64_t b = static_cast<uint64_t>(blockIdx.x) * 32u + threadIdx.x / 8u; b < n_blocks; b += step) {
    const Index row = static_cast<Index>(b) / static_cast<Index>(row_blocks);
    const uint32_t kb = static_cast<uint32_t>(static_cast<Index>(b) - row * static_cast<Index>(row_blocks));
    const uint32_t col = kb * kMxBlock + sub * 4u;
    const float *src = x + static_cast<uint64_t>(row) * F + col;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col + 4u <= F) {
      const Quad q = *reinterpret_cast<const Quad *>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = q.v[i];
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 3; ++i)
        if (col + i < F) v[i] = src[i];
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, kWave)));
    const uint32_t exponent = top >> 23;
    const bool fine = exponent < 255u;
    const uint32_t byte = !fine ? 255u : (exponent > 2u ? exponent - 2u : 0u);
    const float inverse = e8m0_inverse(fine ? byte : 0u);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) word |= e2m1_encode(v[i], inverse) << (4 * i);
    reinterpret_cast<uint16_t *>(codes)[b * 8u + sub] = static_cast<uint16_t>(fine ? word : 0u);
    // the block's scale, and the bytes that fill the last block's row up to whole words
    const uint32_t at = kb + sub;
    if (sub == 0 || (kb + 1 == row_blocks && at < scale_stride))
      scales[static_cast<uint64_t>(row) * scale_stride + at] = static_cast<uint8_t>(sub == 0 ? byte : 0u);
  }
}

// ---- product ----------------------------------------------------------------------------------------
//   out[i, j] (+)= sum_f A[row_ids[i], f] W[j, f]
// v_mfma_scale_f32_16x16x128 takes 16 rows of each operand, 128 values deep: lane l holds row l % 16, the 32 values of block
// l / 16, which are 16 consecutive bytes of the row, and that block's scale.  So the operands go from memory to registers as
// they lie.  W is the first operand: a lane then ends up with four neighbouring columns of one output row.

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
};

__device__ __forceinline__ i32x8 operand(i32x4 c) { return i32x8{c.x, c.y, c.z, c.w, 0, 0, 0, 0}; }

// A lane's part of 128 values of a row: block `block` of it; zeros (and a scale of 1) where there is no such block or row.
__device__ __forceinline__ void load_part(const MxRows &t, uint64_t row, bool there, uint32_t block, const ProductArgs &p,
                                          i32x4 *codes, uint32_t *scale) {
  *codes = i32x4{0, 0, 0, 0};
  *scale = 127u;
  if (there && block < p.row_blocks) {
    *codes = *reinterpret_cast<const i32x4 *>(t.codes + (row * p.row_blocks + block) * 16u);
    *scale = t.scales[row * p.scale_stride + block];
  }
}

template <int MT, int NT>
__global__ __launch_bounds__(256) void mx_product_kernel(ProductArgs p) {
  const uint32_t lane = threadIdx.x & (kWave - 1), r = lane & 15u, part = lane >> 4;
  const uint64_t tiles_n = (p.N + 16u * NT - 1) / (16u * NT), tiles_m = (static_cast<uint64_t>(p.n) + 16u * MT - 1) / (16u * MT);
  const uint64_t waves = static_cast<uint64_t>(gridDim.x) * (256 / kWave);
  for (uint64_t tile = wave_of_grid(); tile < tiles_m * tiles_n; tile += waves) {
    const uint64_t tm = tile / tiles_n, tn = tile - tm * tiles_n;
    uint64_t row[MT], col[NT];
    bool row_there[MT], col_there[NT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint64_t i = (tm * MT + m) * 16u + r;
      row_there[m] = i < p.n;
      row[m] = row_there[m] ? (p.row_ids ? p.row_ids[i] : i) : 0u;
      row_there[m] = row_there[m] && row[m] < p.table_rows;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      col[j] = (tn * NT + j) * 16u + r;
      col_there[j] = col[j] < p.N;
    }
    f32x4 acc[MT][NT] = {};
    for (uint32_t base = 0; base < p.row_blocks; base += 4) {
      i32x4 a[MT], w[NT];
      uint32_t sa[MT], sw[NT];
#pragma unroll
      for (int m = 0; m < MT; ++m) load_part(p.a, row[m], row_there[m], base + part, p, &a[m], &sa[m]);
#pragma unroll
      for (int j = 0; j < NT; ++j) load_part(p.w, col[j], col_there[j], base + part, p, &w[j], &sw[j]);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          acc[m][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w[j]), operand(a[m]), acc[m][j], 4, 4, 0,
                                                                       static_cast<int>(sw[j]), 0, static_cast<int>(sa[m]));
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint64_t i = (tm * MT + m) * 16u + r;
      if (i >= p.n) continue;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint64_t c = (tn * NT + j) * 16u + part * 4u;
        float *dst = p.out + i * p.N + c;
        if (c + 4u <= p.N) {
          Quad q{{acc[m][j].x, acc[m][j].y, acc[m][j].z, acc[m][j].w}};
          if (p.accumulate) {
            const Quad old = *reinterpret_cast<const Quad *>(dst);
#pragma unroll
            for (int k = 0; k < 4; ++k) q.v[k] += old.v[k];
          }
          *reinterpret_cast<Quad *>(dst) = q;
        } else {
#pragma unroll
          for (int k = 0; k < 3; ++k)
            if (c + k < p.N) dst[k] = p.accumulate ? dst[k] + acc[m][j][k] : acc[m][j][k];
        }
      }
    }
  }
}

// ---- gradients --------------------------------------------------------------------------------------
//   rows:    gx[i, f] (+)= sum_j g[i, j] W[j, f]                 P = g,   Q = W,          R = N terms
//   weight:  gw[j, f] (+)= sum_i g[i, j] A[row_ids[i], f]        P = g^T, Q = A by id,    R = n terms
// Q's 4-bit values times their scales are exact in bf16 (one bit of fraction, eight of exponent).  g is split into three bf16
// terms of eight bits of fraction each by cutting off bits, which is exact and cannot overflow, so three bf16 products summed
// in 32 bits keep the accuracy of a 32-bit product.  A block of four wavefronts takes 64 rows of the result by 64
// columns, 32 terms at a time through LDS, where both operands lie with the terms of a row or column side by side.
// The weight's gradient has few results and many terms: blockIdx.z takes its part of the terms, the parts' sums are added in
// order by a second launch, so results do not depend on scheduling.
constexpr uint32_t kGradRows = 64, kGradCols = 64, kGradTerms = 32, kGradPitch = kGradTerms + 8;

struct GradArgs {
  float *out;        // [M, F], or the parts' sums [parts, M, F]
  const float *g;    // [n, N]
  MxRows q;
  uint32_t q_rows;   // rows of Q's table: an id beyond them names a row of zeros
  const uint32_t *row_ids;
  uint32_t M, R, F, g_stride, row_blocks, scale_stride;
  uint32_t part_terms;  // terms a part sums (a multiple of kGradTerms)
  int accumulate;
};

// x = hi + mid + lo as bf16 bits, exactly for finite x; an infinity or NaN goes to hi alone.
__device__ __forceinline__ void split3(float x, uint16_t *hi, uint16_t *mid, uint16_t *lo) {
  const uint32_t b = __float_as_uint(x);
  const bool fine = (b & 0x7F800000u) != 0x7F800000u;
  const float h = __uint_as_float(b & 0xFFFF0000u);
  const float rest = fine ? x - h : 0.0f;
  const float m = __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
  *hi = static_cast<uint16_t>((b >> 16) | ((b & 0x7FFFFFFFu) > 0x7F800000u ? 0x40u : 0u));
  *mid = static_cast<uint16_t>(__float_as_uint(m) >> 16);
  *lo = static_cast<uint16_t>(__float_as_uint(rest - m) >> 16);
}

template <bool WEIGHT>
__global__ __launch_bounds__(256) void mx_grad_kernel(GradArgs p) {
  __shared__ __attribute__((aligned(16))) uint16_t sp[3][kGradRows][kGradPitch];
  __shared__ __attribute__((aligned(16))) uint16_t sq[kGradCols][kGradPitch];
  const uint32_t t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave, r = lane & 15u, part = lane >> 4;
  const uint64_t m0 = static_cast<uint64_t>(blockIdx.x) * kGradRows;
  const uint32_t f0 = blockIdx.y * kGradCols;
  const uint64_t begin = static_cast<uint64_t>(blockIdx.z) * p.part_terms;
  const uint64_t end = min(static_cast<uint64_t>(p.R), begin + p.part_terms);
  f32x4 acc[4] = {};
  for (uint64_t k0 = begin; k0 < end; k0 += kGradTerms) {
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kGradRows * kGradTerms / 256; ++i) {
      const uint32_t at = i * 256 + t;
      const uint32_t m = WEIGHT ? at % kGradRows : at / kGradTerms, k = WEIGHT ? at / kGradRows : at % kGradTerms;
      float v = 0.0f;
      if (m0 + m < p.M && k0 + k < end)
        v = WEIGHT ? p.g[(k0 + k) * p.g_stride + m0 + m] : p.g[(m0 + m) * p.g_stride + k0 + k];
      split3(v, &sp[0][m][k], &sp[1][m][k], &sp[2][m][k]);
    }
    {
      const uint32_t k = t / 8u, f = (t & 7u) * 8u;
      float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (k0 + k < end && f0 + f < p.F) {
        const uint64_t row = WEIGHT && p.row_ids ? p.row_ids[k0 + k] : k0 + k;
        if (row < p.q_rows)
          e2m1_decode8(*reinterpret_cast<const uint32_t *>(p.q.codes + row * p.row_blocks * 16u + (f0 + f) / 2u),
                       e8m0_value(p.q.scales[row * p.scale_stride + (f0 + f) / kMxBlock]), v);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sq[f + i][k] = static_cast<uint16_t>(__float_as_uint(v[i]) >> 16);
    }
    __syncthreads();
    bf16x8 q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const bf16x8 *>(&sq[j * 16 + r][part * 8]);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      const bf16x8 g = *reinterpret_cast<const bf16x8 *>(&sp[s][wave * 16 + r][part * 8]);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q[j], g, acc[j], 0, 0, 0);
    }
  }
  const uint64_t m = m0 + wave * 16 + r;
  if (m >= p.M) return;
  float *out = p.out + (static_cast<uint64_t>(blockIdx.z) * p.M + m) * p.F;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t f = f0 + j * 16 + part * 4 + i;
      if (f < p.F) out[f] = p.accumulate ? out[f] + acc[j][i] : acc[j][i];
    }
}

// out (+)= the sum of `parts` arrays of `count` floats, in order.
__global__ __launch_bounds__(256) void sum_parts_kernel(float *__restrict__ out, const float *__restrict__ from, uint64_t count,
                                                        uint32_t parts, int accumulate) {
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<uint64_t>(gridDim.x) * 256) {
    float sum = 0.0f;
    for (uint32_t k = 0; k < parts; ++k) sum += from[k * count + i];
    out[i] = accumulate ? out[i] + sum : sum;
  }
}

struct Parts {
  uint32_t count, terms;
};
// Parts of the weight's gradient: enough blocks for the chip, none of fewer than 256 terms.
Parts weight_parts(uint32_t n, uint32_t N, uint32_t F) {
  const uint64_t tiles = static_cast<uint64_t>(ceil_div(N, kGradRows)) * ceil_div(F, kGradCols);
  const uint64_t want = std::max<uint64_t>(1, std::min<uint64_t>(1024 / tiles, n / 256));
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
  const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>((blocks + 31) / 32, kMostBlocks)));
  if (blocks <= 0xFFFFFFFFull)
    hipLaunchKernelGGL(mx_quantize_kernel<uint32_t>, grid, dim3(256), 0, stream, codes, scales, x, blocks, F, row_blocks,
                       mx_scale_stride(F));
  else
    hipLaunchKernelGGL(mx_quantize_kernel<uint64_t>, grid, dim3(256), 0, stream, codes, scales, x, blocks, F, row_blocks,
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
  const ProductArgs p{out, {codes, scales}, table_rows, row_ids, n, {w_codes, w_scales}, N, mx_blocks(F), mx_scale_stride(F), accumulate};
  const uint64_t tiles = static_cast<uint64_t>(ceil_div(n, 32)) * ceil_div(N, 64);
  hipLaunchKernelGGL((mx_product_kernel<2, 4>), dim3(static_cast<uint32_t>(std::min<uint64_t>((tiles + 3) / 4, kMostBlocks))),
                     dim3(256), 0, stream, p);
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
  const uint32_t terms = ceil_div(N, kGradTerms) * kGradTerms;
  const GradArgs p{gx, gout, {w_codes, w_scales}, N, nullptr, n, N, F, N, mx_blocks(F), mx_scale_stride(F), terms, accumulate};
  // launches of at most 2^24 - 1 blocks: rows of the result in turns
  const uint32_t cols = ceil_div(F, kGradCols), turn = std::max(1u, kMostBlocks / cols) * kGradRows;
  for (uint64_t first = 0; first < n; first += turn) {
    GradArgs q = p;
    q.out = gx + first * F, q.g = gout + first * N;
    q.M = static_cast<uint32_t>(std::min<uint64_t>(turn, n - first));
    hipLaunchKernelGGL((mx_grad_kernel<false>), dim3(ceil_div(q.M, kGradRows), cols, 1), dim3(256), 0, stream, q);
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
  GradArgs p{gw, gout, {codes, scales}, table_rows, row_ids, N, n, F, N, mx_blocks(F), mx_scale_stride(F), parts.terms, accumulate};
  if (parts.count > 1) p.out = static_cast<float *>(work), p.accumulate = 0;
  hipLaunchKernelGGL((mx_grad_kernel<true>), dim3(ceil_div(N, kGradRows), ceil_div(F, kGradCols), parts.count), dim3(256), 0,
                     stream, p);
  NTS_LAUNCH_CHECK("nts_mxfp4_product_grad_weight");
  if (parts.count > 1) {
    const uint64_t count = static_cast<uint64_t>(N) * F;
    hipLaunchKernelGGL(sum_parts_kernel, dim3(static_cast<uint32_t>(std::min<uint64_t>((count + 255) / 256, 65536))), dim3(256),
                       0, stream, gw, static_cast<const float *>(work), count, parts.count, accumulate);
    NTS_LAUNCH_CHECK("sum_parts_kernel");
  }
  return NTS_OK;
}

}  // extern "C"
