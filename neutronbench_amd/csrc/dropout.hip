// Dropout whose mask is never stored: y = x * 65536 / (65536 - t) where the value's number is at least t, else 0.  The backward
// pass is the same on the gradient.
// A thread takes 8 values, which share one drawing of ten rounds.  2,449,029 rows of 100 in 32 bits: 480 us, 4.08 TB/s, where a copy of as
// much reaches 4.7; vector instructions are under way for a quarter of the time.
#include <algorithm>

#include "launch_size.hpp"
#include "layers.hpp"

namespace nts {
namespace {

struct DropoutArgs {
  void *out;
  const void *in;
  uint32_t row0, F, groups, total;  // a launch's first row, columns, groups of 8 columns of a row and of the launch
  DropArgs drop;
  bool streamed;
};

constexpr uint32_t kAhead = 2;  // groups of a thread that are requested together
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs p) {
  const T *const in = static_cast<const T *>(p.in);
  T *const out = static_cast<T *>(p.out);
  const uint32_t step = drop_step(p.drop), first = blockIdx.x * (256u * kAhead) + threadIdx.x;
  if (p.drop.step_kept && blockIdx.x == 0 && threadIdx.x == 0) *p.drop.step_kept = step;
  float v[kAhead][8];
  uint32_t row[kAhead], group[kAhead];
#pragma unroll
  for (uint32_t u = 0; u < kAhead; ++u) {
    const uint32_t i = first + u * 256u;
    row[u] = i / p.groups, group[u] = i - row[u] * p.groups;
    if (i >= p.total) continue;
    const T *at = in + static_cast<uint64_t>(row[u]) * p.F + group[u] * 8u;
    if (group[u] * 8u + 8u <= p.F) {
      get_values<8>(at, v[u]);
    } else {
#pragma unroll
      for (uint32_t c = 0; c < 7; ++c)
        if (group[u] * 8u + c < p.F) v[u][c] = get_value(at + c);
    }
  }
#pragma unroll
  for (uint32_t u = 0; u < kAhead; ++u) {
    if (first + u * 256u >= p.total) return;
    const uint4 n = row_numbers(p.drop, step, p.row0 + row[u], group[u]);
#pragma unroll
    for (int c = 0; c < 8; ++c) v[u][c] = half_of(n, c) >= p.drop.threshold ? v[u][c] * p.drop.scale : 0.0f;
    T *at = out + static_cast<uint64_t>(row[u]) * p.F + group[u] * 8u;
    if (group[u] * 8u + 8u <= p.F) {
      put_values<8>(at, v[u], p.streamed);
    } else {
#pragma unroll
      for (uint32_t c = 0; c < 7; ++c)
        if (group[u] * 8u + c < p.F) put_value(at + c, v[u][c]);
    }
  }
}

}  // namespace
}  // namespace nts

using namespace nts;

extern "C" {

int nts_dropout(void *out, const void *in, int type, uint32_t n, uint32_t F, const nts_dropout_t *dropout, nts_stream_t stream) {
  NTS_TRACE_RANGE("nts_dropout");
  if (!known_type(type)) return fail(NTS_ERR_INVALID, "nts_dropout: unknown type");
  if (F == 0 || F > kMostColumns) return fail(NTS_ERR_INVALID, "nts_dropout: F is 0 or above 2^17");
  if (!dropout) return fail(NTS_ERR_INVALID, "nts_dropout: null pointer");
  if (bad_dropout(dropout)) return fail(NTS_ERR_INVALID, "nts_dropout: p is not within 0 .. 1");
  if (n == 0) return NTS_OK;
  if (!out || !in) return fail(NTS_ERR_INVALID, "nts_dropout: null pointer");
  if (!aligned_to(out, type_size(type)) || !aligned_to(in, type_size(type))) return fail(NTS_ERR_INVALID, "nts_dropout: a value's alignment");
  DropoutArgs p{out, in, 0u, F, ceil_div(F, 8), 0u, drop_args(dropout), static_cast<uint64_t>(n) * F * type_size(type) >= (32ull << 20)};
  const uint32_t turn = (1u << 30) / p.groups;  // rows of a launch
  for (uint64_t first = 0; first < n; first += turn) {
    const uint32_t rows = static_cast<uint32_t>(std::min<uint64_t>(turn, n - first));
    p.out = static_cast<char *>(out) + first * F * type_size(type), p.in = static_cast<const char *>(in) + first * F * type_size(type);
    p.row0 = static_cast<uint32_t>(first), p.total = rows * p.groups;
    const dim3 grid(ceil_div(p.total, 256 * kAhead));
    if (type == NTS_F32) hipLaunchKernelGGL(dropout_kernel<float>, grid, dim3(256), 0, stream, p);
    else if (type == NTS_BF16) hipLaunchKernelGGL(dropout_kernel<Bf16>, grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(dropout_kernel<F16>, grid, dim3(256), 0, stream, p);
    NTS_LAUNCH_CHECK("nts_dropout");
  }
  return NTS_OK;
}

}  // extern "C"
