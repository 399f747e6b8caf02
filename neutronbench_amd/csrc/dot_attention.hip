// Attention of destinations over the float rows of their edges' sources: lanes, spans and entry points (kernels: dot_attention.hpp).
#include <algorithm>

#include "dot_args.hpp"
#include "edge_spans.hpp"
#include "launch_size.hpp"

namespace nts {
namespace {

constexpr uint32_t kMostHeadWidth = 256, kMostHeads = 1024;
// Above this bound (or without one) a row may be long enough to keep one walker busy after the others are done.
constexpr uint32_t kMostRowEdges = 256;
// Forward, up to so many destinations and edges, a block takes a destination, whatever the degrees (by address a walker does).
constexpr uint32_t kBlockRows = 64, kBlockEdges = 4096;
template <int KIND>
bool by_blocks(uint32_t rows, uint32_t edges, uint32_t max_degree) {
  return KIND == kForward && rows <= kBlockRows && edges <= kBlockEdges && (max_degree == 0 || max_degree > 16);
}
template <int KIND>
bool by_spans(uint32_t rows, uint32_t edges, uint32_t max_degree) {
  return KIND == kBySource || (!by_blocks<KIND>(rows, edges, max_degree) && (max_degree == 0 || max_degree > kMostRowEdges));
}

// How the lanes are laid out.  `slot_edges`: edges of a row for each of its slots.
struct Lanes {
  uint32_t nd, hw_shift, walker_shift, passes;
};
Lanes lanes_for(uint32_t units, uint32_t share, uint32_t D, uint64_t slot_edges) {
  Lanes l;
  l.nd = next_power(ceil_div(D, 16));
  // the query heads of a pass fit a word of the dropout's bits
  uint32_t hw = std::min(kWave / l.nd, next_power(units));
  while (hw > 1 && hw * share > 32u) hw /= 2;
  l.hw_shift = shift_of(hw);
  const uint32_t slots = std::min<uint32_t>(kWave / (l.nd * hw), next_power(static_cast<uint32_t>(std::min<uint64_t>(slot_edges, 64))));
  l.walker_shift = shift_of(l.nd * hw * slots);
  l.passes = ceil_div(units, hw);
  return l;
}

// Positions of a span: 256, so that a part's record is little beside its edges, but as few as `shortest` where that takes 8,192 wavefronts.
// That is 64, as a destination's parts have to be joined (393 destinations of 166 edges, 6 heads of 256 in fp16: 64 us; with 16 78), and by
// source, whose rows wait for each other and have few edges, 32, or 16 of walkers that share a wavefront (35,587 sources of 138,125 edges, a
// head of 20 in bf16: the step 109 us, with 32 158, with 64 194; 1,132 of 39,000, 16 query heads of 200 on 4: 328, 302 and 361).  And no more spans
// than 16,384 wavefronts have walkers or have records of 256 MB, but up to 256 spans whatever theirs take.
struct Spans {
  uint64_t positions, count;
  uint32_t length;
  size_t bytes;
};
template <int KIND>
Spans spans_for(uint32_t rows, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t D, const Lanes &l) {
  Spans s;
  const uint64_t shortest = KIND != kBySource ? 64 : l.walker_shift == 6 ? 32 : 16;
  const uint64_t records = 2 * record_size<KIND>(q_heads, heads, D) * sizeof(float), walkers = kWave >> l.walker_shift;
  s.positions = static_cast<uint64_t>(rows) * kRowCost + edges;
  const uint64_t most = std::max<uint64_t>(256, std::min<uint64_t>(16384 * walkers, (256ull << 20) / records));
  const uint64_t wanted = std::min(most, std::max({uint64_t{1024}, s.positions / 256, std::min(s.positions / shortest, 8192 * walkers)}));
  s.length = static_cast<uint32_t>(std::max<uint64_t>((s.positions + wanted - 1) / wanted, shortest));
  s.count = (s.positions + s.length - 1) / s.length;
  s.bytes = static_cast<size_t>(s.count * (records + sizeof(uint32_t)));
  return s;
}

// Lanes of a pass over `rows` rows of `edges` edges, in spans or (max_degree known) a walker per row.
template <int KIND>
Lanes lanes_of(uint32_t rows, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t D, uint32_t max_degree) {
  const bool spans = by_spans<KIND>(rows, edges, max_degree);
  return lanes_for(KIND == kBySource ? heads : q_heads, KIND == kBySource ? q_heads / heads : 1u, D,
                   by_blocks<KIND>(rows, edges, max_degree) ? kWave : spans ? (static_cast<uint64_t>(edges) / rows + 4) / 4 : (max_degree + 15) / 16);
}

// Lays out lanes and spans for `p`, whose operands are set, and runs it.
template <int KIND>
int run(DotArgs p, int type, uint32_t edges, uint32_t max_degree, void *work, hipStream_t stream) {
  if (p.rows == 0) return NTS_OK;
  const size_t size = type_size(type);
  const uint32_t piece = static_cast<uint32_t>(16 / size);
  const bool spans = by_spans<KIND>(p.rows, edges, max_degree);
  p.blocks = by_blocks<KIND>(p.rows, edges, max_degree);
  p.units = KIND == kBySource ? p.heads : p.q_heads;
  const Lanes l = lanes_of<KIND>(p.rows, edges, p.q_heads, p.heads, p.D, max_degree);
  p.hw_shift = l.hw_shift, p.walker_shift = l.walker_shift, p.passes = l.passes;
  p.chunks = ceil_div(p.D, piece);
  p.narrow = p.D < piece;
  p.partial_piece = p.D % piece != 0;
  p.ragged = p.partial_piece || p.chunks != l.nd * (16 / piece);
  if (spans) {
    const Spans s = spans_for<KIND>(p.rows, edges, p.q_heads, p.heads, p.D, l);
    p.positions = s.positions, p.span = s.length, p.spans = static_cast<uint32_t>(s.count);
    p.partial = static_cast<float *>(work);
    p.tail_row = reinterpret_cast<uint32_t *>(p.partial + s.count * 2 * record_size<KIND>(p.q_heads, p.heads, p.D));
  }
  const uint64_t width = static_cast<uint64_t>(KIND == kBySource ? p.q_heads : p.heads) * p.D * size;
  const void *const x = KIND == kBySource ? p.q : p.k, *const y = KIND == kBySource ? p.g : p.v;
  const bool near = !p.narrow && p.others <= (1u << 24) && p.others * std::max<uint64_t>(width, p.q_heads * sizeof(Ends)) <= kMostNear &&
                    p.D * size % 4 == 0 && aligned_to(x, 4) && aligned_to(y, 4);
  const auto launch_it = type == NTS_F32 ? dot_launch_f32 : type == NTS_BF16 ? dot_launch_bf16 : dot_launch_f16;
  return launch_it(KIND, p, l.nd, near, stream);
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

template <int KIND>
size_t spans_work(uint32_t rows, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t D, uint32_t max_degree) {
  if (rows == 0 || !by_spans<KIND>(rows, edges, max_degree)) return 0;
  return spans_for<KIND>(rows, edges, q_heads, heads, D, lanes_of<KIND>(rows, edges, q_heads, heads, D, max_degree)).bytes;
}
size_t ends_bytes(uint32_t Vd, uint32_t q_heads) { return (static_cast<size_t>(Vd) * q_heads * sizeof(Ends) + 15) / 16 * 16; }

}  // namespace
}  // namespace nts

using namespace nts;

extern "C" {

size_t nts_dot_attention_work_bytes(uint32_t Vd, uint32_t edges, uint32_t q_heads, uint32_t width, uint32_t max_degree) {
  if (q_heads == 0 || q_heads > kMostHeads || width == 0 || width > kMostHeadWidth) return 0;
  return spans_work<kForward>(Vd, edges, q_heads, q_heads, width, max_degree);
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
  if (spans_work<kForward>(Vd, edges, q_heads, q_heads, width, max_degree) && (!work || !aligned_to(work, 16)))
    return fail_in("nts_dot_attention", "needs nts_dot_attention_work_bytes of 16-byte-aligned work");
  DotArgs p{};
  p.out = out, p.lse = lse, p.q = q, p.k = k, p.v = v, p.offsets = co, p.ids = ri, p.rows = Vd, p.others = Vs;
  p.q_heads = q_heads, p.heads = heads, p.share = q_heads / heads, p.D = width, p.score_scale = score_scale, p.drop = drop_args(dropout);
  return run<kForward>(p, type, edges, max_degree, work, stream);
}

size_t nts_dot_attention_grad_work_bytes(uint32_t Vd, uint32_t Vs, uint32_t edges, uint32_t q_heads, uint32_t heads, uint32_t width,
                                         uint32_t max_degree) {
  if (q_heads == 0 || q_heads > kMostHeads || heads == 0 || heads > q_heads || width == 0 || width > kMostHeadWidth) return 0;
  const size_t mine = spans_work<kByDestination>(Vd, edges, q_heads, heads, width, max_degree);
  const size_t theirs = spans_work<kBySource>(Vs, edges, q_heads, heads, width, 0);
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
  p.lse = const_cast<float *>(lse), p.ends = static_cast<Ends *>(work), p.q = q, p.k = k, p.v = v, p.g = g;
  p.q_heads = q_heads, p.heads = heads, p.share = q_heads / heads, p.D = width, p.score_scale = score_scale, p.drop = drop_args(dropout);
  p.drop.step_kept = nullptr;
  void *const rest = static_cast<char *>(work) + ends_bytes(Vd, q_heads);
  p.out = gq, p.offsets = co, p.ids = ri, p.rows = Vd, p.others = Vs;
  if (const int status = run<kByDestination>(p, type, edges, max_degree, rest, stream)) return status;
  p.out = gk, p.out2 = gv, p.offsets = ro, p.ids = ci, p.rows = Vs, p.others = Vd;
  return run<kBySource>(p, type, edges, 0u, rest, stream);
}

}  // extern "C"
