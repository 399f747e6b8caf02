// Attention of destinations over the float rows of their edges' sources, and its gradients.
//   forward       s_e = scale <q[d], k[src e]>, p_e = exp(s_e) / sum, out[d] = sum_e m_e p_e v[src e]; lse = log of the sum
//   by destination (offsets, ids: the edges by destination)
//                 p_e again from lse; c_e = m_e <g[d], v[src e]>, mean = sum_e p_e c_e,
//                 gq[d] = scale sum_e p_e (c_e - mean) k[src e] = scale (sum_e p_e c_e k[src e] - mean sum_e p_e k[src e])
//   by source     (offsets, ids: the edges by source)
//                 gk[s] = scale sum_e p_e (c_e - mean[dst e]) q[dst e], gv[s] = sum_e m_e p_e g[dst e]
// per query head, which shares its keys and values with the other heads of its group; m is the dropout's 0 or 1 / (1 - p).
// Both sums of gq and the mean come from one pass over the edges, so neither `out` nor the scores are kept.  lse was rounded, by
// half a step of its own size, which every p of a destination is off by: the pass sums them, too, and both passes divide by that.  One
// neighbour's p is then 1 whatever its score; with scores of 10^5 it was off by a hundredth.
#pragma once

#include "layers.hpp"

namespace nts {

enum Kind { kForward, kByDestination, kBySource };

// What the pass by destination leaves of a destination's head for the one by source: lse over log 2, mean, 1 / sum of p.
struct Ends {
  float base2, mean, share;
};

// A lane holds 16 columns of one head ("unit": a query head, by source a head of keys) in pieces of 16 bytes that lie ND lanes
// apart, so that neighbouring lanes read neighbouring pieces.  ND lanes (a power of two) cover a unit, 2^hw_shift units lie side by
// side, and further edges of the row go to further such sets of lanes ("slots"), joined at the end.  All slots of a row are a
// walker; a wavefront is one walker or several.  What an edge costs is vector instructions as much as memory: with 8
// columns a lane 98 of them for 8 query heads of 64 in bf16, whose 2.48 M edges took 541 us and kept the units busy for nine tenths of that.
struct DotArgs {
  void *out, *out2;  // out; gq; gk and gv
  float *lse;
  Ends *ends;  // [Vd, q_heads]
  const void *q, *k, *v, *g;
  const uint32_t *offsets, *ids;
  uint32_t rows, others;  // rows that are walked over; rows that ids may name
  uint32_t q_heads, heads, share, D, chunks;
  bool narrow, partial_piece, ragged;  // less than a piece; the last piece is not whole; that, or some lanes have no piece
  float score_scale;
  DropArgs drop;
  uint32_t units, hw_shift, walker_shift, passes;
  bool blocks;           // a block per row
  uint32_t span, spans;  // edges in spans of positions (edge_spans.hpp)
  uint64_t positions;
  float *partial;
  uint32_t *tail_row;
};

// Floats of a span's record.
template <int KIND>
__host__ __device__ __forceinline__ uint64_t record_size(uint32_t q_heads, uint32_t heads, uint32_t D) {
  if (KIND == kForward) return static_cast<uint64_t>(q_heads) * (D + 2u);
  if (KIND == kByDestination) return static_cast<uint64_t>(q_heads) * (2u * D + 2u);
  return 2ull * heads * D;
}

// Tables whose rows are read by 32-bit offsets have at most so many bytes.
constexpr uint64_t kMostNear = 0x60000000u;

// Runs one kind for rows of one type, with lanes and spans as `p` says; nd: lanes of a head, near: rows are read by 32-bit offsets.
int dot_launch_f32(int kind, const DotArgs &p, uint32_t nd, bool near, hipStream_t stream);
int dot_launch_bf16(int kind, const DotArgs &p, uint32_t nd, bool near, hipStream_t stream);
int dot_launch_f16(int kind, const DotArgs &p, uint32_t nd, bool near, hipStream_t stream);

}  // namespace nts
