// How the products of a dense layer and of its gradients are shared out, and what memory they take.  Host logic only.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

#include "launch_size.hpp"
#include "nts_hip.h"

namespace nts {

constexpr uint32_t kTile = 128, kTerms = 32, kPlane = kTile * kTerms;  // rows or columns of a tile, terms of a stage, values of both
constexpr uint32_t kWideTile = 256;

// Bytes of a prepared weight.
inline size_t prepared_bytes(uint32_t planes, uint32_t columns, uint32_t terms) {
  return static_cast<size_t>(ceil_div(columns, kTile)) * ceil_div(terms, kTerms) * kPlane * planes * 2u;
}
// Threads that prepare it, eight terms each; columns and terms of up to 2^17 take 2^31.
inline uint64_t prepare_threads(uint32_t columns, uint32_t terms) {
  return static_cast<uint64_t>(ceil_div(columns, kTile)) * kTile * ceil_div(terms, kTerms) * (kTerms / 8);
}
// Parts of a weight: three of 32 bits; beside dz in 32 bits, which is multiplied as bf16 parts, two of fp16; else the weight itself.
inline uint32_t planes_of(int type, bool dz32) { return type == NTS_F32 ? 3u : dz32 && type == NTS_F16 ? 2u : 1u; }
// Large products by large tiles, where there are enough of them for the chip and rows of many terms; in us by large tiles and by rows:
// 16,384 x 1,024 x 512 26 and 38, 65,536 x 256 x 1,024 42 and 63; of 256 terms 32,768 x 4,096 150 and 129; of 128 tiles 8,192 x 1,024 x 1,024
// 34 and 34.
inline bool by_wide_tiles(int type, uint32_t n, uint32_t N, uint32_t K) {
  return type != NTS_F32 && K >= 512 && K % 8 == 0 && static_cast<uint64_t>(ceil_div(n, kWideTile)) * ceil_div(N, kWideTile) >= 256;
}
// Bytes of a product's weight in the work: as the rows' kernel wants it, or turned for large tiles.
inline size_t weight_bytes(int type, uint32_t n, uint32_t columns, uint32_t terms, bool turned) {
  // operands between aligned addresses take the rows' kernel all the same
  return std::max(prepared_bytes(planes_of(type, false), columns, terms), turned && by_wide_tiles(type, n, columns, terms) ? static_cast<size_t>(columns) * terms * 2 : size_t{0});
}
// How a product's tiles of rows are shared out: every worker takes every `workers`-th of them and leaves a row of column sums.  aligned: the
// operands begin at multiples of 16 bytes, without which there are no large tiles.
struct Share {
  bool wide;
  uint32_t tiles_m, tiles_n, workers;
};
inline Share share_of(int type, uint32_t n, uint32_t N, uint32_t K, bool aligned) {
  Share s;
  s.wide = aligned && by_wide_tiles(type, n, N, K);
  s.tiles_m = ceil_div(n, s.wide ? kWideTile : kTile), s.tiles_n = ceil_div(N, s.wide ? kWideTile : kTile);
  // by rows two blocks to a compute unit, three of 16-bit values
  s.workers = s.wide ? s.tiles_m : std::min(s.tiles_m, std::max(8u, (type == NTS_F32 ? 512u : 768u) / s.tiles_n / 8u * 8u));
  return s;
}
// Rows of column sums that a product may leave, whatever its operands' alignment.
inline uint32_t most_workers(int type, uint32_t n, uint32_t N, uint32_t K) {
  return std::max(share_of(type, n, N, K, false).workers, share_of(type, n, N, K, true).workers);
}
// By rows, workers are launched in eights, one to a chiplet: those behind the last one have no rows.
inline uint32_t launched_workers(const Share &s) { return s.wide ? s.workers : ceil_div(s.workers, 8) * 8u; }
constexpr bool has_rows(uint32_t worker, uint32_t workers) { return worker < workers; }
// Parts of the weight's gradient, of few results and many terms: two blocks for a compute unit, and no part of fewer than 256 terms.
// (All tiles of a part on one chiplet, whose L2 then reads its rows once, took 620 us instead of 515 at 232,965 terms of 256 by 602: the parts
// are then a multiple of eight and fewer.)
struct Parts {
  uint32_t count, terms;
};
inline Parts weight_parts(uint32_t n, uint32_t N, uint32_t F) {
  const uint64_t tiles = static_cast<uint64_t>(ceil_div(N, kTile)) * ceil_div(F, kTile);
  const uint64_t want = std::max<uint64_t>(1, std::min<uint64_t>(512 / tiles, n / 256));
  const uint64_t terms = (n + want - 1) / want;
  Parts p;
  p.terms = static_cast<uint32_t>(std::min<uint64_t>((terms + kTerms - 1) / kTerms * kTerms, 0xFFFFFFE0u));
  p.count = std::max(1u, ceil_div(n, std::max(p.terms, 1u)));
  return p;
}

// The gradient's work: dz, the prepared weight, the parts of the bias's sums and of the weight's.
struct Work {
  bool from_y;   // y says what dz needs
  bool masked;   // and dz is made where it is read
  bool stored;   // dz is stored
  bool beside;   // the bias's sums are made beside the weight's gradient
  bool again;    // z is computed again
  bool dz32;     // and dz is stored in 32 bits, though the operands have 16
  size_t weight_at, sums_at, parts_at, bytes;
  uint32_t sums;  // rows of them that there is room for
  Parts parts;
};
inline Work grad_work(int type, uint32_t n, uint32_t N, uint32_t F, int act, bool dropout, bool has_y, bool rows, bool weight, bool bias) {
  Work w{};
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  // Where more than one tile of columns reads it, dz is made once: a step of 232,965 rows of 602 by 256 takes 1,506 us so, and
  // 1,685 where it is read; one of 337,000 of 100 by 128 takes 421 and 396.
  w.from_y = act == NTS_ACT_RELU && has_y;
  w.masked = w.from_y && F <= kTile && (weight || !bias);
  w.stored = !w.masked && (act != NTS_ACT_NONE || dropout) && n;
  w.beside = bias && weight && !w.stored;
  w.again = w.stored && act != NTS_ACT_NONE && !w.from_y;
  w.dz32 = w.again && type != NTS_F32;
  w.weight_at = w.stored ? up(static_cast<size_t>(n) * N * (type == NTS_F32 || w.dz32 ? 4u : 2u)) : 0;
  const size_t for_z = w.again ? weight_bytes(type, n, N, F, false) : 0;
  const size_t for_rows = !rows || !n ? 0 : w.dz32 ? prepared_bytes(planes_of(type, true), F, N) : weight_bytes(type, n, F, N, true);
  w.sums_at = w.weight_at + up(std::max(for_z, for_rows));
  w.parts = weight_parts(n, N, F);
  w.sums = w.beside ? w.parts.count : w.again ? most_workers(type, n, N, F) : static_cast<uint32_t>(std::min<uint64_t>(1024, ceil_div(n, 64)));
  w.parts_at = w.sums_at + (bias ? up(static_cast<size_t>(w.sums) * N * sizeof(float)) : 0);
  w.bytes = w.parts_at + (weight && w.parts.count > 1 ? static_cast<size_t>(w.parts.count) * N * F * sizeof(float) : 0);
  return w;
}

}  // namespace nts
