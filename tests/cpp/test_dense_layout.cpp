// Which rows of column sums a dense layer's product writes, and which its work has room for (csrc/dense_layout.hpp).  Prints "ok" and
// returns 0, or names what is wrong.
#include "dense_layout.hpp"

#include <stdio.h>

#include <initializer_list>
#include <vector>

using namespace nts;

// Every tile of rows is taken once, and only rows below `room` are written.
static bool fits(const Share &s, uint32_t room, const char *what, int type, uint32_t n, uint32_t N, uint32_t F) {
  std::vector<uint8_t> taken(s.tiles_m);
  for (uint32_t worker = 0; worker < launched_workers(s); ++worker) {
    if (!has_rows(worker, s.workers)) continue;
    if (worker >= room) {
      printf("%s: type %d, %u rows, %u by %u: worker %u writes a row behind %u\n", what, type, n, N, F, worker, room);
      return false;
    }
    for (uint64_t tile = worker; tile < s.tiles_m; tile += s.workers) {
      if (taken[tile]++) {
        printf("%s: type %d, %u rows, %u by %u: tile %llu is taken twice\n", what, type, n, N, F, static_cast<unsigned long long>(tile));
        return false;
      }
    }
  }
  for (uint8_t t : taken)
    if (t != 1) return printf("%s: type %d, %u rows, %u by %u: a tile is not taken\n", what, type, n, N, F), false;
  return true;
}

int main() {
  // what the gradient's products prepare: columns of x or of dz and as many terms as the other has, each once
  for (uint32_t columns : {1u, 127u, 131071u, 131072u})
    for (uint32_t terms : {1u, 33u, 131071u, 131072u})
      if (prepare_threads(columns, terms) / 256 > kMostBlocks || prepare_threads(columns, terms) < static_cast<uint64_t>(columns) * terms / 8)
        return printf("%u by %u: a launch of %llu threads\n", columns, terms, static_cast<unsigned long long>(prepare_threads(columns, terms))), 1;
  for (int type : {NTS_F32, NTS_BF16, NTS_F16})
    for (uint32_t n : {1u, 9u, 128u, 129u, 1000u, 1025u, 4099u, 4352u, 7424u, 9000u, 65536u, 65537u, 337000u})
      for (uint32_t N : {1u, 64u, 129u, 520u, 2048u, 2176u, 3900u, 4096u, 8192u, 131072u})
        for (uint32_t F : {1u, 31u, 128u, 512u, 520u, 2048u, 2176u, 4096u, 8192u, 131072u})
          for (int act : {NTS_ACT_RELU, NTS_ACT_GELU, NTS_ACT_SILU})
            for (uint32_t wanted = 0; wanted < 8; ++wanted) {
              const bool rows = wanted & 1, weight = wanted & 2, bias = wanted & 4;
              const Work w = grad_work(type, n, N, F, act, true, false, rows, weight, bias);
              if (w.bytes < w.parts_at || w.parts_at < w.sums_at + (bias ? 4ull * w.sums * N : 0)) return printf("sums do not fit the work\n"), 1;
              if (!w.again) return printf("z is computed again\n"), 1;
              for (bool aligned : {false, true})
                if (!fits(share_of(type, n, N, F, aligned), bias ? w.sums : 0xFFFFFFFFu, aligned ? "aligned" : "between aligned addresses", type, n, N, F)) return 1;
            }
  printf("ok\n");
  return 0;
}
