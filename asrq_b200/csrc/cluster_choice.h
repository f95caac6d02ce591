// How many blocks (and warps) work on an item where a device may hold some cluster sizes and not others: host rules without CUDA, so that
// they can be tested with devices that are not at hand.
#pragma once

#include <cstdint>

namespace asrq {

constexpr int kRowsWarps = 8;  // of a block of the row kernel, at most
constexpr int kMaxSplit = 16;  // blocks of a cluster

struct RowsChoice {
  int split, warps;
  int64_t cost;
};
// Blocks an item and warps a block: the least (waves of resident blocks) x (chunks a warp walks, and 3 for a block's start and end, one
// more in a cluster).  us by (warps, blocks): 1x5 rows on 1500 keys (6, 8) 5.5, (8, 4) 5.7, (4, 4) 6.0, (8, 8) 9.2 in two waves; 16x5 on 150..1500
// (4, 1) 18.1, (6, 1) 17.5, (8, 1) 20.3, (4, 2) 20.6; 64x5 on 258 + 65 (6, 1) 34.4, (2, 1) 38.1, (4, 1) 42.3; 32x5 on 1500 (2, 1) 41.8, (4, 1) 44.9.
// slots(blocks of a cluster, warps of a block): the blocks that the device holds at once, 0: it holds no such cluster.
template <typename Slots>
RowsChoice choose_rows(uint32_t items, uint32_t chunks, Slots slots) {  // (32-bit divisions: the loop is host time of every call)
  RowsChoice best = {1, kRowsWarps, INT64_MAX};
  for (uint32_t s = 1; s <= uint32_t(kMaxSplit); s *= 2)
    for (uint32_t w = kRowsWarps; w >= 1; --w) {
      const uint32_t n = uint32_t(slots(int(s), int(w)));
      if (n == 0) continue;
      const int64_t cost = int64_t((items * s + n - 1) / n) * ((chunks + s * w - 1) / (s * w) + (s > 1 ? 4 : 3));
      if (cost < best.cost) best = {int(s), int(w), cost};
    }
  return best;
}
// What a device holds of clusters of `split` blocks: `held` of them by its own answer (negative: it has none to give).  Single blocks
// always run, a few at least.
inline int64_t slots_held(int held, int split, int sm_count) {
  if (held > 0) return int64_t(held) * split;
  return split == 1 ? sm_count : 0;
}

// Blocks an utterance of the selection: a block an SM, two where that leaves four; the lists of two at least (us with 16 | 8 | 4 | 2: 1 utterance of 5 x 51866
// 8.2 | 10.4 | 11.9 | 16.2, 9 of them 10.5 | 10.5 | 12.4 | 17.0, 18 14.6 | 13.2 | 12.4 | 17.5, 32 20.6 | 16.7 | 14.1 | 17.8, 64 of 8 x 51866
// 53.4 | 34.7 | 24.0 | 29.4, 200 of 4 x 10000 93.9 | 47.8 | 26.5 | 18.2).  Clusters of 16 are more than every device has to hold (8); fit(blocks): whether the
// segments are short enough, which they are with 8.
template <typename Fit>
int choose_select(int64_t utterances, int sm_count, bool holds_16, Fit fit) {
  int blocks = holds_16 ? 16 : 8;
  while (blocks > 2 && utterances * blocks > (blocks == 4 ? 2 : 1) * sm_count && fit(blocks / 2)) blocks /= 2;
  return blocks;
}

}  // namespace asrq
