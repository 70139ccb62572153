// How trees and lists of blocks are cut into parts: plain arithmetic, on the host and (trees over pages) in the kernels.
#pragma once
#include "../../include/q27b_attn.h"

#include <algorithm>
#include <cstdint>

#ifdef __CUDACC__
#define Q27B_HD __host__ __device__
#else
#define Q27B_HD
#endif

namespace q27b {

// The tensor-core kernel of the tree (decode_tree.cu).
constexpr int TREE_ROWS = 128;         // (draft, head) rows of a KV head in a CTA
constexpr int TREE_MAX_TILES = 65536;  // position tiles of a sequence over pages
Q27B_HD inline int tree_row_tiles(int T) { return (T * Q27B_GQA + TREE_ROWS - 1) / TREE_ROWS; }
Q27B_HD inline int tree_tiles(int n) { return n > 0 ? (n + Q27B_BLOCK - 1) / Q27B_BLOCK : 0; }
// A unit is a row tile of a KV head of a sequence. Its ntot position tiles are cut into parts of equal length, at most `share`.
Q27B_HD inline int tree_parts(int ntot, int share) { return (ntot + share - 1) / share; }
// A batch: `share` so that the parts of all units come to w rounds of the SMs, for the w of the least time: a part takes some 9 us
// and 1.3 us a tile. N tiles and U units that are not empty: N / share + U / 2 parts or so. At most tree_grid(U, n_sm) of them.
Q27B_HD inline int64_t tree_rounds(int64_t U, int n_sm) { return (6 * U / 10) / n_sm + 1; }
Q27B_HD inline int64_t tree_share_of(int64_t N, int64_t U, int64_t w, int n_sm) {
  const int64_t d = w * n_sm - (55 * U + 99) / 100;
  return d < 1 ? N + 1 : (N + d - 1) / d;
}
Q27B_HD inline int64_t tree_grid(int64_t U, int n_sm) { return (tree_rounds(U, n_sm) + 2) * n_sm + U / 2 + 1; }
Q27B_HD inline int tree_share(int64_t N, int64_t U, int n_sm) {
  const int64_t w0 = tree_rounds(U, n_sm);
  int64_t best = 0, cost = 0;
  for (int64_t w = w0; w <= w0 + 2; w++) {
    const int64_t s = tree_share_of(N, U, w, n_sm), c = w * (13 * s + 90);
    if (w == w0 || c < cost) best = s, cost = c;
  }
  return (int)(best < 1 ? 1 : best < TREE_MAX_TILES ? best : TREE_MAX_TILES);
}

// Lists of blocks. Entries of a list that a CTA takes at most:
constexpr int SEL_CHUNK = 128;
// How lists of k blocks are cut into chunks, a CTA each: the plan of the least time in a model of the launch (us). A round of CTAs
// costs 5 and so much a block: a CTA of two tile groups, which has an SM to itself, 0.71 (q8_0) or 1.1 (f16), one of one group, two
// of which share an SM, 1.37. Measured on 14 shapes (1 to 512 lists of 16 to 1,024 blocks): 4 lists of 128 blocks 11.7 us in 32
// chunks of two groups and 14.4 in 64 of one; 16 of 64 14.3 and 15.0; 128 of 64 54.8 in pairs of CTAs and 56.6 in single ones; 256
// of 64 102.6 and 107.1; 256 of 16 34.1 and 39.0. The plan was within 4 % of the best of each. (One group with an SM to itself takes
// 0.97 a block, more than two groups, so CTAs that all find an SM have two.)
struct BlocksPlan {
  int nch;     // chunks
  bool pairs;  // CTAs of one tile group, two to an SM
};
inline BlocksPlan plan_blocks(int64_t lists, int k, int n_sm, bool q8) {
  BlocksPlan best = {1, false};
  double least = 1e300;
  int last = 0;
  for (int nch = (k + SEL_CHUNK - 1) / SEL_CHUNK; nch <= std::min(k, std::max(64, (k + SEL_CHUNK - 1) / SEL_CHUNK)); nch++) {
    const int chunk = (k + nch - 1) / nch;
    if (chunk == last) continue;  // the same chunks
    last = chunk;
    const int64_t ctas = lists * ((k + chunk - 1) / chunk);
    const double merge = 4e-4 * (double)(ctas * Q27B_GQA);
    const double rounds = (double)((ctas + n_sm - 1) / n_sm);
    const double two = rounds * (5.0 + (q8 ? 0.71 : 1.1) * chunk) + merge;
    if (two < least) least = two, best = {(k + chunk - 1) / chunk, false};
    const double one = (double)((ctas + 2 * n_sm - 1) / (2 * n_sm)) * (5.0 + 1.37 * chunk) + merge;
    if (q8 && ctas > n_sm && one < least) least = one, best = {(k + chunk - 1) / chunk, true};
  }
  return best;
}

}  // namespace q27b
