"""How trees and lists of blocks are cut into parts (csrc/rows_plan.h): the memory of the partials and the grids rest on it."""
import os
import subprocess

import pytest

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include "rows_plan.h"
using namespace q27b;
#define CHECK(x, ...) do { if (!(x)) { printf("line %d: " #x " ", __LINE__); printf(__VA_ARGS__); printf("\n"); return 1; } } while (0)

// The most parts that U units of N tiles in all can come to: every unit one tile past a whole number of shares, none longer than a
// sequence can be.
static int64_t most(int64_t N, int64_t U, int share) { return std::min((N - U) / share + U, U * tree_parts(TREE_MAX_TILES, share)); }

static int trees(std::mt19937_64& r) {
  double used = 0;
  for (int n_sm : {1, 2, 20, 132, 148, 160})
    for (int64_t U = 1; U < (int64_t)65535 * 3; U += U < 3000 ? 1 : U / 50)
      for (int i = 0; i < 40; i++) {
        const int bits = (int)(r() % 17);
        const int64_t most_tiles = U * TREE_MAX_TILES, N = i == 0 ? U : i == 1 ? most_tiles : U + (int64_t)(r() % (uint64_t)((U << bits) + 1));
        const int64_t n = N < most_tiles ? N : most_tiles;
        const int share = tree_share(n, U, n_sm);
        CHECK(share >= 1 && share <= TREE_MAX_TILES, "N %lld U %lld share %d", (long long)n, (long long)U, share);
        const int64_t parts = most(n, U, share), grid = tree_grid(U, n_sm);
        CHECK(parts <= grid, "N %lld U %lld n_sm %d: share %d, parts %lld, grid %lld", (long long)n, (long long)U, n_sm, share, (long long)parts, (long long)grid);
        if ((double)parts / grid > used) used = (double)parts / grid;
      }
  // sequences as the kernel counts them: parts of a sequence, one after another, for every unit; the grid is that of all of them,
  // those that are empty too
  for (int i = 0; i < 100000; i++) {
    const int B = 1 + (int)(r() % 40), units = 1 + (int)(r() % 12), top = 1 << (1 + r() % 16), n_sm = 148;
    int n[40];
    int64_t N = 0, U = 0, sum = 0;
    for (int b = 0; b < B; b++) n[b] = r() % 4 ? (int)(r() % top) : 0, N += n[b], U += n[b] > 0;
    const int share = tree_share(N * units, U * units, n_sm);
    for (int b = 0; b < B; b++) {
      const int parts = tree_parts(n[b], share);
      int64_t last = 0;
      for (int z = 0; z < parts; z++) {  // every tile once, no part empty or longer than `share`
        const int64_t from = (int64_t)n[b] * z / parts, to = (int64_t)n[b] * (z + 1) / parts;
        CHECK(from == last && to > from && to - from <= share, "n %d parts %d share %d", n[b], parts, share);
        last = to;
      }
      CHECK(last == n[b], "n %d parts %d", n[b], parts);
      sum += parts;
    }
    CHECK(sum * units <= tree_grid((int64_t)B * units, n_sm), "B %d units %d: %lld parts", B, units, (long long)(sum * units));
  }
  printf("grid used %.3f\n", used);
  return 0;
}

static int blocks() {
  int64_t one = 0, pairs = 0;
  for (int n_sm : {20, 132, 148})
    for (int q8 = 0; q8 < 2; q8++)
      for (int64_t lists : {1, 2, 3, 4, 7, 8, 16, 17, 37, 64, 100, 128, 149, 256, 500, 1024, 5000, 65535 * 4})
        for (int k = 1; k <= 16384; k += k < 300 ? 1 : k / 9) {
          const BlocksPlan p = plan_blocks(lists, k, n_sm, q8);
          const int chunk = (k + p.nch - 1) / p.nch;
          CHECK(p.nch >= 1 && p.nch <= k && chunk <= SEL_CHUNK, "lists %lld k %d: %d chunks of %d", (long long)lists, k, p.nch, chunk);
          CHECK((int64_t)(p.nch - 1) * chunk < k, "k %d: an empty chunk", k);
          CHECK(!p.pairs || (q8 && lists * p.nch > n_sm), "pairs for %lld CTAs", (long long)(lists * p.nch));
          (p.pairs ? pairs : one)++;
        }
  CHECK(one > 0 && pairs > 0, "%lld %lld", (long long)one, (long long)pairs);  // both forms are taken
  return 0;
}

int main() {
  std::mt19937_64 r(1);
  return trees(r) || blocks();
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    import __graft_entry__ as ge
    d = tmp_path_factory.mktemp("plan")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(ge.PKG_DIR, "csrc"), str(d / "h.cpp"), "-o", str(d / "h")])
    return str(d / "h")


def test_parts_and_chunks(harness):
    """No plan has more parts than the grid and the partials have room for, every tile belongs to one part, no chunk is empty or
    longer than a CTA's list, and every form that a plan can ask for is asked for."""
    r = subprocess.run([harness], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
