"""How the workspace of the calls over pages grows (csrc/ws_buf.h), with a stand-in for the device's memory."""
import os
import subprocess

import pytest

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include "ws_buf.h"
// argv: free floats on the device, then requests ("s" with spare room, "e" exact, then a number); a line of state after each
int main(int argc, char** argv) {
  long long left = atoll(argv[1]);
  int asked = 0;
  q27b::GrowingWs ws;
  auto alloc = [&](size_t floats, float** p) {
    asked++;
    if ((long long)floats > left) return 7;
    left -= floats;
    *p = (float*)(uintptr_t)(0x1000 + asked);
    return 0;
  };
  for (int i = 2; i < argc; i++) {
    asked = 0;
    const int rc = ws.reserve((size_t)atoll(argv[i] + 1), argv[i][0] == 's', alloc);
    printf("%d %zu %zu %zu %d\n", rc, ws.live.floats, ws.outgrown.size(), ws.floats_held(), asked);
  }
}
"""


@pytest.fixture(scope="module")
def grow(tmp_path_factory):
    import __graft_entry__ as ge
    d = tmp_path_factory.mktemp("ws")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-include", "cstdint", "-I", os.path.join(ge.PKG_DIR, "csrc"),
                           str(d / "h.cpp"), "-o", str(d / "h")])

    def run(free, *requests):
        out = subprocess.check_output([str(d / "h"), str(free), *requests], text=True)
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]  # error, size, outgrown buffers, held, allocations
    return run


def test_a_growing_batch_leaves_few_buffers(grow):
    assert grow(10 ** 9, "s100", "s100", "s40", "s101", "s150", "s151", "s1000") == [
        (0, 100, 0, 100, 1), (0, 100, 0, 100, 0), (0, 100, 0, 100, 0), (0, 150, 1, 250, 1), (0, 150, 1, 250, 0),
        (0, 225, 2, 475, 1), (0, 1000, 3, 1475, 1)]


def test_what_fits_is_not_refused_for_the_spare_room(grow):
    """100 and 120 of 240 are to be had, 100 and 150 are not."""
    assert grow(240, "s100", "s120") == [(0, 100, 0, 100, 1), (0, 120, 1, 220, 2)]


def test_a_refusal_changes_nothing(grow):
    assert grow(240, "s100", "s141", "s100", "s130") == [(0, 100, 0, 100, 1), (7, 100, 0, 100, 2), (0, 100, 0, 100, 0), (0, 130, 1, 230, 2)]


def test_a_fixed_size_is_what_was_asked_for(grow):
    assert grow(10 ** 6, "s100", "e110", "e300") == [(0, 100, 0, 100, 1), (0, 110, 1, 210, 1), (0, 300, 2, 510, 1)]
