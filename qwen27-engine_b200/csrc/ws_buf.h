// Buffers of the per-device workspace, and how one grows. No CUDA here: memory comes from the caller's function.
#pragma once
#include <algorithm>
#include <cstddef>
#include <new>
#include <vector>

namespace q27b {

struct WsBuf {
  float* p = nullptr;
  size_t floats = 0;
};

// A buffer that captured graphs may name while later calls need more: what it was before stays allocated.
struct GrowingWs {
  WsBuf live;
  std::vector<WsBuf> outgrown;

  size_t floats_held() const {
    size_t n = live.floats;
    for (const WsBuf& b : outgrown) n += b.floats;
    return n;
  }
  // Room for `floats`, `spare`: and for half as much again as there was, so that a growing batch leaves few buffers behind, unless
  // only `floats` themselves are to be had. alloc(size, &pointer) gives 0 or an error, which is returned with nothing changed.
  template <class Alloc>
  int reserve(size_t floats, bool spare, Alloc alloc) {
    if (live.floats >= floats) return 0;
    outgrown.reserve(outgrown.size() + 1);  // (throws std::bad_alloc)
    WsBuf next;
    next.floats = spare ? std::max(floats, live.floats + live.floats / 2) : floats;
    int rc = alloc(next.floats, &next.p);
    if (rc && next.floats > floats) {
      next.floats = floats;
      rc = alloc(next.floats, &next.p);
    }
    if (rc) return rc;
    if (live.p) outgrown.push_back(live);
    live = next;
    return 0;
  }
};

}  // namespace q27b
