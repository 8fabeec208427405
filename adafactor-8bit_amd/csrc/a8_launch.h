// Launches of more work than one grid takes: HIP's limit is 2^32 - 1 work-items along x.  No device code, so that
// a host compiler can check it.
#pragma once
#include <stdint.h>

namespace a8 {

constexpr int64_t most_groups(int threads) { return (int64_t)0xFFFFFFFF / threads; }

// f(first, count) for runs of at most `most` that cover [0, total) in order, up to the first non-zero result
template <typename F>
int in_runs(int64_t total, int64_t most, F&& f) {
  for (int64_t first = 0; first < total; first += most) {
    const int64_t left = total - first;
    if (const int e = f(first, left < most ? left : most)) return e;
  }
  return 0;
}

}  // namespace a8
