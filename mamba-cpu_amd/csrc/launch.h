// Launches of any number of workgroups.
#pragma once

#include <algorithm>
#include <cstdint>

namespace mcpu {

// A launch takes fewer than 2^32 threads a dimension; beyond that the runtime
// starts only some of the workgroups, without an error. f(first, count) launches
// the workgroups first to first + count - 1 of `groups` of `threads` each.
template <typename F> void launch_all(int64_t groups, int64_t threads, F&& f) {
  const int64_t most = ((int64_t{1} << 32) - 1) / threads;
  for (int64_t first = 0; first < groups; first += most)
    f(first, static_cast<unsigned>(std::min(most, groups - first)));
}

}  // namespace mcpu
