// Ranges of rows that one launch of the norm takes.  Host arithmetic.
#pragma once
#include <algorithm>

namespace kfac {

// A launch has fewer than 2^32 threads; half of that here.
constexpr long LAUNCH_THREADS = 1L << 31;

// launch(first row, rows, workgroups) for ranges that cover `rows` rows in order, `per` rows to a workgroup of
// `threads` threads.
template <class F>
void for_row_ranges(long rows, int threads, int per, F&& launch) {
  const long most = LAUNCH_THREADS / threads * per;
  for (long first = 0; first < rows; first += most) {
    const long n = std::min(most, rows - first);
    launch(first, n, (unsigned)((n + per - 1) / per));
  }
}

}  // namespace kfac
