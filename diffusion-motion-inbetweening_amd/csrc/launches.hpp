// A launch holds fewer than 2^32 threads: more blocks than that go out in several.
#pragma once
#include <stdint.h>

namespace cmdi {

// launch(first, count) for consecutive parts of `blocks` blocks of `threads` threads, at most 2^31 threads each; blocks are never parted
// within a run of `whole` of them (`first` counts runs).  Stops at the first result that is not 0 and returns it.
template <class F>
auto in_launches(int64_t blocks, int threads, int64_t whole, F&& launch) -> decltype(launch(int64_t(), unsigned())) {
    const int64_t runs = blocks / whole, most = ((int64_t)1 << 31) / threads / whole;
    for (int64_t first = 0; first < runs; first += most) {
        const auto r = launch(first, (unsigned)((runs - first < most ? runs - first : most) * whole));
        if (r) return r;
    }
    return {};
}

}  // namespace cmdi
