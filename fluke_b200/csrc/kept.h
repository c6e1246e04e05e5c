// kept.h -- a positive number that is asked for once and kept, for any number of host threads. An answer that is not positive is a failure
// (of this call's state, of the device's) and not kept: the next call asks again.
#pragma once
#include <atomic>

namespace fluke_sm100 {

template <typename Ask>
int kept(std::atomic<int> &slot, Ask ask) {
    int v = slot.load(std::memory_order_relaxed);   // threads that ask at the same time get the same answer
    if (v > 0) return v;
    v = ask();
    if (v > 0) slot.store(v, std::memory_order_relaxed);
    return v;
}

}  // namespace fluke_sm100
