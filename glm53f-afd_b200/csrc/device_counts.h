// Host only: a count that is asked of each device once and kept, such as how many clusters of a size it holds at a time.
#pragma once

#include <atomic>

namespace kda {

// CHOICES counts a device.  A caller never sees a count that is still being asked for: two that ask at once both ask, and both get the answer.  An
// answer below zero (the query failed) is 0 for this call and is asked for again by the next.
template <int CHOICES>
class DeviceCounts {
  public:
    template <typename Ask>
    int get(int device, int choice, Ask ask) {
        const bool kept = device >= 0 && device < kDevices;
        if (kept) {
            const int n = counts_[device][choice].load(std::memory_order_acquire);
            if (n != 0) return n - 1;
        }
        const int n = ask();
        if (n < 0) return 0;
        if (kept) counts_[device][choice].store(n + 1, std::memory_order_release);
        return n;
    }

  private:
    static constexpr int kDevices = 64;
    std::atomic<int> counts_[kDevices][CHOICES] = {};  // the count and one; 0: not asked for yet
};

}  // namespace kda
