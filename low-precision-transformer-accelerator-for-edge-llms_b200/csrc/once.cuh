// once.cuh -- what a launcher sets up once a device, whichever threads call it first.
#pragma once

#include <atomic>

namespace tl {

// Whether `set` has succeeded for device i, run by a thread that finds that it
// has not. Threads that come first together may each run it.
template <int N>
class Once {
  std::atomic<bool> done_[N] = {};

 public:
  template <typename F>
  bool operator()(int i, F set) {
    if (i < 0 || i >= N) return false;
    if (done_[i].load(std::memory_order_acquire)) return true;
    if (!set()) return false;
    done_[i].store(true, std::memory_order_release);
    return true;
  }
};

}  // namespace tl
