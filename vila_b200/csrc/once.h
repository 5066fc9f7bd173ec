// Setup that a process does once per device, before its first launch of a kernel.
#pragma once
#include <atomic>
#include <mutex>

namespace vb {

// run(device, f): f() the first time, by whichever host thread comes first; the others wait until it is done.  f returns 0, or an error
// that run hands on, and the next call tries again.
class OncePerDevice {
  static constexpr int kMost = 64;      // devices beyond: f every time
  std::atomic<bool> done_[kMost] = {};
  std::mutex one_at_a_time_;

 public:
  template <typename F>
  int run(int device, F&& f) {
    const bool counted = device >= 0 && device < kMost;
    if (counted && done_[device].load(std::memory_order_acquire)) return 0;
    std::lock_guard<std::mutex> held(one_at_a_time_);
    if (counted && done_[device].load(std::memory_order_relaxed)) return 0;
    const int rc = f();
    if (rc == 0 && counted) done_[device].store(true, std::memory_order_release);
    return rc;
  }
};

}  // namespace vb
