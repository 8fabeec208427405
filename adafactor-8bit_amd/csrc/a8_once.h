// What has to be set once for each device before a kernel's first launch there.  No device code, so that a
// host compiler can check it.
#pragma once
#include <stdint.h>

#include <atomic>

namespace a8 {

class OncePerDevice {
 public:
  // set() on the first call for the device, and again after a failure; the first 64 devices are remembered.
  // Its result, 0 for success.  Calls at the same time may both set.
  template <typename F>
  int operator()(int device, F&& set) {
    const uint64_t bit = device >= 0 && device < 64 ? (uint64_t)1 << device : 0;
    if (done_.load(std::memory_order_acquire) & bit) return 0;
    const int r = set();
    if (r == 0) done_.fetch_or(bit, std::memory_order_release);
    return r;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

}  // namespace a8
