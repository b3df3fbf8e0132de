// attr_once.hpp -- "done once per device" flags of the launch code.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include <atomic>

namespace wj {

// hipFuncSetAttribute applies to the CURRENT device: a "done once" flag per kernel has to remember which devices it was
// done on, or a process that opens contexts on two devices launches on the second one without the attribute.  Threads on
// several devices share the flag: each marks the device that is current to itself.
struct AttrOnce {
  std::atomic<uint64_t> mask{0};
  static uint64_t bit() {
    int dev = 0;
    (void)hipGetDevice(&dev);
    return 1ull << (dev & 63);
  }
  bool need() const { return !(mask.load(std::memory_order_acquire) & bit()); }
  void done() { mask.fetch_or(bit(), std::memory_order_release); }
};

}  // namespace wj
