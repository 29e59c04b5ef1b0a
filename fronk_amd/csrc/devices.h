// devices.h - what has to be done once for each device, in plain C++ so that it is
// tested on the host.
#pragma once
#include <stdint.h>

#include <atomic>

namespace fronk {

// The devices on which something was done.
typedef std::atomic<uint64_t> Devices;

// Does it (act: 0 for success) where it was not done yet; what failed is tried
// again the next time.
template <typename Act> int once_a_device(Devices* done, int device, Act act) {
  const uint64_t bit = (unsigned)device < 64 ? 1ull << device : 0;
  if (done->load(std::memory_order_acquire) & bit) return 0;
  const int rc = act();
  if (!rc) done->fetch_or(bit, std::memory_order_release);
  return rc;
}

}  // namespace fronk
