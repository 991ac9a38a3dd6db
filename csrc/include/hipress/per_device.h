// What is settled once for each device of the process.
#pragma once
#include <atomic>

namespace hipress {

constexpr int kMostDevices = 64;   // of a process; beyond them nothing is remembered

// A positive number for each device, found on the first use there.  Attributes of a kernel belong to the
// device that was current when they were set.  Only what was found is kept: a call that failed
// is made again.  Threads that come first together find the same.
class PerDevice {
 public:
  // `find(int* value)` returns zero or an error code, which get() returns too
  template <typename Find>
  int get(int device, Find find, int* value) {
    const bool kept = device >= 0 && device < kMostDevices;
    *value = kept ? values_[device].load(std::memory_order_acquire) : 0;
    if (*value > 0) return 0;
    const int rc = find(value);
    if (rc == 0 && kept) values_[device].store(*value, std::memory_order_release);
    return rc;
  }

 private:
  std::atomic<int> values_[kMostDevices] = {};
};

}  // namespace hipress
