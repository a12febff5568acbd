// cluster_count.h — how many clusters of one kernel and size a device holds side by side, asked once per device.
#pragma once

#include <atomic>

namespace oxg {

class ClusterCount {
 public:
  // query(): the number, or 0 or less where it could not be had: then this call goes by `otherwise`, and the next
  // one asks again.
  template <class Query>
  int get(int device, int otherwise, Query &&query) {
    const bool kept = device >= 0 && device < kDevices;
    if (kept) {
      const int n = known_[device].load(std::memory_order_relaxed);
      if (n > 0) return n;
    }
    const int n = query();
    if (n <= 0) return otherwise;
    if (kept) known_[device].store(n, std::memory_order_relaxed);
    return n;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> known_[kDevices] = {};
};

}  // namespace oxg
