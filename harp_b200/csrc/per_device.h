// What a kernel's launches need to know or set up once for each device: a function
// attribute, an occupancy.  A static of a launcher holds one, so that a process that
// uses several devices sets each of them up, and an attempt that failed is made again.
#pragma once

#include <atomic>
#include <mutex>

namespace harp {

template <typename T>
class PerDevice {
 public:
  // `make()` of this device, called with the device current.  Its exceptions pass
  // through and nothing is kept of them.
  template <typename Make>
  T get(int device, Make&& make) {
    if (device < 0 || device >= kDevices) return make();
    Slot& s = slots_[device];
    if (!s.made.load(std::memory_order_acquire)) {
      std::lock_guard<std::mutex> lock(mu_);
      if (!s.made.load(std::memory_order_relaxed)) {
        s.value = make();
        s.made.store(true, std::memory_order_release);
      }
    }
    return s.value;
  }

 private:
  static constexpr int kDevices = 64;
  struct Slot {
    std::atomic<bool> made{false};
    T value{};
  };
  Slot slots_[kDevices];
  std::mutex mu_;
};

}  // namespace harp
