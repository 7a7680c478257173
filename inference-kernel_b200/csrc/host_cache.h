// What launchers ask the driver once per device (an occupancy, a kernel's
// shared-memory limit), kept for as long as the process runs.
#pragma once

#include <cstdint>
#include <mutex>

namespace aotk {

constexpr int kMaxDevices = 64;

// Up to kPerDevice values for each device, so that one device's never push out
// another's: a table shared by all of them overflowed with the second, whose small
// products then queried the driver up to seven times per call.  Keys are not 0.  Fixed
// storage (no allocation, so nothing to throw through the C ABI); a value that finds
// no room is worked out again.
template <int kPerDevice>
class DeviceCache {
  static_assert((kPerDevice & (kPerDevice - 1)) == 0, "a power of two");

 public:
  // The value of `key` on `device`: from `make(&value)` the first time, which returns
  // 0 or an error that is passed on and not kept.
  template <typename Make>
  int get(int device, uint64_t key, int* value, Make make) {
    if (device < 0 || device >= kMaxDevices) return make(value);
    Table& t = tables_[device];
    std::lock_guard<std::mutex> lock(t.mu);
    Entry* free = nullptr;
    // Fibonacci hashing: the top bits of a product with 2^64 / golden ratio.
    const uint64_t at = (key * 0x9E3779B97F4A7C15ull) >> 32;
    for (int i = 0; i < kPerDevice; ++i) {
      Entry& e = t.entries[(at + static_cast<uint64_t>(i)) & (kPerDevice - 1)];
      if (e.key == key) {
        *value = e.value;
        return 0;
      }
      if (e.key == 0) {
        free = &e;
        break;
      }
    }
    int v = 0;
    if (int status = make(&v)) return status;
    if (free) *free = Entry{key, v};
    *value = v;
    return 0;
  }

 private:
  struct Entry {
    uint64_t key = 0;
    int value = 0;
  };
  struct Table {
    std::mutex mu;
    Entry entries[kPerDevice];
  };
  Table tables_[kMaxDevices];
};

}  // namespace aotk
