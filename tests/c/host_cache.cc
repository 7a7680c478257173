// DeviceCache by itself: every device keeps its own values, errors are not kept, a full
// table still answers, and threads that ask at once get one value.
#include "host_cache.h"

#include <cstdio>
#include <thread>
#include <vector>

#define CHECK(x)                                     \
  do {                                               \
    if (!(x)) {                                      \
      std::printf("failed line %d: %s\n", __LINE__, #x); \
      return 1;                                      \
    }                                                \
  } while (0)

namespace {

aotk::DeviceCache<256> cache;
aotk::DeviceCache<8> small;

// The keys of the occupancy queries: shared-memory size and cluster size.
uint64_t key_of(int smem, int cs) { return static_cast<uint64_t>(smem) << 8 | cs; }

}  // namespace

int main() {
  const int sizes[] = {33792, 50176, 66560, 78848, 82944, 99328, 105552, 115712};
  int made = 0;
  for (int round = 0; round < 3; ++round) {
    for (int device = 0; device < aotk::kMaxDevices; ++device) {
      for (int smem : sizes) {
        for (int cs = 2; cs <= 8; ++cs) {
          int v = -1;
          const int st = cache.get(device, key_of(smem, cs), &v, [&](int* p) {
            ++made;
            *p = device * 1000000 + smem * 10 + cs;
            return 0;
          });
          CHECK(st == 0 && v == device * 1000000 + smem * 10 + cs);
        }
      }
    }
    CHECK(made == aotk::kMaxDevices * 8 * 7);  // none was asked for twice
  }
  std::printf("ok every device keeps its values\n");

  int v = 5, tries = 0;
  auto fails = [&](int*) { ++tries; return 7; };
  CHECK(cache.get(3, 999, &v, fails) == 7 && cache.get(3, 999, &v, fails) == 7 && tries == 2 && v == 5);
  CHECK(cache.get(3, 999, &v, [](int* p) { *p = 4; return 0; }) == 0 && v == 4);
  CHECK(cache.get(3, 999, &v, fails) == 0 && v == 4 && tries == 2);
  std::printf("ok errors are passed on and not kept\n");

  made = 0;
  for (int round = 0; round < 2; ++round)
    for (uint64_t k = 1; k <= 20; ++k) {
      CHECK(small.get(0, k, &v, [&](int* p) { ++made; *p = static_cast<int>(k) * 3; return 0; }) == 0);
      CHECK(v == static_cast<int>(k) * 3);
    }
  CHECK(made == 20 + 12);
  for (int device : {-1, aotk::kMaxDevices})
    CHECK(small.get(device, 1, &v, [](int* p) { *p = 11; return 0; }) == 0 && v == 11);
  std::printf("ok a full table and an unknown device are asked again\n");

  static aotk::DeviceCache<64> shared;
  static int counts[32] = {};
  std::vector<std::thread> threads;
  bool right[8] = {};
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&right, t] {
      bool ok = true;
      for (int i = 0; i < 20000; ++i) {
        const int k = 1 + (i * 7 + t) % 32;
        int got = 0;
        shared.get(5, k, &got, [&](int* p) { *p = ++counts[k - 1] + k * 10; return 0; });
        ok = ok && got == 1 + k * 10;
      }
      right[t] = ok;
    });
  for (auto& t : threads) t.join();
  for (bool r : right) CHECK(r);
  for (int c : counts) CHECK(c == 1);
  std::printf("ok threads share one value\n");
  return 0;
}
