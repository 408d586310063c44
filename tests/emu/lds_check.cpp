// cx_lds.hpp against a HIP of its own: two devices, an attribute call that fails.
#include <algorithm>
#include <cstdio>
#include <thread>
#include <vector>

typedef int hipError_t;
enum { hipSuccess = 0, hipFuncAttributeMaxDynamicSharedMemorySize = 8 };
static thread_local int device = 0;
static int limits[100], calls, fail;
static hipError_t hipGetDevice(int* d) { *d = device; return hipSuccess; }
static hipError_t hipFuncSetAttribute(const void*, int, int bytes) {
  ++calls;
  if (fail) return fail;
  limits[device] = bytes;
  return hipSuccess;
}
#include "cx_lds.hpp"

#define CHECK(c) if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; }

int main() {
  cx::LdsLimit x;
  CHECK(x.raise(nullptr, 70000) == 0 && limits[0] == 70000);
  CHECK(x.raise(nullptr, 70000) == 0 && x.raise(nullptr, 66000) == 0 && calls == 1 && limits[0] == 70000);
  // a second device has a limit of its own
  device = 1;
  CHECK(x.raise(nullptr, 66000) == 0 && limits[1] == 66000 && limits[0] == 70000);
  // a failure is reported, and the next call tries again
  device = 2;
  fail = 98;
  CHECK(x.raise(nullptr, 70000) == 98 && x.raise(nullptr, 70000) == 98);
  fail = 0;
  CHECK(x.raise(nullptr, 70000) == 0 && limits[2] == 70000);
  // more devices than are remembered
  device = 80;
  CHECK(x.raise(nullptr, 70000) == 0 && x.raise(nullptr, 80000) == 0 && limits[80] == 80000);
  // threads with different needs: the limit is at the highest in the end
  cx::LdsLimit y;
  std::vector<std::thread> t;
  for (int i = 0; i < 8; ++i)
    t.emplace_back([&y, i] { for (int b = 0; b < 2000; ++b) y.raise(nullptr, 65536 + (b * 7 + i) % 9973); });
  for (auto& th : t) th.join();
  int most = 0;
  for (int i = 0; i < 8; ++i)
    for (int b = 0; b < 2000; ++b) most = std::max(most, 65536 + (b * 7 + i) % 9973);
  CHECK(limits[0] == most);
  printf("ok\n");
}
