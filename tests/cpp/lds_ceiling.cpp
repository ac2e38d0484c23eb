// LdsCeiling against stand-ins for the runtime's calls: which device was current when the attribute was set.
#include "ep_launch.h"

#include <cstdio>
#include <cstdlib>
#include <vector>

static int current = 0;
static hipError_t answer = hipSuccess;
static std::vector<int> raised_on;

extern "C" {
hipError_t hipGetDevice(int* device) { return *device = current, hipSuccess; }
hipError_t hipSetDevice(int device) { return current = device, hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t stream, hipDevice_t* device) {
  return *device = static_cast<int>(reinterpret_cast<long>(stream)), hipSuccess;  // the handle says the device
}
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) {
  if (answer == hipSuccess) raised_on.push_back(current);
  return answer;
}
}

static void check(bool ok, const char* what) {
  if (ok) return;
  std::printf("failed: %s\n", what);
  std::exit(1);
}

int main() {
  static mi_ep::LdsCeiling ceiling;
  const auto stream_of = [](long device) { return reinterpret_cast<hipStream_t>(device); };
  int kernel = 0;
  answer = hipErrorInvalidValue;
  check(ceiling.raise(&kernel, 1, stream_of(3)) == hipErrorInvalidValue && current == 0, "an error, and the device put back");
  answer = hipSuccess;
  check(ceiling.raise(&kernel, 1, stream_of(3)) == hipSuccess && current == 0, "another device's stream");
  check(raised_on == std::vector<int>{3}, "raised on the stream's device, after an error too");
  check(ceiling.raise(&kernel, 1, stream_of(3)) == hipSuccess && raised_on.size() == 1, "once");
  check(ceiling.raise(&kernel, 1, nullptr) == hipSuccess && raised_on == (std::vector<int>{3, 0}), "the null stream");
  current = 5;
  check(ceiling.raise(&kernel, 1, nullptr) == hipSuccess && raised_on == (std::vector<int>{3, 0, 5}), "the null stream elsewhere");
  check(ceiling.raise(&kernel, 1, stream_of(64)) == hipErrorInvalidDevice && current == 5, "a device out of range");
  std::printf("ok\n");
}
