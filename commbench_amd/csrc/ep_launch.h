// Host-side pieces of the expert layer's launchers.
#pragma once

#include <hip/hip_runtime_api.h>

#include <atomic>

namespace mi_ep {

// A kernel's ceiling of dynamic LDS, raised once on every device that it is launched on.  One object for each kernel, of
// static storage; its flags only ever go from 0 to 1.
struct LdsCeiling {
  static constexpr int kDevices = 64;
  std::atomic<int> raised[kDevices];

  // For the device `stream` belongs to (the current one for null).  The runtime sets attributes on the current device: the
  // stream's is made current for the call, and the caller's put back.
  hipError_t raise(const void* kernel, int bytes, hipStream_t stream) {
    int device = 0, current = 0;
    hipError_t e = hipGetDevice(&current);
    if (e != hipSuccess) return e;
    device = current;
    if (stream != nullptr && (e = hipStreamGetDevice(stream, &device)) != hipSuccess) return e;
    if (device < 0 || device >= kDevices) return hipErrorInvalidDevice;
    if (raised[device].load(std::memory_order_acquire) != 0) return hipSuccess;
    if (device != current && (e = hipSetDevice(device)) != hipSuccess) return e;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (device != current) {
      const hipError_t back = hipSetDevice(current);
      if (e == hipSuccess) e = back;
    }
    if (e == hipSuccess) raised[device].store(1, std::memory_order_release);
    return e;
  }
};

}  // namespace mi_ep
