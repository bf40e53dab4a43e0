// What the library's host files share: device lookup and per-device state, the sticky
// device-error check, the tensor-map encoder and the bounded waits' limit. Defined in
// attn_fwd.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdint>

namespace apex {
namespace host {

constexpr int kMaxDevices = 64;

// What a launch needs to know of its device.
struct Device {
  int* status = nullptr;         // device status word (bitmask of kStatus*)
  int* host_flag_dev = nullptr;  // mapped pinned word that a failing kernel sets to 1
  int num_sms = 0;
};

// The device that owns `ptr`; -1 when it is not device memory.
int device_of(const void* ptr);

// Sets up `dev` on its first use and reads the sticky error flag: APEX_ATTN_OK and *out, or
// the status to return. The caller has made `dev` current.
int acquire(int dev, Device* out);

// cuTensorMapEncodeTiled; not null after a successful acquire().
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

unsigned long long wait_timeout_ns();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Makes `dev` current for a scope.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) {
      (void)cudaGetLastError();
      prev = -1;
    }
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};

}  // namespace host
}  // namespace apex
