// What the C entry points of every translation unit share: the error that fisr_last_error(NULL) reports, the device a call's
// work belongs to, launch sizes.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

namespace fisr {
// Sets the calling thread's error text and returns `code` (fisr_api.hip).
int set_error(int code, const std::string& msg);
}  // namespace fisr

namespace {

// Every entry point that launches work selects the device the work belongs to and restores the caller's
// current device on return (a host may drive several GPUs, one ctx each, from one thread; torch's notion of
// the current device must not change behind its back).
struct DeviceGuard {
  int prev = -1;
  bool switched = false;
  hipError_t err = hipSuccess;
  explicit DeviceGuard(int dev) {
    if (dev < 0) return;
    err = hipGetDevice(&prev);
    if (err == hipSuccess && prev != dev) { err = hipSetDevice(dev); switched = err == hipSuccess; }
  }
  ~DeviceGuard() { if (switched) (void)hipSetDevice(prev); }
};
// Device that owns a device pointer (glue entry points have no ctx: the output tensor decides); -1 if unknown.
inline int device_of(const void* p) {
  hipPointerAttribute_t a;
  if (!p || hipPointerGetAttributes(&a, p) != hipSuccess) { (void)hipGetLastError(); return -1; }
  return a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged ? a.device : -1;
}
inline int grid_for(size_t work, int block = 256) {
  size_t g = (work + block - 1) / block;
  return (int)std::min<size_t>(std::max<size_t>(g, 1), 256 * 16);
}

}  // namespace
