// Host-side helpers shared by the sources of the C ABI: the calling thread's error message, status codes
// from HIP errors, and the device's CU count.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "phantom_attn.h"

namespace pa {

inline thread_local char g_err[512] = "";

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

inline int hip_status(hipError_t e, const char* name) {
  if (e == hipSuccess) return PA_OK;
  return fail((int)e, "%s: HIP error: %s", name, hipGetErrorString(e));
}

// Compute units of the current device (looked up once per device), 0 if unknown.
inline int device_cus() {
  static std::atomic<int> cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  int n = cus[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    cus[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace pa
