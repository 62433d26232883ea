// pkv_device.h — what the host code of several kernels asks of the current device.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <atomic>

namespace pkv {

// Compute units of the current device, asked for once per device (256 without one).
inline int compute_units() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Whether a launch of `blocks` in one dimension is possible: its threads must count in 32 bits.
inline bool fits_grid(int64_t blocks, int threads) { return blocks * threads <= (int64_t)UINT32_MAX; }

}  // namespace pkv
