// pkv_device.h — what the host code of several kernels asks of the current device and of a
// call's tensors.
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

// Whether the `bytes` bytes from `out` on meet any of `rows` rows of `row` bytes, which lie
// `stride` (at least `row`) bytes apart from `at` on.
inline bool meets_rows(const void* out, int64_t bytes, const void* at, int64_t rows, int64_t stride, int64_t row) {
  const int64_t from = (int64_t)((uintptr_t)out - (uintptr_t)at);
  const int64_t i = from < row ? 0 : (from - row) / stride + 1;  // the first row that ends behind `out`
  return i < rows && i * stride < from + bytes;
}

}  // namespace pkv
