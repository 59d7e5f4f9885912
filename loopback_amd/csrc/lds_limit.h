// lds_limit.h -- launches whose workgroups hold more than 64 KiB of LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

namespace {

// The dynamic LDS that a kernel is allowed has to be raised where, with the `fixed` bytes that the kernel declares, it is past 64 KiB:
// once per kernel and device, to `bytes`, the most that any launch of it takes
template <typename K, K KERNEL> int allow_lds(int bytes, int fixed = 0) {
  static std::atomic<uint64_t> done{0};   // a bit per device
  int dev = 0;
  if (bytes + fixed <= 65536) return 0;
  int e = (int)hipGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e || (done.load(std::memory_order_relaxed) & bit)) return e;
  e = (int)hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (!e && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}
#define ALLOW_LDS(BYTES, ...) allow_lds<decltype(&__VA_ARGS__), &__VA_ARGS__>(BYTES)
#define ALLOW_LDS_BESIDE(FIXED, BYTES, ...) allow_lds<decltype(&__VA_ARGS__), &__VA_ARGS__>(BYTES, FIXED)

}  // namespace
