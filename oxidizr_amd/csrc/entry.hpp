// What the C entries without a plan share: the call's device, and checks of their arguments.
#pragma once
#include <initializer_list>

#include "host.hpp"

namespace moe {

// Makes `device` current for one call and the caller's device current after it.
struct DeviceScope {
  int before = -1, device;
  bool changed = false;
  explicit DeviceScope(int d) : device(d) {}
  hipError_t enter() {
    hipError_t e = hipGetDevice(&before);
    if (e != hipSuccess || before == device) return e;
    e = hipSetDevice(device);
    changed = e == hipSuccess;
    return e;
  }
  ~DeviceScope() {
    if (changed) (void)hipSetDevice(before);
  }
};

inline moe_status check_pointers(std::initializer_list<const void*> needed,
                          std::initializer_list<const void*> optional = {}) {
  for (const void* p : needed) {
    if (!p) return fail(MOE_ERR_INVALID, "a required pointer is NULL");
    if (!aligned16(p)) return fail(MOE_ERR_INVALID, "device pointers must be 16-byte aligned");
  }
  for (const void* p : optional)
    if (p && !aligned16(p)) return fail(MOE_ERR_INVALID, "device pointers must be 16-byte aligned");
  return MOE_OK;
}

inline moe_status check_dtype(int dtype) {
  if (dtype != MOE_DTYPE_F32 && dtype != MOE_DTYPE_BF16)
    return fail(MOE_ERR_INVALID, "unknown dtype %d", dtype);
  return MOE_OK;
}

// Integer arrays (indices, orders, offsets) need their own alignment only: they may be
// slices of one allocation.
inline moe_status check_ints(std::initializer_list<const void*> needed, size_t bytes = 4) {
  for (const void* p : needed) {
    if (!p) return fail(MOE_ERR_INVALID, "a required pointer is NULL");
    if ((uintptr_t)p % bytes) return fail(MOE_ERR_INVALID, "an integer array is not aligned");
  }
  return MOE_OK;
}

// Whether a launch of `blocks` workgroups of `threads` fits a grid.
constexpr int64_t kMaxGridThreads = int64_t(1) << 32;
inline moe_status check_grid(int64_t blocks, int threads) {
  if (blocks * threads >= kMaxGridThreads)
    return fail(MOE_ERR_UNSUPPORTED, "too many rows or tiles for one launch: split the batch");
  return MOE_OK;
}

}  // namespace moe
