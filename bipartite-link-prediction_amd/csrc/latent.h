// Shared by the latent-factor operators (latent.hip, lookup.hip, scores8.hip).
#pragma once

#include "blp_internal.h"
#include "tile.h"

namespace blp {

// `device` current while it lives, then the one before.
struct DeviceGuard {
  int before = -1, rc = 0;
  const int device;
  explicit DeviceGuard(int d) : device(d) {
    hipError_t e = hipGetDevice(&before);
    if (e == hipSuccess && before != device) e = hipSetDevice(device);
    if (e != hipSuccess) rc = hip_fail(e, "hipSetDevice", __FILE__, __LINE__);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  ~DeviceGuard() {
    if (before >= 0 && before != device) (void)hipSetDevice(before);
  }
};

// Row ids in int32 or int64: the id of entry i, or -1 where it lies outside [0, rows).
struct Ids {
  const void* at;
  int wide;
  int64_t rows;
  __device__ int64_t operator()(int64_t i) const {
    const int64_t t = wide ? reinterpret_cast<const int64_t*>(at)[i] : reinterpret_cast<const int32_t*>(at)[i];
    return t >= 0 && t < rows ? t : -1;
  }
};

// n / d for n < 2^31 by a multiplication (d >= 1): with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// the quotient is (n + floor(m n / 2^32)) >> s. A vector unit has no integer division.
struct FastDiv {
  uint32_t d, m, s;
  __host__ explicit FastDiv(uint32_t by) : d(by), s(0) {
    while ((1ull << s) < by) ++s;
    m = (uint32_t)((((1ull << s) - by) << 32) / by + 1);
  }
  __device__ uint32_t operator()(uint32_t n) const { return (n + __umulhi(m, n)) >> s; }
};

}  // namespace blp
