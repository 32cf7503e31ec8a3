// Shared by the latent-factor operators (latent.hip, lookup.hip, scores8.hip).
#pragma once

#include "blp_internal.h"
#include "tile.h"

namespace blp {

inline int64_t div_up(int64_t v, int64_t by) { return (v + by - 1) / by; }
inline int64_t up(int64_t v, int64_t to) { return div_up(v, to) * to; }

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
  const void* from(int64_t i) const { return (const char*)at + i * (wide ? 8 : 4); }
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

namespace rows {

using namespace tile;

// ---- vectors of a row
// NE elements of 16 bytes, wherever they start (global memory takes any alignment); the row's last
// vector may be short.
template <int T>
struct Vec {
  static constexpr int NE = 16 / size_of(T);
  f32x4 v[NE / 4];
};
template <int T>
__device__ inline Vec<T> load_vec(const char* at, int left) {
  constexpr int NE = Vec<T>::NE;
  Vec<T> r;
  if (left >= NE) {
    const i32x4 raw = reinterpret_cast<const Unaligned16*>(at)->v;
    if constexpr (T == F32) {
      r.v[0] = __builtin_bit_cast(f32x4, raw);
    } else if constexpr (T == BF16) {
      const bf16x8 b = __builtin_bit_cast(bf16x8, raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) r.v[e >> 2][e & 3] = (float)b[e];
    } else {
      const f16x8 b = __builtin_bit_cast(f16x8, raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) r.v[e >> 2][e & 3] = (float)b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e) r.v[e >> 2][e & 3] = e < left ? load1<T>(at + e * size_of(T)) : 0.f;
  }
  return r;
}

template <int T>
__device__ inline void store_vec(char* at, int left, const Vec<T>& r) {
  constexpr int NE = Vec<T>::NE;
  if (left >= NE) {
    Unaligned16 raw;
    if constexpr (T == F32) {
      raw.v = __builtin_bit_cast(i32x4, r.v[0]);
    } else if constexpr (T == BF16) {
      bf16x8 b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = (__bf16)r.v[e >> 2][e & 3];
      raw.v = __builtin_bit_cast(i32x4, b);
    } else {
      f16x8 b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = (_Float16)r.v[e >> 2][e & 3];
      raw.v = __builtin_bit_cast(i32x4, b);
    }
    *reinterpret_cast<Unaligned16*>(at) = raw;
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e)
      if (e < left) store1<T>(at + e * size_of(T), r.v[e >> 2][e & 3]);
  }
}

}  // namespace rows

}  // namespace blp
