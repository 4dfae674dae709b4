#ifndef GP_DEVICE_HPP_
#define GP_DEVICE_HPP_

// gp_device.hpp — what the expert row routing (gp_route.hip) and the clipped
// updates (gp_clip.hip) share: the error macro, element types in 16-byte
// groups, wave and block sums.  Internal: not part of the C-ABI
// (include/gp_reduce.h); anonymous namespace, one copy per translation unit.

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <string>

#include "gp_reduce.h"

namespace gp_internal {
int set_error(int code, const char *msg);  // gp_reduce.hip
}

namespace {

inline int set_error(int code, const std::string &msg) { return gp_internal::set_error(code, msg.c_str()); }

#define GP_HIP_TRY(expr)                                                                    \
  do {                                                                                      \
    hipError_t e_ = (expr);                                                                 \
    if (e_ != hipSuccess) {                                                                 \
      (void)hipGetLastError(); /* a failed call's error must not fail a later launch */     \
      return set_error(GP_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(e_));      \
    }                                                                                       \
  } while (0)

#define GP_REQUIRE(cond, msg) \
  do {                        \
    if (!(cond)) return set_error(GP_ERR_INVALID, msg); \
  } while (0)

constexpr int kWave = 64;

// CU count per device, cached on first use (256, the MI355X count, where it
// cannot be asked: no device).
inline int device_cus() {
  constexpr int kMax = 64;
  static std::atomic<int> cus[kMax];
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMax) {
    (void)hipGetLastError();
    return 256;
  }
  int n = cus[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) {
    (void)hipGetLastError();
    n = 256;
  }
  cus[dev].store(n, std::memory_order_relaxed);
  return n;
}

inline size_t type_size(int type) { return type == GP_F32 ? 4 : 2; }
inline bool type_known(int type) { return type == GP_F32 || type == GP_BF16 || type == GP_F16; }

// [a, a + an) and [b, b + bn) share a byte.
inline bool bytes_overlap(const void *a, size_t an, const void *b, size_t bn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return an && bn && x < y + bn && y < x + an;
}

// ---------------------------------------------------------------------------
// 16 bytes of a row as floats.  The accesses ask for the element's alignment
// only: gfx950 takes a 16-byte global access at any address, so a row of odd
// width (or a buffer at an odd element) goes the same way as an aligned one.
// ---------------------------------------------------------------------------
template <typename E>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(E);
  typedef E Raw __attribute__((ext_vector_type(N)));
  typedef Raw Loose __attribute__((aligned(sizeof(E))));
  typedef float F __attribute__((ext_vector_type(N)));
};

template <typename E, bool NT = false>
__device__ __forceinline__ typename Vec<E>::Raw load_raw(const E *p) {
  const auto *q = reinterpret_cast<const typename Vec<E>::Loose *>(p);
  if constexpr (NT) return __builtin_nontemporal_load(q);
  return *q;
}

template <typename E, bool NT = false>
__device__ __forceinline__ void store_raw(E *p, typename Vec<E>::Raw v) {
  auto *q = reinterpret_cast<typename Vec<E>::Loose *>(p);
  if constexpr (NT)
    __builtin_nontemporal_store(v, q);
  else
    *q = v;
}

// The first n < Vec::N elements of a group (a row's ragged end); zeros after.
template <typename E>
__device__ __forceinline__ typename Vec<E>::Raw load_part(const E *p, int n) {
  typename Vec<E>::Raw v;
#pragma unroll
  for (int i = 0; i < Vec<E>::N; ++i) v[i] = i < n ? p[i] : (E)0.0f;
  return v;
}

template <typename E>
__device__ __forceinline__ void store_part(E *p, typename Vec<E>::Raw v, int n) {
#pragma unroll
  for (int i = 0; i < Vec<E>::N; ++i)
    if (i < n) p[i] = v[i];
}

template <typename E>
__device__ __forceinline__ typename Vec<E>::F to_float(typename Vec<E>::Raw v) {
  return __builtin_convertvector(v, typename Vec<E>::F);
}

// One rounding to the element's type, to nearest even.
template <typename E>
__device__ __forceinline__ typename Vec<E>::Raw from_float(typename Vec<E>::F v) {
  return __builtin_convertvector(v, typename Vec<E>::Raw);
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) v += __shfl_xor(v, d, kWave);
  return v;
}

}  // namespace

#endif  // GP_DEVICE_HPP_
