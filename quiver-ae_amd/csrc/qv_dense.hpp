// qv_dense.hpp -- what the dense scoring calls share: element types and loads, the
// caller's device, argument checks.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "qv_common.hpp"
#include "qv_hip_util.hpp"

namespace qv {
namespace dense {

typedef __bf16 bf16;
typedef _Float16 f16;

// Makes `device` current for a call and the caller's own device again after it:
// these calls run inside other programs' threads.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    HIP_OK(hipGetDevice(&was_));
    if (was_ != device) {
      HIP_OK(hipSetDevice(device));
      moved_ = true;
    }
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(was_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int was_ = 0;
  bool moved_ = false;
};

inline int value_size(int32_t type) {
  if (type == QV_FLOAT) return 4;
  if (type == QV_BFLOAT16 || type == QV_FLOAT16) return 2;
  fail(QV_EINVAL, "type must be float, bfloat16 or float16");
}

// 16 bytes of a row at once, whatever the row's alignment (its elements' own).
typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
typedef raw4 raw4_any __attribute__((aligned(2), may_alias));

template <class T>
constexpr int kVec = 16 / (int)sizeof(T);

template <class T>
__device__ __forceinline__ raw4 load_raw(const T* p) {
  return *reinterpret_cast<const raw4_any*>(p);
}

template <class T>
__device__ __forceinline__ void unpack(raw4 r, float* v) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(r[i]);
    } else if constexpr (std::is_same<T, bf16>::value) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    } else {
      typedef f16 h2 __attribute__((ext_vector_type(2)));
      const h2 h = __builtin_bit_cast(h2, (uint32_t)r[i]);
      v[2 * i] = (float)h[0];
      v[2 * i + 1] = (float)h[1];
    }
  }
}

// The vector at p of which `valid` elements are in the row, `other` past them.
template <class T>
__device__ __forceinline__ void load_tail(const T* p, int64_t valid, float other, float* v) {
  if (valid >= kVec<T>) {
    unpack<T>(load_raw(p), v);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; i++) v[i] = i < valid ? (float)p[i] : other;
  }
}

// A launch holds less than 2^32 threads.  f(first, count) launches workgroups first, first + 1, ... of them.
template <class F>
void in_launches(int64_t workgroups, int threads, F f) {
  const int64_t most = (int64_t{1} << 31) / threads;
  for (int64_t first = 0; first < workgroups; first += most) f(first, (unsigned)std::min(most, workgroups - first));
}

// The wave's number in its workgroup, in a scalar register: what is derived from it
// (row pointers, tile corners) is then scalar arithmetic.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64)); }

// A matrix that the call reads or writes: there, aligned to its elements, rows that do not overlap.
inline void check_matrix(const char* name, const void* p, int64_t rows, int64_t cols, int64_t stride, int size) {
  if (rows < 0 || cols < 0) fail(QV_EINVAL, std::string(name) + ": negative size");
  if (rows == 0 || cols == 0) return;
  if (!p) fail(QV_EINVAL, std::string(name) + ": null pointer");
  if (reinterpret_cast<uintptr_t>(p) % size) fail(QV_EINVAL, std::string(name) + ": not aligned to its elements");
  if (stride < cols) fail(QV_EINVAL, std::string(name) + ": rows overlap");
  if (stride > INT64_MAX / 8 / rows) fail(QV_EINVAL, std::string(name) + ": too large");
}

// ... of 4-byte elements.
inline void check_vector(const char* name, const void* p, int64_t count) {
  if (count > 0) check_matrix(name, p, 1, count, count, 4);
}

}  // namespace dense
}  // namespace qv
