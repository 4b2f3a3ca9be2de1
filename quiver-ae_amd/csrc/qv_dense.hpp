// qv_dense.hpp -- what the dense scoring calls share: element types, the caller's
// device, argument checks.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

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

inline void check_vector(const char* name, const void* p, int64_t count, int size = 4) {
  if (count > 0) check_matrix(name, p, 1, count, count, size);
}

}  // namespace dense
}  // namespace qv
