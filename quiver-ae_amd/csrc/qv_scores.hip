// qv_scores.hip -- rows to 8 bits with a scale each, and the integer product of two
// such matrices.
#include <algorithm>

#include "qv_dense.hpp"
#include "qv_device.hpp"

using namespace qv;
using namespace qv::dev;
using namespace qv::dense;

namespace {

constexpr float kTiny = 0x1p-119f;  // below it 127 / a comes near the largest float: the row counts as zeros

__device__ __forceinline__ float wave_max(float v) {
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

// One wave per row, the row read twice.
template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t n, int64_t dim, int64_t stride,
                                                       int8_t* __restrict__ codes, int64_t code_stride,
                                                       float* __restrict__ scales) {
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  const int lane = lane_id();
  if (row >= n) return;
  const T* src = x + row * stride;
  float top = 0.f;
  bool odd = false;  // an infinity or a NaN in the row
  for (int64_t j = lane; j < dim; j += kWave) {
    const float v = fabsf((float)src[j]);
    odd |= !(v < __builtin_inff());
    top = fmaxf(top, v);
  }
  top = wave_max(top);
  odd = __any(odd);
  const bool some = !odd && top >= kTiny;
  const float inv = some ? 127.f / top : 0.f;
  for (int64_t j = lane; j < dim; j += kWave)
    codes[row * code_stride + j] = some ? (int8_t)rintf((float)src[j] * inv) : (int8_t)0;
  if (lane == 0) scales[row] = odd ? __builtin_nanf("") : some ? top / 127.f : 0.f;
}

// A 16 x 16 tile of the output per workgroup, one thread per element, both
// operands' rows staged 64 bytes at a time.
template <class O>
__global__ __launch_bounds__(256) void product_kernel(const int8_t* __restrict__ a, int64_t a_stride,
                                                      const float* __restrict__ a_scales, int64_t m,
                                                      const int8_t* __restrict__ b, int64_t b_stride,
                                                      const float* __restrict__ b_scales,
                                                      const float* __restrict__ bias, int64_t n, int64_t k,
                                                      O* __restrict__ out, int64_t out_stride, int64_t tiles_n) {
  __shared__ int8_t sa[16][68], sb[16][68];
  const int tid = threadIdx.x, r = tid / 16, c = tid % 16;
  const int64_t i0 = (int64_t)blockIdx.x / tiles_n * 16, j0 = (int64_t)blockIdx.x % tiles_n * 16;
  int32_t acc = 0;
  for (int64_t k0 = 0; k0 < k; k0 += 64) {
    for (int u = tid; u < 16 * 64; u += 256) {
      const int64_t row = u / 64, at = k0 + u % 64;
      sa[row][u % 64] = i0 + row < m && at < k ? a[(i0 + row) * a_stride + at] : (int8_t)0;
      sb[row][u % 64] = j0 + row < n && at < k ? b[(j0 + row) * b_stride + at] : (int8_t)0;
    }
    __syncthreads();
    for (int u = 0; u < 64; u++) acc += (int32_t)sa[r][u] * (int32_t)sb[c][u];
    __syncthreads();
  }
  if (i0 + r < m && j0 + c < n) {
    float v = ((float)acc * a_scales[i0 + r]) * b_scales[j0 + c];
    if (bias) v = v + bias[j0 + c];
    out[(i0 + r) * out_stride + j0 + c] = (O)v;
  }
}

template <class T>
void quantize(const void* x, int64_t n, int64_t dim, int64_t stride, int8_t* codes, int64_t code_stride, float* scales,
              hipStream_t st) {
  hipLaunchKernelGGL(quantize_kernel<T>, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, static_cast<const T*>(x), n,
                     dim, stride, codes, code_stride, scales);
  HIP_OK(hipGetLastError());
}

template <class O>
void product(const int8_t* a, int64_t a_stride, const float* a_scales, int64_t m, const int8_t* b, int64_t b_stride,
             const float* b_scales, const float* bias, int64_t n, int64_t k, void* out, int64_t out_stride,
             hipStream_t st) {
  const int64_t tm = (m + 15) / 16, tn = (n + 15) / 16;
  hipLaunchKernelGGL(product_kernel<O>, dim3((unsigned)(tm * tn)), dim3(256), 0, st, a, a_stride, a_scales, m, b,
                     b_stride, b_scales, bias, n, k, static_cast<O*>(out), out_stride, tn);
  HIP_OK(hipGetLastError());
}

}  // namespace

extern "C" {

int qv_quantize_rows(const void* d_x, int32_t type, int64_t n, int64_t dim, int64_t x_stride, int8_t* d_codes,
                     int64_t code_stride, float* d_scales, int device, void* stream) {
  return qv::guard([&] {
    check_matrix("x", d_x, n, dim, x_stride, value_size(type));
    check_matrix("codes", d_codes, n, dim, code_stride, 1);
    check_vector("scales", d_scales, n);
    if (n > INT32_MAX) qv::fail(QV_EUNSUPPORTED, "more than 2^31 - 1 rows");
    if (n == 0) return;
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (type == QV_FLOAT) quantize<float>(d_x, n, dim, x_stride, d_codes, code_stride, d_scales, st);
    else if (type == QV_BFLOAT16) quantize<bf16>(d_x, n, dim, x_stride, d_codes, code_stride, d_scales, st);
    else quantize<f16>(d_x, n, dim, x_stride, d_codes, code_stride, d_scales, st);
  });
}

int qv_int8_product(const int8_t* d_a, int64_t a_stride, const float* d_a_scales, int64_t m, const int8_t* d_b,
                    int64_t b_stride, const float* d_b_scales, const float* d_bias, int64_t n, int64_t k, void* d_out,
                    int32_t out_type, int64_t out_stride, int device, void* stream) {
  return qv::guard([&] {
    if (m < 0 || n < 0 || k < 0) qv::fail(QV_EINVAL, "negative size");
    if (k > QV_PRODUCT_MAX_K) qv::fail(QV_EUNSUPPORTED, "rows longer than 131071: their sums may overflow 32 bits");
    const int size = value_size(out_type);
    if (m == 0 || n == 0) return;
    check_matrix("a", d_a, m, k, a_stride, 1);
    check_matrix("b", d_b, n, k, b_stride, 1);
    check_matrix("out", d_out, m, n, out_stride, size);
    check_vector("a_scales", d_a_scales, m);
    check_vector("b_scales", d_b_scales, n);
    if (d_bias) check_vector("bias", d_bias, n);
    if (m > INT32_MAX || n > INT32_MAX || (m + 15) / 16 * ((n + 15) / 16) > INT32_MAX)
      qv::fail(QV_EUNSUPPORTED, "more tiles than one launch has");
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto go = [&](auto* o) {
      product<std::remove_pointer_t<decltype(o)>>(d_a, a_stride, d_a_scales, m, d_b, b_stride, d_b_scales, d_bias, n, k,
                                                  d_out, out_stride, st);
    };
    if (out_type == QV_FLOAT) go(static_cast<float*>(nullptr));
    else if (out_type == QV_BFLOAT16) go(static_cast<bf16*>(nullptr));
    else go(static_cast<f16*>(nullptr));
  });
}

}  // extern "C"
