// qv_log_probs.hip -- log probabilities of given columns, entropy and best
// alternatives of each row of logits, and their gradient.
#include <algorithm>

#include "qv_dense.hpp"
#include "qv_device.hpp"

using namespace qv;
using namespace qv::dev;
using namespace qv::dense;

namespace {

constexpr float kInf = __builtin_inff();

// Orders as the values do, larger first by larger key, equal values (the two
// zeros among them) the lower column first; never 0 for a value above -inf.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t column) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t order = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((uint64_t)order << 32) | (uint32_t)~column;
}

template <class F>
__device__ float block_fold(float v, float* tmp, F f) {
  __syncthreads();
  tmp[threadIdx.x] = v;
  __syncthreads();
  for (int s = 128; s; s >>= 1) {
    if ((int)threadIdx.x < s) tmp[threadIdx.x] = f(tmp[threadIdx.x], tmp[threadIdx.x + s]);
    __syncthreads();
  }
  return tmp[0];
}

// One workgroup per row; the row is read once for its largest value, once for the
// sums, and once for each alternative.
template <class T>
__global__ __launch_bounds__(256) void log_probs_kernel(const T* __restrict__ logits, int64_t rows, int cols,
                                                        int64_t stride, float inv_t, const int32_t* __restrict__ targets,
                                                        int per_row, int topk, float* __restrict__ target,
                                                        float* __restrict__ entropy, float* __restrict__ lse,
                                                        float* __restrict__ stats, int32_t* __restrict__ top_ids,
                                                        float* __restrict__ top) {
  __shared__ float tmp[256];
  __shared__ uint64_t keys[256];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  const int tid = threadIdx.x;
  float m = -kInf, odd = 0.f;
  for (int64_t j = tid; j < cols; j += 256) {
    const float v = (float)x[j];
    if (!(v < kInf)) odd = 1.f;
    m = fmaxf(m, v);
  }
  m = block_fold(m, tmp, [](float a, float b) { return fmaxf(a, b); });
  odd = block_fold(odd, tmp, [](float a, float b) { return fmaxf(a, b); });
  const float ref = m == -kInf ? 0.f : m;
  float s = 0.f, w = 0.f;
  for (int64_t j = tid; j < cols; j += 256) {
    const float y = fmaxf(((float)x[j] - ref) * inv_t, -200.f);
    const float e = expf(y);
    s += e;
    w += e * y;
  }
  s = block_fold(s, tmp, [](float a, float b) { return a + b; });
  w = block_fold(w, tmp, [](float a, float b) { return a + b; });
  const bool empty = m == -kInf && odd == 0.f;
  const float nan = __builtin_nanf("");
  const float ln_s = odd != 0.f ? nan : empty ? -kInf : logf(s);
  if (odd != 0.f) m = nan;
  auto lp = [&](float v) { return odd != 0.f ? nan : v == -kInf ? -kInf : (v - ref) * inv_t - ln_s; };
  if (tid == 0) {
    if (entropy) entropy[row] = odd != 0.f ? nan : empty ? 0.f : ln_s - w / s;
    if (lse) lse[row] = empty ? -kInf : m * inv_t + ln_s;
    stats[2 * row] = m;
    stats[2 * row + 1] = ln_s;
  }
  for (int t = tid; t < per_row; t += 256) {
    const int32_t j = targets[row * per_row + t];
    target[row * per_row + t] = j < 0 ? 0.f : j >= cols ? nan : lp((float)x[j]);
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < topk; k++) {
    uint64_t best = 0;
    for (int64_t j = tid; j < cols; j += 256) {
      const float v = (float)x[j];
      const uint64_t key = rank_key(v, (uint32_t)j);
      if (v > -kInf && key < last && key > best) best = key;
    }
    __syncthreads();
    keys[tid] = best;
    __syncthreads();
    for (int q = 128; q; q >>= 1) {
      if (tid < q) keys[tid] = umax64(keys[tid], keys[tid + q]);
      __syncthreads();
    }
    last = keys[0];
    if (tid == 0) {
      const bool none = last == 0 || odd != 0.f;
      top_ids[row * topk + k] = none ? -1 : (int32_t)~(uint32_t)last;
      top[row * topk + k] = odd != 0.f ? nan : none ? -kInf : lp((float)x[~(uint32_t)last]);
    }
  }
}

// One workgroup per row: every column by the formula's first two terms, then the
// columns that targets or alternatives name.
template <class T>
__global__ __launch_bounds__(256) void log_probs_grad_kernel(
    const T* logits, int64_t rows, int cols, int64_t stride, float inv_t, const float* __restrict__ stats,
    const float* __restrict__ entropy, const int32_t* __restrict__ targets, int per_row,
    const int32_t* __restrict__ top_ids, int topk, const float* __restrict__ g_target,
    const float* __restrict__ g_entropy, const float* __restrict__ g_lse, const float* __restrict__ g_top, T* grad,
    int64_t grad_stride) {
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  T* dx = grad + row * grad_stride;
  const int tid = threadIdx.x;
  const float m = stats[2 * row], ln_s = stats[2 * row + 1];
  const float ge = g_entropy ? g_entropy[row] : 0.f, h = g_entropy ? entropy[row] : 0.f;
  float g = g_lse ? -g_lse[row] : 0.f;
  const int named = (g_target ? per_row : 0) + (g_top ? topk : 0);
  auto name = [&](int i, float& w) {
    const int t = g_target ? per_row : 0;
    const int32_t j = i < t ? targets[row * per_row + i] : top_ids[row * topk + i - t];
    w = i < t ? g_target[row * per_row + i] : g_top[row * topk + i - t];
    return j;
  };
  for (int i = 0; i < named; i++) {
    float w;
    if (name(i, w) >= 0) g += w;
  }
  auto dense = [&](float v) {
    if (m == -kInf || m != m) return m == -kInf ? 0.f : m;
    const float lp = fmaxf((v - m) * inv_t - ln_s, -1000.f);
    const float p = expf(lp);
    return v == -kInf ? 0.f : -p * g - ge * (p * (lp + h));
  };
  // a named column's value: its weights added in their order
  auto value = [&](int i, float v) {
    float w, sum = dense(v);
    const int32_t j = name(i, w);
    for (int q = 0; q < named; q++)
      if (name(q, w) == j && m != -kInf) sum += w;
    return sum * inv_t;
  };
  float w, patch = 0.f;
  __shared__ float kept[256];
  const bool shared_rows = named <= 256;
  if (shared_rows && tid < named) {
    const int32_t j = name(tid, w);
    if (j >= 0 && j < cols) patch = (float)x[j];
  }
  kept[tid] = patch;
  __syncthreads();
  for (int64_t j = tid; j < cols; j += 256) dx[j] = (T)(dense((float)x[j]) * inv_t);
  __syncthreads();
  if (tid < named) {
    const int32_t j = name(tid, w);
    if (j >= 0 && j < cols) dx[j] = (T)value(tid, kept[tid]);
  }
}

void check_rows(int32_t type, int64_t rows, int64_t cols, int64_t stride, const void* x, float temperature,
                const int32_t* targets, int32_t per_row, int32_t topk) {
  check_matrix("logits", x, rows, cols, stride, value_size(type));
  if (!(temperature > 0.f) || !(1.f / temperature < kInf) || !(1.f / temperature > 0.f))
    qv::fail(QV_EINVAL, "temperature must be positive, and its reciprocal a finite float");
  if (cols > INT32_MAX || rows > INT32_MAX) qv::fail(QV_EUNSUPPORTED, "more than 2^31 - 1 rows or columns");
  if (per_row < 0) qv::fail(QV_EINVAL, "targets_per_row must not be negative");
  if (per_row > QV_LOG_PROBS_MAX_TARGETS) qv::fail(QV_EUNSUPPORTED, "more than 64 targets per row");
  if (topk < 0) qv::fail(QV_EINVAL, "topk must not be negative");
  if (topk > QV_LOG_PROBS_MAX_TOPK) qv::fail(QV_EUNSUPPORTED, "topk above 64");
  check_vector("targets", targets, rows * per_row);
}

}  // namespace

extern "C" {

int64_t qv_log_probs_workspace(int64_t rows, int64_t cols, int32_t topk) {
  int64_t bytes = 0;
  const int rc = qv::guard([&] {
    if (rows < 0 || cols < 0 || topk < 0) qv::fail(QV_EINVAL, "negative size");
    if (topk > QV_LOG_PROBS_MAX_TOPK) qv::fail(QV_EUNSUPPORTED, "topk above 64");
  });
  return rc == QV_OK ? bytes : rc;
}

int qv_log_probs(const void* d_logits, int32_t type, int64_t rows, int64_t cols, int64_t stride, float temperature,
                 const int32_t* d_targets, int32_t targets_per_row, int32_t topk, float* d_target, float* d_entropy,
                 float* d_lse, float* d_stats, int32_t* d_top_ids, float* d_top, void* d_workspace,
                 int64_t workspace_bytes, int device, void* stream) {
  return qv::guard([&] {
    check_rows(type, rows, cols, stride, d_logits, temperature, d_targets, targets_per_row, topk);
    check_vector("target", d_target, rows * targets_per_row);
    check_vector("stats", d_stats, 2 * rows);
    check_vector("top_ids", d_top_ids, rows * topk);
    check_vector("top", d_top, rows * topk);
    if (rows == 0) return;
    const OnDevice on(device);
    auto go = [&](auto* x) {
      hipLaunchKernelGGL(log_probs_kernel, dim3((unsigned)rows), dim3(256), 0, static_cast<hipStream_t>(stream), x, rows,
                         (int)cols, stride, 1.f / temperature, d_targets, targets_per_row, topk, d_target, d_entropy,
                         d_lse, d_stats, d_top_ids, d_top);
      HIP_OK(hipGetLastError());
    };
    if (type == QV_FLOAT) go(static_cast<const float*>(d_logits));
    else if (type == QV_BFLOAT16) go(static_cast<const bf16*>(d_logits));
    else go(static_cast<const f16*>(d_logits));
  });
}

int qv_log_probs_grad(const void* d_logits, int32_t type, int64_t rows, int64_t cols, int64_t stride, float temperature,
                      const float* d_stats, const float* d_entropy, const int32_t* d_targets, int32_t targets_per_row,
                      const int32_t* d_top_ids, int32_t topk, const float* d_g_target, const float* d_g_entropy,
                      const float* d_g_lse, const float* d_g_top, void* d_grad, int64_t grad_stride, int device,
                      void* stream) {
  return qv::guard([&] {
    check_rows(type, rows, cols, stride, d_logits, temperature, d_targets, targets_per_row, topk);
    check_matrix("grad", d_grad, rows, cols, grad_stride, value_size(type));
    check_vector("stats", d_stats, 2 * rows);
    if (d_g_entropy) check_vector("entropy", d_entropy, rows);
    if (d_g_top) check_vector("top_ids", d_top_ids, rows * topk);
    if (rows == 0 || cols == 0) return;
    const OnDevice on(device);
    auto go = [&](auto* x) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
      hipLaunchKernelGGL(log_probs_grad_kernel, dim3((unsigned)rows), dim3(256), 0, static_cast<hipStream_t>(stream), x,
                         rows, (int)cols, stride, 1.f / temperature, d_stats, d_entropy, d_targets, targets_per_row,
                         d_top_ids, topk, d_g_target, d_g_entropy, d_g_lse, d_g_top, static_cast<T*>(d_grad),
                         grad_stride);
      HIP_OK(hipGetLastError());
    };
    if (type == QV_FLOAT) go(static_cast<const float*>(d_logits));
    else if (type == QV_BFLOAT16) go(static_cast<const bf16*>(d_logits));
    else go(static_cast<const f16*>(d_logits));
  });
}

}  // extern "C"
