// qv_layer_norm.hip -- layer norm over the rows of a matrix, and its gradient with those
// of the weight and the bias.
//
// y = x^ w + b,  x^ = (x - mean) / sqrt(var + eps), mean and var over the row.  With h = g w
// the gradient is dx = (h - mean(h) - x^ mean(h x^)) / sqrt(var + eps), dw = sum g x^ and
// db = sum g over the rows.
//
// A row is read once and stays in the registers of R threads, E vectors of four values each,
// between its sums and what is made of them; weights stay there from row to row.  The
// deviations d = x - mean are summed too: what the mean's rounding left of them comes off
// again, in d and in var = sum d^2 / n - (sum d / n)^2.  The gradient takes mean(h) and
// mean(h x^) from the same exchange as var.  A row whose moments are not finite is taken
// again times 2^-90 (its values may be up to the largest float), so only rows that hold an
// infinity or a NaN give NaN; one whose sum of h d is none, times about 1 / s.  All sums
// are fp32, in a fixed order.
#include <algorithm>
#include <cfloat>

#include "qv_dense.hpp"
#include "qv_device.hpp"

using namespace qv;
using namespace qv::dev;
using namespace qv::dense;

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

// Four values of a row, whatever the row's alignment.
template <class T>
__device__ __forceinline__ f4 load_four(const T* p, int64_t valid) {
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (valid >= 4) {
    if constexpr (sizeof(T) == 4) {
      const raw4 r = load_raw(p);
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = __uint_as_float(r[i]);
    } else {
      T t[4];
      __builtin_memcpy(t, p, 8);
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = (float)t[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (i < valid) v[i] = (float)p[i];
  }
  return v;
}

// ... and back, past the L2 if there is more than it holds (kStreamBytes).
template <class T>
__device__ __forceinline__ void store_four(T* p, int64_t valid, f4 v, bool stream) {
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; i++) t[i] = (T)v[i];
  if (valid >= 4) {
    typedef uint32_t raw __attribute__((ext_vector_type(sizeof(T))));
    typedef raw raw_any __attribute__((aligned(sizeof(T)), may_alias));
    store_past(__builtin_bit_cast(raw, t), reinterpret_cast<raw_any*>(p), stream);
  } else {
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (i < valid) p[i] = t[i];
  }
}

// Weights or biases of any of the types; `none` without.
__device__ __forceinline__ f4 load_params(const void* p, int type, int64_t j, int64_t dim, float none) {
  if (!p) return f4{none, none, none, none};
  if (type == QV_FLOAT) return load_four(static_cast<const float*>(p) + j, dim - j);
  if (type == QV_BFLOAT16) return load_four(static_cast<const bf16*>(p) + j, dim - j);
  return load_four(static_cast<const f16*>(p) + j, dim - j);
}

__device__ __forceinline__ void store_param(void* p, int type, int64_t j, float v) {
  if (type == QV_FLOAT) static_cast<float*>(p)[j] = v;
  else if (type == QV_BFLOAT16) static_cast<bf16*>(p)[j] = (bf16)v;
  else static_cast<f16*>(p)[j] = (f16)v;
}

template <int CONTROL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CONTROL, 0xF, 0xF, true));
}

// The sum over the R lanes (a power of two, up to a wave) that the lane is one of, the same bits in each.
template <int R>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (R >= 2) v = add_dpp<0xB1>(v);
  if constexpr (R >= 4) v = add_dpp<0x4E>(v);
  if constexpr (R >= 8) v = add_dpp<0x141>(v);   // row_half_mirror
  if constexpr (R >= 16) v = add_dpp<0x128>(v);  // row_ror:8
  if constexpr (R >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (R >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}

// A thread's part of a row, E vectors of four values, every R-th of the row's: asked for a row ahead, unpacked when they
// are used.  All loads are whole: the one that the row ends in begins four values before the end, and values() moves
// what it has down and fills up with zeros.
template <class T, int R, int E>
struct Part {
  uint32_t raw[E][sizeof(T)];
  __device__ __forceinline__ void load_one(int e, const T* row, int lane, int dim, bool four) {
    const int j = (e * R + lane) * 4;
    if (four) {
      __builtin_memcpy(raw[e], row + min(j, dim - 4), 4 * sizeof(T));
    } else {
      T t[4] = {};
#pragma unroll
      for (int i = 0; i < 3; i++)
        if (j + i < dim) t[i] = row[i];
      __builtin_memcpy(raw[e], t, sizeof(t));
    }
  }
  // TOGETHER: all behind one branch; with one for each, some wait for those before.  That is better only in the forward pass of
  // floats within a wave (us: 60,001 x 1,001 88, together 94, 1M x 128 172, 180; but 5,000 x 16,384 118, each 130, and the
  // gradient of 16,384 x 768 35, each 41, 200,000 x 128 62, 75, 5,000 x 6,000 90, 107, 500,000 x 64 76, 88).
  template <bool TOGETHER>
  __device__ __forceinline__ void load(const T* row, int lane, int dim) {
    if (TOGETHER && dim >= 4) {
#pragma unroll
      for (int e = 0; e < E; e++) load_one(e, row, lane, dim, true);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) load_one(e, row, lane, dim, !TOGETHER && dim >= 4);
    }
  }
  __device__ __forceinline__ f4 values(int e, int lane, int dim) const {
    T t[4];
    __builtin_memcpy(t, raw[e], sizeof(t));
    f4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (float)t[i];
    if ((e + 1) * R * 4 > dim) {
      const int over = dim >= 4 ? (e * R + lane) * 4 - (dim - 4) : (e * R + lane) * 4;
      if (over > 0) {
        if (over & 1) v = f4{v[1], v[2], v[3], 0.f};
        if (over & 2) v = f4{v[2], v[3], 0.f, 0.f};
        if (over >= 4) v = f4{0.f, 0.f, 0.f, 0.f};
      }
    }
    return v;
  }
};

// Rows whose sum of squares passes kLargest are taken times kSmaller: 2^24 squares of the largest float are then below it, and
// those of rows that passed it far above the smallest float.
constexpr float kSmaller = 0x1p-90f, kLargest = FLT_MAX / 2.f;

// Of the sums of d, d^2 and, of four, h and h d: whether what is made of them stays finite.  What the mean's rounding left is
// at most the root of kLargest, so 2^57 for the sum of h keeps their product finite too.
template <int N>
__device__ __forceinline__ bool within(const float (&v)[N], float most) {
  if constexpr (N == 4) return __builtin_fmaf(__builtin_fabsf(v[2]), 0x1p70f, v[1] + __builtin_fabsf(v[3])) <= most;
  else return v[1] <= most;
}

// Sums over the R threads of a row: a part of a wave, or whole waves, which exchange theirs through two areas of LDS in
// turn (so one barrier each: nobody writes an area again before everyone has met at the other one's).
template <int R, int T>
struct Row {
  static constexpr int kWaves = R / kWave;  // of a row, where it has whole ones
  static constexpr int kFloats = R > kWave ? 2 * 4 * (T / kWave) : 1;
  float* lds;  // 16-byte aligned
  int turn = 0;
  bool any_wide = false;
  // CHECK: `any_wide` is set where a row of the wave is not within() kLargest; or, where rows have more than a wave's threads,
  // a wave's part of any row of the workgroup not within a 16th of it: all that meet at a barrier agree on it, and no row whose
  // sums (of 16 parts at most) are not within kLargest is left out.
  template <bool CHECK, int N>
  __device__ __forceinline__ void sum(float (&v)[N]) {
    static_assert(N <= 4, "an area has four sums of each wave");
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = lanes_sum<R < kWave ? R : kWave>(v[i]);
    if constexpr (R > kWave) {
      float* area = lds + turn * 4 * (T / kWave);
      turn ^= 1;
      const int wave = wave_id();
      if (lane_id() == 0)
#pragma unroll
        for (int i = 0; i < N; i++) area[4 * wave + i] = v[i];
      __syncthreads();
      const float* from = area + wave / kWaves * kWaves * 4;
      if constexpr (CHECK) {
        float part[N];
        __builtin_memcpy(part, __builtin_assume_aligned(area + 4 * (lane_id() % (T / kWave)), 16), sizeof(part));
        any_wide = __any(lane_id() < T / kWave && !within(part, kLargest / 16.f));
      }
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = from[i];
#pragma unroll
      for (int w = 1; w < kWaves; w++)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += from[4 * w + i];
    } else if constexpr (CHECK) {
      any_wide = __any(!within(v, kLargest));
    }
  }
};

// The variance, of the mean square of deviations from what is the mean but for `rest`.  Where all values are equal, only
// roundings are left of it, and of the deviations less `rest` as many units of 2^-24 of it as sums have additions in a row:
// no less than 2^-12 of it keeps their quotients small.  One value of up to 2^20 that differs from the others has more.
__device__ __forceinline__ float variance(float square, float rest) {
  return max(__builtin_fmaf(-rest, rest, square), rest * rest * 0x1p-24f);
}

// The mean of h x^ is that of h d times 1 / s.  Where sums of h d are not finite, and with an eps for which products of h with
// a small d may be lost (they are below 2^-126 for an h of 2^-106 and a d of the root of kSmallEps), values are taken times the
// power of two below 1 / s, d is then about x^.  (Of values that are not all equal none is more than 2^40 s.)
constexpr float kSmallEps = 0x1p-40f;
__device__ __forceinline__ float power_below(float v) { return __uint_as_float(__float_as_uint(v) & 0x7f800000u); }

// What a row's values are to be taken times in the gradient's next turn, after turns 0 and 1.
__device__ __forceinline__ float next_scale(int turn, float scale, bool bad, bool wide, float var, float rstd, float eps) {
  if (turn == 0 && bad) return kSmaller;
  if (var == 0.f) return scale;
  if (turn == 0 && (wide || eps < kSmallEps)) return power_below(rstd);
  if (turn == 1 && scale == kSmaller) return kSmaller * power_below(rstd);
  return scale;
}

// Turns a thread's part of a row (0 past its end), values(e), into deviations v, of the values times `scale`; returns
// 1 / sqrt(var + eps) of those.  With GRAD, means[0] and means[1] come out as the means of h = g w and of h x^.
//
// Rows out of the ordinary take further turns, from their values on (next_scale).  All that meet take them, and the other rows'
// results come out as before.
template <bool GRAD, int R, int T, int E, class F>
__device__ __forceinline__ float centre(F values, f4 (&v)[E], const f4 (&g)[E], const f4 (&w)[E], int lane, int dim,
                                        float eps, Row<R, T>& row, float& scale, float (&means)[2]) {
  const float per = 1.f / (float)dim;
  scale = 1.f;
  for (int turn = 0;; turn++) {
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < E; e++) s[0] += (v[e][0] + v[e][1]) + (v[e][2] + v[e][3]);
    row.template sum<false>(s);
    const float mean = s[0] * per;
    float m[GRAD ? 4 : 2] = {};
#pragma unroll
    for (int e = 0; e < E; e++) {
      v[e] = v[e] - mean;
      if ((e + 1) * R * 4 > dim) {  // not the whole vector of every thread is in the row
#pragma unroll
        for (int i = 0; i < 4; i++) v[e][i] = (e * R + lane) * 4 + i < dim ? v[e][i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        m[0] += v[e][i];
        m[1] = __builtin_fmaf(v[e][i], v[e][i], m[1]);
        if constexpr (GRAD) {
          const float h = g[e][i] * w[e][i];
          m[2] += h;
          m[3] = __builtin_fmaf(h, v[e][i], m[3]);
        }
      }
    }
    row.template sum<true>(m);
    const float rest = m[0] * per, var = variance(m[1] * per, rest);
    const bool bad = !(m[1] <= kLargest);
    const float of_eps = eps * scale * scale;
    auto root = [&] { return 1.f / __builtin_sqrtf(bad ? __builtin_nanf("") : var == 0.f ? eps : var + of_eps); };
    float rstd;
    if constexpr (GRAD) rstd = root();
    if (GRAD ? turn == 2 || turn == 0 && !row.any_wide && !(eps < kSmallEps) : turn == 1 || !row.any_wide) {
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = v[e] - rest;
      scale = var == 0.f ? 1.f : scale;  // all deviations are 0, times any scale
      if constexpr (!GRAD) rstd = root();
      if constexpr (GRAD) {
        means[0] = m[2] * per;
        means[1] = (m[3] - rest * m[2]) * per * rstd;
      }
      return rstd;
    }
    if constexpr (GRAD) scale = next_scale(turn, scale, bad, !within(m, kLargest), var, rstd, eps);
    else scale = bad ? kSmaller : 1.f;
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = values(e) * scale;
  }
}

template <class T, int R, int E, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_kernel(const T* x, int64_t n, int dim, int64_t stride, const void* weight,
                                                       const void* bias, int param_type, float eps, T* y, int64_t y_stride,
                                                       bool stream) {
  constexpr int kGroups = THREADS / R;
  __shared__ __align__(16) float lds[Row<R, THREADS>::kFloats];
  Row<R, THREADS> across{lds};
  const int lane = threadIdx.x % R;
  f4 w[E], b[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = (e * R + lane) * 4;
    w[e] = load_params(weight, param_type, j, dim, 1.f);
    b[e] = load_params(bias, param_type, j, dim, 0.f);
  }
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / R;
  constexpr bool kTogether = R > kWave;
  Part<T, R, E> part;
  part.template load<kTogether>(x + min(row, n - 1) * stride, lane, dim);
  for (int64_t base = (int64_t)blockIdx.x * kGroups; base < n; base += step, row += step) {
    f4 v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = part.values(e, lane, dim);
    if (base + step < n) part.template load<kTogether>(x + min(row + step, n - 1) * stride, lane, dim);
    auto again = [&](int e) {
      Part<T, R, E> same;
      same.template load<kTogether>(x + min(row, n - 1) * stride, lane, dim);
      return same.values(e, lane, dim);
    };
    float scale, none[2];
    const float rstd = centre<false>(again, v, v, v, lane, dim, eps, across, scale, none);
    if (row >= n) continue;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int j = (e * R + lane) * 4;
      f4 o;
#pragma unroll
      for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(v[e][i] * rstd, w[e][i], b[e][i]);
      store_four(y + row * y_stride + j, dim - j, o, stream);
    }
  }
}

// Adds up the rows that its groups have seen of a column's sums: `part` of this workgroup, its sums of g x^, then those of g.
template <class T, int R, int E, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_grad_kernel(const T* x, int64_t n, int dim, int64_t stride, const T* grad,
                                                            int64_t grad_stride, const void* weight, int param_type,
                                                            float eps, T* dx, int64_t dx_stride, float* parts, int pitch,
                                                            bool stream) {
  constexpr int kGroups = THREADS / R;
  constexpr int kWide = R * E * 4;
  __shared__ __align__(16) float lds[Row<R, THREADS>::kFloats];
  __shared__ __align__(16) float columns[kGroups > 1 ? kGroups * kWide : 1];
  Row<R, THREADS> across{lds};
  const int lane = threadIdx.x % R, group = threadIdx.x / R;
  f4 w[E], dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    w[e] = load_params(weight, param_type, (e * R + lane) * 4, dim, 1.f);
    dw[e] = db[e] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  // A row of 16 bits ahead, as in norm_kernel, where few waves run anyway (5,000 x 12,288: 131 -> 111 us, 16,641 x 768: 27 -> 26);
  // else it takes registers for which fewer would (65,536 x 1,024 of 16 bits: 91 -> 108).  (Floats where few run would gain too
  // since their loads are together: 16,384 x 768 35 -> 33, 4,096 x 4,096 53 -> 48; not done.)
  constexpr bool kAhead = THREADS == 512 && sizeof(T) == 2;
  Part<T, R, E> part, part_g;
  auto load = [&](int64_t row) {
    part.template load<true>(x + min(row, n - 1) * stride, lane, dim);
    part_g.template load<true>(grad + min(row, n - 1) * grad_stride, lane, dim);
  };
  if (kAhead) load(row);
  for (int64_t base = (int64_t)blockIdx.x * kGroups; base < n; base += step, row += step) {
    if (!kAhead) load(row);
    f4 v[E], g[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      v[e] = part.values(e, lane, dim);
      g[e] = part_g.values(e, lane, dim);
    }
    if (kAhead && base + step < n) load(row + step);
    auto again = [&](int e) {
      Part<T, R, E> same;
      same.template load<true>(x + min(row, n - 1) * stride, lane, dim);
      return same.values(e, lane, dim);
    };
    float scale, means[2];
    const float rstd = centre<true>(again, v, g, w, lane, dim, eps, across, scale, means);
    if (row >= n) continue;
    // x^ = d rstd; dx = scale rstd (h - c1 - x^ c2)
    const float c1 = means[0], c2 = means[1];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int j = (e * R + lane) * 4;
      f4 o;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float hat = v[e][i] * rstd;
        o[i] = __builtin_fmaf(-hat, c2, g[e][i] * w[e][i] - c1) * (rstd * scale);
        dw[e][i] = __builtin_fmaf(g[e][i], hat, dw[e][i]);
        db[e][i] += g[e][i];
      }
      if (dx) store_four(dx + row * dx_stride + j, dim - j, o, stream);
    }
  }
  if (!parts) return;
  float* sums = parts + (int64_t)blockIdx.x * 2 * pitch;
#pragma unroll
  for (int of = 0; of < 2; of++) {
    if constexpr (kGroups == 1) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int j = (e * R + lane) * 4;
        if (j < dim) *reinterpret_cast<f4*>(sums + of * pitch + j) = of ? db[e] : dw[e];
      }
    } else {
      if (of) __syncthreads();
#pragma unroll
      for (int e = 0; e < E; e++) *reinterpret_cast<f4*>(columns + group * kWide + (e * R + lane) * 4) = of ? db[e] : dw[e];
      __syncthreads();
      for (int j = threadIdx.x; j < dim; j += THREADS) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < kGroups; q++) s += columns[q * kWide + j];
        sums[of * pitch + j] = s;
      }
    }
  }
}

// The columns' sums over `count` parts: 32 columns per workgroup, 32 threads each.
__global__ __launch_bounds__(1024) void join_columns_kernel(const float* parts, int64_t count, int dim, int pitch, void* dweight,
                                                            void* dbias, int param_type) {
  __shared__ float sums[32][33];
  const int column = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int j = blockIdx.x * 32 + column;
  void* out = blockIdx.y ? dbias : dweight;
  if (!out) return;
  float s = 0.f;
  if (j < dim)
    for (int64_t q = slice; q < count; q += 32) s += parts[(q * 2 + blockIdx.y) * pitch + j];
  sums[slice][column] = s;
  __syncthreads();
  if (slice == 0 && j < dim) {
#pragma unroll
    for (int q = 1; q < 32; q++) s += sums[q][column];
    store_param(out, param_type, j, s);
  }
}

// ---- long rows (kLong, kLongGrad) ----------------------------------------------------
//
// A workgroup per row, which is read again for each step (from the caches while it fits).  The gradient
// goes column by column then, with what it needs of the rows in `Moments`.  2,000 x 20,000, us (at 4.9 TB/s, each matrix once):
// floats 90 (66), gradient 173 (98); 16 bits 53 (33), gradient 145 (49); 5,000 x 16,384 of 16 bits, gradient 291 (101); 8 x 1M
// floats, eight workgroups in all, 325 (13).

struct Moments {
  float mean, rest, rstd, scale, c1, c2, none[2];
};

template <bool GRAD, class T>
__device__ __forceinline__ Moments long_moments(const T* x, const T* g, const void* weight, int param_type, int64_t dim,
                                                float eps, Row<1024, 1024>& across) {
  const float per = 1.f / (float)dim;
  Moments r = {0.f, 0.f, 0.f, 1.f, 0.f, 0.f, {0.f, 0.f}};
  for (int turn = 0;; turn++) {
    float s[1] = {0.f};
    for (int64_t j = threadIdx.x * 4; j < dim; j += 4096) {
      const f4 v = load_four(x + j, dim - j) * r.scale;
      s[0] += (v[0] + v[1]) + (v[2] + v[3]);
    }
    across.template sum<false>(s);
    r.mean = s[0] * per;
    float m[GRAD ? 4 : 2] = {};
    for (int64_t j = threadIdx.x * 4; j < dim; j += 4096) {
      const f4 v = load_four(x + j, dim - j);
      f4 h = {};
      if constexpr (GRAD) h = load_four(g + j, dim - j) * load_params(weight, param_type, j, dim, 1.f);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float d = j + i < dim ? v[i] * r.scale - r.mean : 0.f;
        m[0] += d;
        m[1] = __builtin_fmaf(d, d, m[1]);
        if constexpr (GRAD) {
          m[2] += h[i];
          m[3] = __builtin_fmaf(h[i], d, m[3]);
        }
      }
    }
    across.template sum<true>(m);
    r.rest = m[0] * per;
    const bool bad = !(m[1] <= kLargest);
    const float var = variance(m[1] * per, r.rest);
    r.rstd = 1.f / __builtin_sqrtf(bad ? __builtin_nanf("") : var == 0.f ? eps : var + eps * r.scale * r.scale);
    if (turn == (GRAD ? 2 : 1) || turn == 0 && !across.any_wide && !(GRAD && eps < kSmallEps)) {
      if constexpr (GRAD) {
        r.c1 = m[2] * per;
        r.c2 = (m[3] - r.rest * m[2]) * per * r.rstd;
      }
      if (var == 0.f) {  // all deviations are 0, times any scale
        r.mean *= 1.f / r.scale;
        r.scale = 1.f;
      }
      return r;
    }
    if constexpr (GRAD) r.scale = next_scale(turn, r.scale, bad, !within(m, kLargest), var, r.rstd, eps);
    else if (turn == 0) r.scale = bad ? kSmaller : 1.f;
  }
}

template <class T>
__global__ __launch_bounds__(1024) void norm_long_kernel(const T* x, int64_t n, int64_t dim, int64_t stride, const void* weight,
                                                         const void* bias, int param_type, float eps, T* y, int64_t y_stride,
                                                       bool stream) {
  __shared__ __align__(16) float lds[Row<1024, 1024>::kFloats];
  Row<1024, 1024> across{lds};
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const T* from = x + row * stride;
    const Moments r = long_moments<false, T>(from, nullptr, nullptr, 0, dim, eps, across);
    for (int64_t j = threadIdx.x * 4; j < dim; j += 4096) {
      const f4 v = load_four(from + j, dim - j), w = load_params(weight, param_type, j, dim, 1.f),
               b = load_params(bias, param_type, j, dim, 0.f);
      f4 o;
#pragma unroll
      for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf((v[i] * r.scale - r.mean - r.rest) * r.rstd, w[i], b[i]);
      store_four(y + row * y_stride + j, dim - j, o, stream);
    }
  }
}

template <class T>
__global__ __launch_bounds__(1024) void long_moments_kernel(const T* x, int64_t n, int64_t dim, int64_t stride, const T* grad,
                                                            int64_t grad_stride, const void* weight, int param_type, float eps,
                                                            Moments* moments) {
  __shared__ __align__(16) float lds[Row<1024, 1024>::kFloats];
  Row<1024, 1024> across{lds};
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const Moments r = long_moments<true, T>(x + row * stride, grad + row * grad_stride, weight, param_type, dim, eps, across);
    if (threadIdx.x == 0) moments[row] = r;
  }
}

// 1,024 columns of every gridDim.y-th row: its gradient, and this part of the columns' sums.
template <class T>
__global__ __launch_bounds__(256) void long_grad_kernel(const T* x, int64_t n, int64_t dim, int64_t stride, const T* grad,
                                                        int64_t grad_stride, const void* weight, int param_type,
                                                        const Moments* moments, T* dx, int64_t dx_stride, float* parts, int pitch,
                                                        bool stream) {
  const int64_t j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (j >= dim) return;
  const f4 w = load_params(weight, param_type, j, dim, 1.f);
  f4 dw = {0.f, 0.f, 0.f, 0.f}, db = dw;
  for (int64_t row = blockIdx.y; row < n; row += gridDim.y) {
    const Moments r = moments[row];
    const f4 v = load_four(x + row * stride + j, dim - j), g = load_four(grad + row * grad_stride + j, dim - j);
    f4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float hat = (v[i] * r.scale - r.mean - r.rest) * r.rstd;
      o[i] = __builtin_fmaf(-hat, r.c2, g[i] * w[i] - r.c1) * (r.rstd * r.scale);
      dw[i] = __builtin_fmaf(g[i], hat, dw[i]);
      db[i] += g[i];
    }
    if (dx) store_four(dx + row * dx_stride + j, dim - j, o, stream);
  }
  if (!parts) return;
  float* part = parts + (int64_t)blockIdx.y * 2 * pitch;
  *reinterpret_cast<f4*>(part + j) = dw;
  *reinterpret_cast<f4*>(part + pitch + j) = db;
}

// ---- host side -----------------------------------------------------------------------

// Longer rows do not stay in a workgroup's registers; the gradient keeps five values for each of the forward pass's three.
constexpr int64_t kLong = 16384, kLongGrad = 12288;

// The gradient's workgroups for rows of r threads, and so parts of the columns' sums: as many as run at once, or for few
// rows one per CU, since each part is written and read again.  Measured, us, with 256 of 512 threads and 768 of 256: 4,096 x
// 768 of 16 bits 12.9, 17.5; 16,384 x 768 24, 28; 65,536 x 768 77, 72; 4,096 x 4,096 31, 36; 44,479 x 96 14, 18; 60,001 x 1,001
// floats 147, 147; 500,000 x 64 83, 75.
struct Grid {
  int threads;
  int64_t blocks;
};
constexpr Grid grad_grid(int64_t n, int r) {
  const bool few = r <= 256 && n * r <= 64 * 32768;
  const int threads = few || r > 256 ? 512 : 256;
  const int64_t groups = threads / r;
  return {threads, std::min<int64_t>((n + groups - 1) / groups, few ? 256 : r <= 256 ? 768 : 512)};
}

// f(r, vectors), r one of R, 2 R, ... MOST.
template <int R, int MOST, class F, class E>
void with_threads(int64_t r, F f, E vectors) {
  if (r == R) f(std::integral_constant<int, R>(), vectors);
  else if constexpr (R < MOST) with_threads<2 * R, MOST>(r, f, vectors);
}

// f(threads per row, vectors per thread) for rows of `dim`, with one of the given numbers of vectors: the fewest places
// for them (those past the row stay idle), the number named first if there are several; at most MOST threads.
// Measured with 1 to 8 vectors: values of 16 bits take 12 to 35 % more with one or two of them, 10 % more with six or eight,
// floats 10 and 20 % (fewer bytes on their way for each wave, or fewer waves).
template <int MOST, int FIRST, int... MORE, class F>
void by_width(int64_t dim, F f) {
  auto threads = [&](int64_t vectors) {
    int64_t r = 4;
    while (r * 4 * vectors < dim) r *= 2;
    return r;
  };
  int best = FIRST;
  ((best = threads(MORE) <= MOST && (threads(best) > MOST || threads(MORE) * MORE < threads(best) * best) ? MORE : best), ...);
  const int64_t r = threads(best);
  auto go = [&](auto vectors) {
    using E = decltype(vectors);
    if (E::value != best) return;
    with_threads<4, MOST>(r, f, E());
  };
  go(std::integral_constant<int, FIRST>());
  (go(std::integral_constant<int, MORE>()), ...);
}

// The same for the gradient.  Past 8,192 six vectors: 1,024 threads would not have the registers (5,000 x 12,288 of 16 bits:
// 110 us; before a row was asked for ahead 126, then with 1,024 threads 185, as long rows 246).  Rows of up to 64 values one or
// two vectors, or three (with four: 1M x 64 of 16 bits 143 us, here 90; 1M x 32 65, 51; 2M x 16 114, 67; 500,000 x 64 floats
// 81, 75).
template <class F>
void by_grad_width(int64_t dim, F f) {
  if (dim > 8192) f(std::integral_constant<int, 512>(), std::integral_constant<int, 6>());
  else if (dim <= 64) by_width<8, 2, 3, 1>(dim, f);
  else by_width<512, 4, 3>(dim, f);
}

int pitch_of(int64_t dim) { return (int)((dim + 3) / 4 * 4); }

int64_t long_slices(int64_t n, int64_t dim) { return std::min<int64_t>(n, std::max<int64_t>(1, 2048 / ((dim + 1023) / 1024))); }

int64_t workspace_bytes(int64_t n, int64_t dim) {
  if (n == 0 || dim == 0) return 0;
  if (dim > kLongGrad) return n * (int64_t)sizeof(Moments) + long_slices(n, dim) * 2 * pitch_of(dim) * 4;
  int64_t blocks = 0;
  by_grad_width(dim, [&](auto threads, auto) { blocks = grad_grid(n, decltype(threads)::value).blocks; });
  return blocks * 2 * pitch_of(dim) * 4;
}

// Whether results go past the L2: rows of whole lines or halves of them (300,000 x 96 of 16 bits: 28 -> 24 us), or long enough that their ends'
// lines do not matter (100,000 x 401 of 16 bits 43 -> 40, 60,001 x 1,001 floats 93 -> 88; but 200,000 x 255 53 -> 64).
template <class T>
bool past_the_l2(const T* out, int64_t n, int64_t dim, int64_t stride) {
  const bool whole = (reinterpret_cast<uintptr_t>(out) | stride * sizeof(T) | dim * sizeof(T)) % 64 == 0;
  return n * dim * (int64_t)sizeof(T) >= kStreamBytes && (whole || dim * sizeof(T) >= 768);
}

template <class T>
void norm(const void* x, int64_t n, int64_t dim, int64_t stride, const void* weight, const void* bias, int param_type,
          float eps, void* y, int64_t y_stride, hipStream_t st) {
  const T* in = static_cast<const T*>(x);
  T* out = static_cast<T*>(y);
  const bool stream = past_the_l2<T>(out, n, dim, y_stride);
  if (dim > kLong) {
    hipLaunchKernelGGL(norm_long_kernel<T>, dim3((unsigned)std::min<int64_t>(n, 1 << 20)), dim3(1024), 0, st, in, n, dim,
                       stride, weight, bias, param_type, eps, out, y_stride, stream);
  } else {
    auto go = [&](auto threads, auto vectors) {
      constexpr int R = decltype(threads)::value, E = decltype(vectors)::value, T0 = R > 256 ? R : 256;
      const int64_t blocks = std::min<int64_t>((n + T0 / R - 1) / (T0 / R), 256 * 2048 / T0);
      hipLaunchKernelGGL((norm_kernel<T, R, E, T0>), dim3((unsigned)blocks), dim3(T0), 0, st, in, n, (int)dim, stride, weight,
                         bias, param_type, eps, out, y_stride, stream);
    };
    // Short rows of floats that are no whole lines: one vector per thread where that takes no more of them (500,000 x 100:
    // 90 us, with four vectors 117, 300,000 x 200: 108, 115; whole lines the other way: 500,000 x 128: 106, 99).
    // And rows of up to 64 values: floats one vector (1M x 64: 93 us, with four 105; 1M x 48: 76, with three 92; 2M x 32: 92, 126), 16 bits two
    // of more than 32 values (1M x 64: 61, with four 113) or one (3M x 16: 49, with three 79).
    if (sizeof(T) == 4 && dim <= 64) by_width<16, 1>(dim, go);
    else if (dim <= 32) by_width<8, 1>(dim, go);
    else if (dim <= 64) by_width<8, 2, 3>(dim, go);
    else if (sizeof(T) == 4 && dim <= 256 && dim % 32) by_width<64, 1, 3, 4>(dim, go);
    else by_width<1024, 3, 4>(dim, go);
  }
  HIP_OK(hipGetLastError());
}

template <class T>
void norm_grad(const void* x, int64_t n, int64_t dim, int64_t stride, const void* grad, int64_t grad_stride,
               const void* weight, int param_type, float eps, void* dx, int64_t dx_stride, void* dweight, void* dbias,
               void* workspace, hipStream_t st) {
  const T *in = static_cast<const T*>(x), *g = static_cast<const T*>(grad);
  T* out = static_cast<T*>(dx);
  const bool stream = past_the_l2<T>(out, n, dim, dx_stride);
  const int pitch = pitch_of(dim);
  const bool columns = dweight || dbias;
  float* parts = static_cast<float*>(workspace);
  int64_t count = 0;
  if (n > 0 && dim > kLongGrad) {
    Moments* moments = static_cast<Moments*>(workspace);
    parts = reinterpret_cast<float*>(moments + n);
    count = long_slices(n, dim);
    const unsigned wide = (unsigned)((dim + 1023) / 1024);
    hipLaunchKernelGGL(long_moments_kernel<T>, dim3((unsigned)std::min<int64_t>(n, 1 << 20)), dim3(1024), 0, st, in, n, dim,
                       stride, g, grad_stride, weight, param_type, eps, moments);
    hipLaunchKernelGGL(long_grad_kernel<T>, dim3(wide, (unsigned)count), dim3(256), 0, st, in, n, dim, stride, g, grad_stride,
                       weight, param_type, moments, out, dx_stride, columns ? parts : nullptr, pitch, stream);
  } else if (n > 0) {
    auto go = [&](auto threads, auto vectors) {
      constexpr int R = decltype(threads)::value, E = decltype(vectors)::value;
      const Grid grid = grad_grid(n, R);
      count = grid.blocks;
      auto launch = [&](auto workgroup) {
        constexpr int T0 = decltype(workgroup)::value;
        hipLaunchKernelGGL((norm_grad_kernel<T, R, E, T0>), dim3((unsigned)count), dim3(T0), 0, st, in, n, (int)dim, stride,
                           g, grad_stride, weight, param_type, eps, out, dx_stride, columns ? parts : nullptr, pitch, stream);
      };
      if (R > 256 || grid.threads == 512) launch(std::integral_constant<int, 512>());
      else if constexpr (R <= 256) launch(std::integral_constant<int, 256>());
    };
    by_grad_width(dim, go);
  }
  HIP_OK(hipGetLastError());
  if (columns) {
    hipLaunchKernelGGL(join_columns_kernel, dim3((unsigned)((dim + 31) / 32), 2), dim3(1024), 0, st, parts, count, (int)dim,
                       pitch, dweight, dbias, param_type);
    HIP_OK(hipGetLastError());
  }
}

void check_params(const char* name, const void* p, int64_t dim, int type) {
  if (p && dim > 0) check_matrix(name, p, 1, dim, dim, value_size(type));
}

void check_eps(float eps) {
  if (!(eps >= FLT_MIN && eps <= FLT_MAX)) qv::fail(QV_EINVAL, "eps must be positive, normal and finite");
}

void check_sizes(int64_t n, int64_t dim) {
  if (n < 0 || dim < 0) qv::fail(QV_EINVAL, "negative size");
  if (n > INT32_MAX) qv::fail(QV_EUNSUPPORTED, "more than 2^31 - 1 rows");
  if (dim > QV_LAYER_NORM_MAX_DIM) qv::fail(QV_EUNSUPPORTED, "rows longer than 2^24, the last whole number before a float leaves some out");
}

}  // namespace

extern "C" {

int qv_layer_norm(const void* d_x, int32_t type, int64_t rows, int64_t dim, int64_t x_stride, const void* d_weight,
                  const void* d_bias, int32_t param_type, float eps, void* d_y, int64_t y_stride, int device, void* stream) {
  return qv::guard([&] {
    check_sizes(rows, dim);
    check_matrix("x", d_x, rows, dim, x_stride, value_size(type));
    check_matrix("y", d_y, rows, dim, y_stride, value_size(type));
    value_size(param_type);
    check_params("weight", d_weight, dim, param_type);
    check_params("bias", d_bias, dim, param_type);
    check_eps(eps);
    if (rows == 0 || dim == 0) return;
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (type == QV_FLOAT) norm<float>(d_x, rows, dim, x_stride, d_weight, d_bias, param_type, eps, d_y, y_stride, st);
    else if (type == QV_BFLOAT16) norm<bf16>(d_x, rows, dim, x_stride, d_weight, d_bias, param_type, eps, d_y, y_stride, st);
    else norm<f16>(d_x, rows, dim, x_stride, d_weight, d_bias, param_type, eps, d_y, y_stride, st);
  });
}

int64_t qv_layer_norm_grad_workspace(int64_t rows, int64_t dim) {
  int64_t bytes = 0;
  const int rc = qv::guard([&] {
    check_sizes(rows, dim);
    bytes = workspace_bytes(rows, dim);
  });
  return rc == QV_OK ? bytes : rc;
}

int qv_layer_norm_grad(const void* d_x, int32_t type, int64_t rows, int64_t dim, int64_t x_stride, const void* d_grad,
                       int64_t grad_stride, const void* d_weight, int32_t param_type, float eps, void* d_dx,
                       int64_t dx_stride, void* d_dweight, void* d_dbias, void* d_workspace, int64_t workspace_bytes,
                       int device, void* stream) {
  return qv::guard([&] {
    check_sizes(rows, dim);
    check_matrix("x", d_x, rows, dim, x_stride, value_size(type));
    check_matrix("grad", d_grad, rows, dim, grad_stride, value_size(type));
    if (d_dx) check_matrix("dx", d_dx, rows, dim, dx_stride, value_size(type));
    value_size(param_type);
    check_params("weight", d_weight, dim, param_type);
    check_params("dweight", d_dweight, dim, param_type);
    check_params("dbias", d_dbias, dim, param_type);
    check_eps(eps);
    if (dim == 0 || (!d_dx && !d_dweight && !d_dbias)) return;
    const int64_t need = ::workspace_bytes(rows, dim);
    if (need > 0 && (!d_workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(d_workspace) % 16))
      qv::fail(QV_EINVAL, "workspace: missing, too small or not 16-byte aligned");
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto go = [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      norm_grad<T>(d_x, rows, dim, x_stride, d_grad, grad_stride, d_weight, param_type, eps, d_dx, dx_stride, d_dweight,
                   d_dbias, d_workspace, st);
    };
    if (type == QV_FLOAT) go(static_cast<float*>(nullptr));
    else if (type == QV_BFLOAT16) go(static_cast<bf16*>(nullptr));
    else go(static_cast<f16*>(nullptr));
  });
}

}  // extern "C"
