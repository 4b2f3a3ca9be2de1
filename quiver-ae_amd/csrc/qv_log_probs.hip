// qv_log_probs.hip -- log probabilities of given columns, entropy and best
// alternatives of each row of logits, and their gradient.
//
// Everything is computed in base 2 relative to a running largest value m: with c =
// log2(e) / T, s = sum 2^y and w = sum y 2^y over y = x c - m c, a row's ln S is
// log2(s) ln 2 and its entropy ln 2 (log2(s) - w / s).  One pass over the row: a lane
// keeps its own m, s and w and moves them to a new m only when a batch of its values
// holds a larger one.
// The reference subtracted is fl(m c), not m c, so that y is one fused multiply-add;
// the difference r = fma(m, c, -fl(m c)), exact, is the y of m itself and enters once at
// the end.  It is half a unit in the last place of m c at most: 1/32 below |m c| = 2^20,
// so that s >= 0.97, w <= s / 32, and no cancellation in log2(s) or the entropy passes
// that.  From 2^20 on (a lane that has seen only masks of some large finite value, or
// logits and temperatures far from common ones) it would grow past what 2^y can hold:
// there the reference is m c itself and y = (x - m) c (as half the difference, which no
// two floats make infinite, and twice c), two instructions.  Sums of lanes on
// different sides of 2^20 differ by r, which shift_of counts in.
//
// What bounds it: reading the logits, beside about 10 vector instructions and one
// exponential for each.  256 x 200,000 bfloat16 with 20 alternatives: 28 us a pass, 3.7
// TB/s (without alternatives 20.6, 5.0 TB/s); 1,000 x 100,003 floats with 50: 92 us, 4.4
// TB/s (73); 10,000 lists of 100 with 10: 9.4 us; one row of 1M: 13 us, of which the two
// launches are 6.  Gradient: 1,000 x 100,003 floats 137 us, 5.8 TB/s.
#include <algorithm>
#include <cmath>

#include "qv_dense.hpp"
#include "qv_device.hpp"

using namespace qv;
using namespace qv::dev;
using namespace qv::dense;

namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kBig = 0x1p20f;  // |m c| from here on: differences are taken before they are multiplied
constexpr float kNone = -200.f;  // 2^-200 is 0 in fp32: stands for -inf where it would be multiplied by 0
constexpr float kHalfNone = -150.f;  // the same where 2^y is squared

// ---- values ------------------------------------------------------------------

template <class T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  raw4 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      r[i] = __float_as_uint(v[i]);
    } else {
      typedef T t2 __attribute__((ext_vector_type(2)));
      t2 h;
      h[0] = (T)v[2 * i];
      h[1] = (T)v[2 * i + 1];
      r[i] = __builtin_bit_cast(uint32_t, h);
    }
  }
  *reinterpret_cast<raw4_any*>(p) = r;
}

// Maxima without the compiler's quieting of each operand (a NaN among the values
// shows in s).
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// A commutative f folded over the wave, the same in every lane: neighbours 1, 2, 4 and 8
// apart by DPP (within quads, then the mirrored half row and the rotated row, whose lanes
// agree by then), 16 and 32 by the permlane swaps.
template <class F>
__device__ __forceinline__ float wave_fold(float v, F f) {
  auto dpp = [&](auto control) {
    constexpr int kControl = decltype(control)::value;
    v = f(v, __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), kControl, 0xF, 0xF, true)));
  };
  dpp(std::integral_constant<int, 0xB1>());   // quad_perm [1,0,3,2]
  dpp(std::integral_constant<int, 0x4E>());   // quad_perm [2,3,0,1]
  dpp(std::integral_constant<int, 0x141>());  // row_half_mirror
  dpp(std::integral_constant<int, 0x128>());  // row_ror:8
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_fold(v, [](float a, float b) { return a + b; });
}

// ---- keys of the alternatives --------------------------------------------------

// Orders as the values do, larger first by larger key, equal values (the two
// zeros among them) the lower column first; never 0 for a value above -inf.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t rank) {
  return __uint_as_float(rank & 0x80000000u ? rank ^ 0x80000000u : ~rank);
}
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t column) {
  return ((uint64_t)rank_of(x) << 32) | (uint32_t)~column;
}

// The 64 largest of two lists of 64, both and the result in descending order.
__device__ __forceinline__ uint64_t merge_desc(uint64_t a, uint64_t b) {
  const int lane = opaque_lane();
  const int from = (63 - lane) << 2;
  const uint64_t r = ((uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)(b >> 32)) << 32) |
                     (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)b);
  uint64_t key = umax64(a, r);
  key = cx_stage<32>(key, lane, false);
  key = cx_stage<16>(key, lane, false);
  key = cx_stage<8>(key, lane, false);
  key = cx_stage<4>(key, lane, false);
  key = cx_stage<2>(key, lane, false);
  key = cx_stage<1>(key, lane, false);
  return key;
}

constexpr uint32_t kLowest = 0x00800000u;  // the lowest finite value's rank

// The largest t (of the top 16 bits) that at least k of the lanes' ranks reach.
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t rank, int k) {
  uint32_t t = 0;
#pragma unroll
  for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
    if (__popcll(__ballot(rank >= (t | bit))) >= k) t |= bit;
  return t;
}

// Descending across the wave; the first `count` lanes hold distinct keys, the others 0.
// Few are placed by counting the larger ones (4 instructions each, the bitonic sort
// about 230).
__device__ __forceinline__ uint64_t sort_desc(uint64_t key, int count) {
  if (count > 40) return wave_sort_desc(key);
  const int lane = lane_id();
  int place = 0;
  for (int l = 0; l < count; l += 4) {  // (what it counts past `count` are zeros)
#pragma unroll
    for (int e = 0; e < 4; e++) place += read_lane_u64(key, l + e) > key ? 1 : 0;
  }
  const int to = (lane < count ? place : lane) << 2;
  return ((uint64_t)(uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)(key >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)key);
}

// A wave's best keys: entry i of the list in lane i.  Candidates wait in LDS until
// there are 64 of them, or the pass ends; VALUES: as a value's bits and its column,
// which become a key when they are sorted.
constexpr int kPool = 128;

template <bool VALUES>
struct Best {
  uint64_t list = 0;
  uint64_t* pool;  // [kPool], this wave's
  int count = 0;   // in the pool
  bool some = false;
  int k;

  __device__ Best(uint64_t* pool_, int k_) : pool(pool_), k(k_) {}

  __device__ __forceinline__ uint64_t waiting(int i, int n) const {
    const uint64_t c = i < n ? pool[i] : 0;
    return !VALUES ? c : i < n ? rank_key(__uint_as_float((uint32_t)(c >> 32)), (uint32_t)c) : 0;
  }
  __device__ __forceinline__ void merge(uint64_t key, int n) {
    key = sort_desc(key, n);
    list = some ? merge_desc(list, key) : key;
    some = true;
  }
  __device__ __forceinline__ void offer(bool take, uint64_t candidate) {
    const uint64_t mask = __ballot(take);
    if (mask == 0) return;
    if (take) pool[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = candidate;
    count += __popcll(mask);
    if (count >= kWave) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      count -= kWave;
      merge(waiting(count + lane_id(), kPool), kWave);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  __device__ __forceinline__ void finish() {
    if (count == 0) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    merge(waiting(lane_id(), count), count);
    count = 0;
  }
  // Puts what is left of the list and the pool, from rank `least` on, behind the other waves' in `all`.
  __device__ __forceinline__ void hand_over(uint64_t* all, int* total, uint32_t least) const {
    auto put = [&](uint64_t key) {
      const bool take = key && (uint32_t)(key >> 32) >= least;
      const uint64_t mask = __ballot(take);
      if (mask == 0) return;
      int at = 0;
      if (lane_id() == 0) at = atomicAdd(total, __popcll(mask));
      at = read_lane_i32(at, 0);
      if (take) all[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = key;
    };
    if (some) put(list);
    if (count) put(waiting(lane_id(), count));
  }
};

// The best of what W waves handed over, by one wave, whatever order it lies in.
__device__ __forceinline__ uint64_t best_of(const uint64_t* all, int total, uint64_t* pool, int k) {
  Best<false> best(pool, k);
  for (int i = 0; i < total; i += kWave) {
    const uint64_t key = i + lane_id() < total ? all[i + lane_id()] : 0;
    best.offer(key != 0, key);
  }
  best.finish();
  return best.list;
}

// The bound that a workgroup's waves give together, from one each that ceil(k / waves) of its values reach.
__device__ __forceinline__ uint32_t common_bound(const volatile uint32_t* bounds, int waves, int k) {
  const int share = (k + waves - 1) / waves;
  return kth_of_lanes(lane_id() < waves ? bounds[lane_id()] : 0, (k + share - 1) / share);
}

// ---- sums ----------------------------------------------------------------------

__device__ __forceinline__ float scaled(float m, float c) { return m == -kInf ? 0.f : m * c; }
__device__ __forceinline__ bool is_big(float mc) { return !(fabsf(mc) < kBig); }

// Half of a - b, which is finite where both are (a - b itself passes the largest float at most by a factor of two).
__device__ __forceinline__ float half_apart(float a, float b) { return __fmaf_rn(a, 0.5f, -0.5f * b); }

// What the reference of m lacks of m c; mc: scaled(m, c).
__device__ __forceinline__ float residue(float m, float mc, float c) { return is_big(mc) ? 0.f : __fmaf_rn(m, c, -mc); }

// log2 of what sums relative to m are multiplied by when the reference becomes
// to >= m: the two references' difference, of rounded ones as they are, else from the
// difference of m and to.
__device__ __forceinline__ float shift_of(float m, float to, float c) {
  if (m == -kInf) return kNone;
  const float a = scaled(m, c), b = scaled(to, c);
  float d = a - b;
  if (is_big(a) || is_big(b)) d = m == to ? 0.f : half_apart(m, to) * (2.f * c) + (residue(to, b, c) - residue(m, a, c));
  return max2(d, kNone);
}

struct Sums {
  float m = -kInf, s = 0.f, w = 0.f;

  __device__ __forceinline__ void move(float to, float c) {
    const float d = shift_of(m, to, c), f = __builtin_amdgcn_exp2f(d);
    w = f * __fmaf_rn(d, s, w);
    s = f * s;
    m = to;
  }
  __device__ __forceinline__ void add(Sums o, float c) {
    const float to = max2(m, o.m);
    move(to, c);
    o.move(to, c);
    s = s + o.s;
    w = w + o.w;
  }
  __device__ __forceinline__ float4 packed() const { return make_float4(m, s, w, 0.f); }
  static __device__ __forceinline__ Sums of(float4 p) {
    Sums o;
    o.m = p.x;
    o.s = p.y;
    o.w = p.z;
    return o;
  }
  // Over the wave, in a fixed order, the same in every lane.
  __device__ __forceinline__ void fold(float c) {
    move(wave_fold(m, [](float a, float b) { return max2(a, b); }), c);
    s = wave_sum(s);
    w = wave_sum(w);
  }
};

// One wave's pass over columns [from, to) of a row, every `step` batches of N U-vector loads.
template <class T, int U, bool TOP>
struct Pass {
  static constexpr int N = U * kVec<T>;
  static constexpr int kBatch = kWave * N;  // columns of a batch: vector u of lane l at (64 u + l) kVec
  Sums sum;
  float c, mc = 0.f;
  bool big = false;
  float least = -__FLT_MAX__;  // values below it are not among the k largest
  Best<true> best;

  __device__ Pass(float c_, uint64_t* pool, int k) : c(c_), best(pool, k) {}

  // `shared`: the `waves` waves' bounds when all of them have batches (ranks), or null.
  __device__ __forceinline__ void values(const float (&v)[N], int column, int turn, int waves, volatile uint32_t* shared) {
    constexpr int kGroup = 4;
    float part[N / kGroup], top;
#pragma unroll
    for (int g = 0; g < N / kGroup; g++)
      part[g] = max2(max3(v[kGroup * g], v[kGroup * g + 1], v[kGroup * g + 2]), v[kGroup * g + 3]);
    if constexpr (N == 4) top = part[0];
    else if constexpr (N == 8) top = max2(part[0], part[1]);
    else top = max2(max3(part[0], part[1], part[2]), part[3]);
    if (__any(top > sum.m)) {
      sum.move(max2(sum.m, top), c);
      mc = scaled(sum.m, c);
      big = __any(is_big(mc));
    }
    float s = 0.f, w = 0.f;
    if (!big) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float y = __fmaf_rn(v[i], c, -mc), e = __builtin_amdgcn_exp2f(y);
        s = s + e;
        w = __fmaf_rn(e, max2(y, kNone), w);
      }
    } else {
      const bool far = is_big(mc);
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float y = far ? half_apart(v[i], sum.m) * (2.f * c) : __fmaf_rn(v[i], c, -mc), e = __builtin_amdgcn_exp2f(y);
        s = s + e;
        w = __fmaf_rn(e, max2(y, kNone), w);
      }
    }
    sum.s = sum.s + s;
    sum.w = sum.w + w;
    if constexpr (TOP) {
      if (turn == 0 || __any(top >= least)) {
        // k lanes have seen a value that large (then about 64 ln(64 / (64 - k)) values pass in all), or their share of k
        // in each of the workgroup's waves (with four of them a third of what passes by their own bounds); renewed in
        // turns 0, 1, 3, 7, ...
        if ((turn & (turn + 1)) == 0) {
          uint32_t t;
          if (shared) {
            t = kth_of_lanes(rank_of(sum.m), (best.k + waves - 1) / waves);
            if (lane_id() == 0) shared[wave_id()] = t;
            if (turn == 0) __syncthreads();
            t = common_bound(shared, waves, best.k);
          } else {
            t = kth_of_lanes(rank_of(sum.m), best.k);
          }
          least = max2(least, value_of(max(kLowest, t)));
        }
#pragma unroll
        for (int g = 0; g < N / kGroup; g++) {
          if (!__any(part[g] >= least)) continue;
#pragma unroll
          for (int i = kGroup * g; i < kGroup * (g + 1); i++) {
            const int at = column + (i / kVec<T>)*kWave * kVec<T> + i % kVec<T>;
            best.offer(v[i] >= least, (uint64_t)__float_as_uint(v[i]) << 32 | (uint32_t)at);
          }
        }
      }
    }
  }

  // Batches b, b + step, ... of columns [from, to), the next one's values on their way.  Always inline: in a function of
  // its own the uniform bounds count as per-lane ones, with a stack and three times the time.
  __device__ __forceinline__ void run(const T* __restrict__ x, int64_t from, int64_t to, int b, int step,
                                      volatile uint32_t* shared) {
    const int lane = lane_id();
    int turn = 0;
    raw4 r[U];
    int64_t at = from + (int64_t)b * kBatch;
    auto load = [&](int64_t where) {
#pragma unroll
      for (int u = 0; u < U; u++) r[u] = load_raw(x + where + (u * kWave + lane) * kVec<T>);
    };
    if (at + kBatch <= to) load(at);
    while (at < to) {
      float v[N];
      const int64_t mine = at + lane * kVec<T>, next = at + (int64_t)step * kBatch;
      if (at + kBatch <= to) {
#pragma unroll
        for (int u = 0; u < U; u++) unpack<T>(r[u], v + u * kVec<T>);
      } else {
#pragma unroll
        for (int u = 0; u < U; u++)
          load_tail(x + mine + u * kWave * kVec<T>, to - mine - u * kWave * kVec<T>, -kInf, v + u * kVec<T>);
      }
      if (next + kBatch <= to) load(next);
      values(v, (int)mine, turn++, step, shared);
      at = next;
    }
    sum.fold(c);
  }
};

struct Out {
  const int32_t* targets;
  int per_row, topk;
  float *target, *entropy, *lse, *stats;
  int32_t* top_ids;
  float* top;
};

// A lane's given column and its logit, asked for before the row's pass.
struct Given {
  int32_t column = -1;
  float logit = 0.f;
};
template <class T>
__device__ __forceinline__ Given given_of(const T* __restrict__ x, int64_t row, int cols, const Out& o) {
  Given g;
  if (lane_id() < o.per_row) {
    g.column = o.targets[row * o.per_row + lane_id()];
    if (g.column >= 0 && g.column < cols) g.logit = (float)x[g.column];
  }
  return g;
}

// A row's results from its sums (in every lane) and its list, by one wave.
__device__ __forceinline__ void finish_row(const Given& given, int64_t row, int cols, const Sums& sum, uint64_t list,
                                           float c, float inv_t, const Out& o) {
  const int lane = lane_id();
  const bool odd = sum.s != sum.s, empty = sum.s == 0.f;
  const float nan = __builtin_nanf("");
  const float mc = scaled(sum.m, c);
  const float log2_s = log2f(sum.s) - residue(sum.m, mc, c);  // of the sum relative to m c itself
  const float ln_s = odd ? nan : empty ? -kInf : log2_s * kLn2;
  auto lp = [&](float v) { return odd ? nan : v == -kInf ? -kInf : __fmaf_rn(half_apart(v, sum.m), 2.f * inv_t, -ln_s); };
  if (lane == 0) {
    if (o.entropy) o.entropy[row] = odd ? nan : empty ? 0.f : (log2f(sum.s) - sum.w / sum.s) * kLn2;
    if (o.lse) o.lse[row] = odd ? nan : empty ? -kInf : __fmaf_rn(sum.m, inv_t, ln_s);
    o.stats[2 * row] = odd ? nan : sum.m;
    o.stats[2 * row + 1] = ln_s;
  }
  if (lane < o.per_row) {
    const int32_t j = given.column;
    o.target[row * o.per_row + lane] = j < 0 ? 0.f : j >= cols ? nan : lp(given.logit);
  }
  if (lane < o.topk) {
    const bool none = odd || list == 0;
    o.top_ids[row * o.topk + lane] = none ? -1 : (int32_t)~(uint32_t)list;
    o.top[row * o.topk + lane] = odd ? nan : none ? -kInf : lp(value_of((uint32_t)(list >> 32)));
  }
}

// One wave per row: no barrier, no join.
template <class T, int U, bool TOP>
__global__ __launch_bounds__(256) void log_probs_wave_kernel(const T* __restrict__ logits, int64_t rows, int cols,
                                                             int64_t stride, float c, float inv_t, Out o,
                                                             int64_t first_block) {
  __shared__ uint64_t pool[TOP ? 4 * kPool : 1];
  const int wave = wave_id();
  const int64_t row = (first_block + blockIdx.x) * 4 + wave;
  if (row >= rows) return;
  const T* x = logits + row * stride;
  const Given given = given_of(x, row, cols, o);
  Pass<T, U, TOP> pass(c, TOP ? pool + wave * kPool : pool, o.topk);
  pass.run(x, 0, cols, 0, 1, nullptr);
  if constexpr (TOP) pass.best.finish();
  finish_row(given, row, cols, pass.sum, pass.best.list, c, inv_t, o);
}

// One workgroup of W waves per chunk of a row.  With one chunk per row its results, else the
// chunk's sums and keys, for join_kernel.
template <class T, int U, bool TOP, int W>
__global__ __launch_bounds__(64 * W) void log_probs_block_kernel(const T* __restrict__ logits, int cols, int64_t stride,
                                                              float c, float inv_t, int64_t chunk, int splits, Out o,
                                                              float4* __restrict__ part,
                                                              uint64_t* __restrict__ part_keys) {
  __shared__ uint64_t pool[TOP ? W * kPool : 1];
  __shared__ uint64_t all[TOP ? 2 * W * kWave : 1];
  __shared__ float4 sums[W];
  __shared__ uint32_t bounds[W];
  __shared__ int total;
  const int tid = threadIdx.x, wave = wave_id(), lane = lane_id();
  const int64_t row = blockIdx.x / (unsigned)splits;
  const int split = (int)(blockIdx.x - row * splits);
  const T* x = logits + row * stride;
  if constexpr (TOP) {
    if (tid < W) bounds[tid] = 0;
    if (tid == 0) total = 0;
    __syncthreads();
  }
  Given given;
  if (splits == 1 && wave == 0) given = given_of(x, row, cols, o);
  using P = Pass<T, U, TOP>;
  P pass(c, TOP ? pool + wave * kPool : pool, o.topk);
  const int64_t from = (int64_t)split * chunk, to = min((int64_t)cols, from + chunk);
  pass.run(x, from, to, wave, W, to - from > (W - 1) * P::kBatch ? bounds : nullptr);
  if (lane == 0) sums[wave] = pass.sum.packed();
  if constexpr (TOP) {
    __syncthreads();
    pass.best.hand_over(all, &total, common_bound(bounds, W, o.topk));
  }
  __syncthreads();
  if (wave) return;
  Sums sum = Sums::of(sums[0]);
#pragma unroll
  for (int q = 1; q < W; q++) sum.add(Sums::of(sums[q]), c);
  const uint64_t list = TOP ? best_of(all, total, pool, o.topk) : 0;
  if (splits == 1) {
    finish_row(given, row, cols, sum, list, c, inv_t, o);
  } else {
    if (lane == 0) part[blockIdx.x] = sum.packed();
    if (TOP && lane < o.topk) part_keys[(int64_t)blockIdx.x * o.topk + lane] = list;
  }
}

// One workgroup per row joins its chunks.
template <class T, bool TOP>
__global__ __launch_bounds__(256) void join_kernel(const T* __restrict__ logits, int cols, int64_t stride, float c,
                                                   float inv_t, int splits, Out o, const float4* __restrict__ part,
                                                   const uint64_t* __restrict__ part_keys) {
  __shared__ uint64_t pool[TOP ? 4 * kPool : 1];
  __shared__ uint64_t all[TOP ? 2 * 4 * kWave : 1];
  __shared__ uint32_t leasts[4];
  __shared__ float4 sums[4];
  __shared__ int total;
  const int tid = threadIdx.x, wave = wave_id(), lane = lane_id();
  const int64_t row = blockIdx.x;
  Given given;
  if (wave == 0) given = given_of(logits + row * stride, row, cols, o);
  // the first keys are asked for before the sums
  const uint64_t* keys = TOP ? part_keys + row * splits * o.topk : nullptr;
  const int head = wave * kWave + lane, keys_of_row = splits * o.topk;
  uint64_t of_chunk = 0, ahead = 0;
  if constexpr (TOP) {
    if (head < splits) of_chunk = keys[(int64_t)head * o.topk];
    if (head < keys_of_row) ahead = keys[head];
  }
  Sums sum;
  for (int i = tid; i < splits; i += 256) {
    sum.add(Sums::of(part[row * splits + i]), c);
  }
  sum.fold(c);
  Best<false> best(TOP ? pool + wave * kPool : pool, o.topk);
  if constexpr (TOP) {
    // k of 64 chunks have a key with a rank that large
    const uint32_t mine = kth_of_lanes((uint32_t)(of_chunk >> 32), o.topk);
    if (lane == 0) leasts[wave] = mine;
    if (tid == 0) total = 0;
    __syncthreads();
    const uint32_t least = max(max(leasts[0], leasts[1]), max(leasts[2], leasts[3]));
    for (int i = wave * kWave; i < keys_of_row; i += 256) {
      const uint64_t key = ahead;
      ahead = i + 256 + lane < keys_of_row ? keys[i + 256 + lane] : 0;
      best.offer(key && (uint32_t)(key >> 32) >= least, key);
    }
    best.hand_over(all, &total, least);
  }
  if (lane == 0) sums[wave] = sum.packed();
  __syncthreads();
  if (wave) return;
  sum = Sums::of(sums[0]);
#pragma unroll
  for (int q = 1; q < 4; q++) sum.add(Sums::of(sums[q]), c);
  const uint64_t list = TOP ? best_of(all, total, pool, o.topk) : 0;
  finish_row(given, row, cols, sum, list, c, inv_t, o);
}

// ---- gradient ------------------------------------------------------------------

struct Weights {
  const float *stats, *entropy;
  const int32_t* targets;
  int per_row;  // 0 without g_target
  const int32_t* top_ids;
  int topk;     // 0 without g_top
  const float *g_target, *g_entropy, *g_lse, *g_top;
};

// One wave per chunk of a row: every column by the first two terms, p (a + b log2
// p) / T, then the columns that targets or alternatives name, whose weights add up in
// their order.  The named columns' logits are read before any column is written
// (the gradient may take the logits' place); a wave's stores to one address stay
// in order.
template <class T, int U>
__global__ __launch_bounds__(256) void log_probs_grad_kernel(const T* logits, int64_t units, int cols, int64_t stride,
                                                             float c, float inv_t, float root_inv_t, int chunk,
                                                             int splits, Weights g, T* grad, int64_t grad_stride,
                                                             int64_t first_block) {
  constexpr int N = U * kVec<T>, kBatch = kWave * N;
  const int64_t unit = (first_block + blockIdx.x) * 4 + wave_id();
  if (unit >= units) return;
  const int lane = lane_id();
  const int64_t row = unit / splits;
  const int64_t from = (unit - row * splits) * chunk, to = min((int64_t)cols, from + chunk);
  const T* x = logits + row * stride;
  T* dx = grad + row * grad_stride;
  const float m = g.stats[2 * row], ln_s = g.stats[2 * row + 1], log2_s = ln_s * kLog2e;
  const bool odd = m != m, empty = m == -kInf;

  int32_t id[2] = {-1, -1};
  float weight[2] = {0.f, 0.f}, total = 0.f;
  const int named = g.per_row + g.topk;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int i = h * kWave + lane;
    if (i >= named) continue;
    const bool t = i < g.per_row;
    const int64_t at = t ? row * g.per_row + i : row * g.topk + i - g.per_row;
    id[h] = t ? g.targets[at] : g.top_ids[at];
    weight[h] = t ? g.g_target[at] : g.g_top[at];
    // the log probability of a column past the row's end is NaN, and with it the derivative of what weighs it
    if (id[h] >= 0) total = total + (t && id[h] >= cols && weight[h] != 0.f ? __builtin_nanf("") : weight[h]);
  }
  if (named) total = wave_sum(total);
  if (g.g_lse) total = total - g.g_lse[row];
  const float ge = g.g_entropy ? g.g_entropy[row] : 0.f, h = g.g_entropy ? g.entropy[row] : 0.f;
  const float nan = __builtin_nanf("");
  const float a = odd ? nan : empty ? 0.f : -(total + ge * h);
  const float b = empty ? 0.f : -2.f * (ge * kLn2);
  // Half of log2 p.  The instruction gives 0 below 2^-126, which p passes and its root does not (4,096 x 4,096 bfloat16:
  // 12.8 us; with such p taken 2^64 larger and back 13.3).
  auto half_log2 = [&](float v) { return max2(__fmaf_rn(half_apart(v, m), c, -0.5f * log2_s), kHalfNone); };
  // The root of 1 / T goes with the root of p: 1 / T times a and b may be infinite where p is 0.
  auto dense = [&](float v) {
    const float y = half_log2(v), root = __builtin_amdgcn_exp2f(y) * root_inv_t;
    return __fmaf_rn(b, y, a) * root * root;
  };
  auto named_one = [&](float v, float weight) {
    const float y = half_log2(v), root = __builtin_amdgcn_exp2f(y);
    return (__fmaf_rn(b, y, a) * root * root + (empty ? 0.f : weight)) * inv_t;
  };

  float extra[2] = {0.f, 0.f}, kept[2] = {0.f, 0.f};
  uint64_t here[2] = {0, 0};
  if (named) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      here[q] = __ballot(id[q] >= from && id[q] < to);
      if (here[q] >> lane & 1) kept[q] = (float)x[id[q]];
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
      for (uint64_t left = here[q]; left; left &= left - 1) {
        const int l = __ffsll((long long)left) - 1;
        const int32_t j = read_lane_i32(id[q], l);
        const float w = read_lane_f32(weight[q], l);
        if (id[0] == j) extra[0] = extra[0] + w;
        if (id[1] == j) extra[1] = extra[1] + w;
      }
    }
  }
  for (int64_t at = from; at < to; at += kBatch) {
    const int64_t mine = at + lane * kVec<T>;
    if (at + kBatch <= to) {
      raw4 r[U];
#pragma unroll
      for (int u = 0; u < U; u++) r[u] = load_raw(x + mine + u * kWave * kVec<T>);
#pragma unroll
      for (int u = 0; u < U; u++) {
        float v[kVec<T>];
        unpack<T>(r[u], v);
#pragma unroll
        for (int i = 0; i < kVec<T>; i++) v[i] = dense(v[i]);
        store_vec(dx + mine + u * kWave * kVec<T>, v);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t p = mine + u * kWave * kVec<T>, valid = to - p;
        float v[kVec<T>];
        load_tail(x + p, valid, -kInf, v);
#pragma unroll
        for (int i = 0; i < kVec<T>; i++) v[i] = dense(v[i]);
        if (valid >= kVec<T>) {
          store_vec(dx + p, v);
        } else {
#pragma unroll
          for (int i = 0; i < kVec<T>; i++)
            if (i < valid) dx[p + i] = (T)v[i];
        }
      }
    }
  }
  if (here[0] | here[1]) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int q = 0; q < 2; q++)
      if (here[q] >> lane & 1)
        dx[id[q]] = (T)named_one(kept[q], extra[q]);
  }
}

// ---- launches --------------------------------------------------------------------

// How a call's rows are cut.
struct Plan {
  int waves;      // per workgroup; 1: one wave per row
  int splits;     // chunks per row (workgroups)
  int64_t chunk;  // columns
};

constexpr int64_t kStep = 4096;  // columns: one batch of each of a workgroup's four waves

// Measured with 10 alternatives of bfloat16 (with none in brackets), us by 1, 4 and 16 waves per row and cut into
// chunks of 4 waves each:
//   4,096 x 4,096: 14 (9), 23 (12), 72 (33)     2,000 x 20,000: 28 (17), 29 (17), 60 (29)
//   500 x 32,000: -, 18 (10), 21 (14), 21 (13)  300 x 128,000: -, 41 (22), 34 (24), 31 (20)
//   200 x 8,000: -, 9 (11), 11 (12), 13 (13)    200 x 128,000: -, 37 (20), 21 (15), 25 (16)
//   64 x 32,000: -, 16 (8), 13 (8), 16 (10)     64 x 128,000: -, 35 (20), 21 (14), 17 (10)
// So one wave per row where rows alone fill the GPU or are too short for more; else a workgroup per row, of 16 waves
// where there is at most one for each CU; and chunks, whose join costs 5 us, where long rows leave CUs without work.
Plan plan_of(int64_t rows, int64_t cols) {
  if (cols <= 1024 || rows >= 2048) return {1, 1, cols};
  if (rows > 256) {
    if (rows >= 400 || cols <= 65536) return {4, 1, cols};
  } else {
    if (cols <= 8192) return {4, 1, cols};
    if (cols <= 32768 || (rows > 96 && cols <= 131072) || rows > 204) return {16, 1, cols};
  }
  const int64_t most = (cols + kStep - 1) / kStep;
  const int64_t want = std::min<int64_t>(most, 1024 / rows);
  const int64_t steps = (most + want - 1) / want;
  return {4, (int)((most + steps - 1) / steps), steps * kStep};
}

// What the kernels multiply by.
float log2e_over(float temperature) { return (float)(1.44269504088896340736 / (double)temperature); }
float one_over(float temperature) { return (float)(1.0 / (double)temperature); }

template <class T, bool TOP>
void log_probs(const T* x, int64_t rows, int64_t cols, int64_t stride, float temperature, const Out& o, void* work,
               hipStream_t st) {
  const float c = log2e_over(temperature), inv_t = one_over(temperature);
  const Plan p = plan_of(rows, cols);
  if (p.waves == 1) {
    auto* kernel = cols <= kWave * kVec<T> ? log_probs_wave_kernel<T, 1, TOP> : log_probs_wave_kernel<T, 16 / kVec<T>, TOP>;
    in_launches((rows + 3) / 4, 256, [&](int64_t first, unsigned count) {
      hipLaunchKernelGGL(kernel, dim3(count), dim3(256), 0, st, x, rows, (int)cols, stride, c, inv_t, o, first);
      HIP_OK(hipGetLastError());
    });
    return;
  }
  float4* part = static_cast<float4*>(work);
  uint64_t* keys = reinterpret_cast<uint64_t*>(part + rows * p.splits);
  auto* kernel = p.waves == 16 ? log_probs_block_kernel<T, 16 / kVec<T>, TOP, 16> : log_probs_block_kernel<T, 16 / kVec<T>, TOP, 4>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * p.splits)), dim3(64 * p.waves), 0, st, x, (int)cols, stride, c, inv_t,
                     p.chunk, p.splits, o, part, keys);
  HIP_OK(hipGetLastError());
  if (p.splits > 1) {
    hipLaunchKernelGGL((join_kernel<T, TOP>), dim3((unsigned)rows), dim3(256), 0, st, x, (int)cols, stride, c, inv_t,
                       p.splits, o, part, keys);
    HIP_OK(hipGetLastError());
  }
}

template <class T>
void log_probs_grad(const T* x, int64_t rows, int64_t cols, int64_t stride, float temperature, const Weights& g,
                    T* grad, int64_t grad_stride, hipStream_t st) {
  constexpr int U = 16 / kVec<T>;
  const float c = log2e_over(temperature), inv_t = one_over(temperature);
  const int64_t chunk = 4 * kWave * U * kVec<T>;
  const int64_t splits = (cols + chunk - 1) / chunk, units = rows * splits;
  in_launches((units + 3) / 4, 256, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL((log_probs_grad_kernel<T, U>), dim3(count), dim3(256), 0, st, x, units, (int)cols, stride, c,
                       inv_t, std::sqrt(inv_t), (int)chunk, (int)splits, g, grad, grad_stride, first);
    HIP_OK(hipGetLastError());
  });
}

int64_t workspace_of(int64_t rows, int64_t cols, int32_t topk) {
  const Plan p = plan_of(rows, cols);
  return p.splits > 1 ? rows * p.splits * (int64_t)(sizeof(float4) + sizeof(uint64_t) * topk) : 0;
}

void check_rows(int32_t type, int64_t rows, int64_t cols, int64_t stride, const void* x, float temperature,
                const int32_t* targets, int32_t per_row, int32_t topk) {
  check_matrix("logits", x, rows, cols, stride, value_size(type));
  if (!(temperature > 0.f) || !(2.f * log2e_over(temperature) < kInf) || !(one_over(temperature) > 0.f))
    qv::fail(QV_EINVAL, "temperature must be positive and finite, and 2 log2(e) / temperature a finite float");
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
    if (rows > INT32_MAX || cols > INT32_MAX) qv::fail(QV_EUNSUPPORTED, "more than 2^31 - 1 rows or columns");
    if (rows) bytes = workspace_of(rows, cols, topk);
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
    const int64_t need = workspace_of(rows, cols, topk);
    if (need) {
      if (workspace_bytes < need) qv::fail(QV_EINVAL, "workspace too small");
      check_matrix("workspace", d_workspace, 1, need, need, 16);
    }
    const OnDevice on(device);
    const Out o{d_targets, targets_per_row, topk, d_target, d_entropy, d_lse, d_stats, d_top_ids, d_top};
    auto go = [&](auto* x) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
      const hipStream_t st = static_cast<hipStream_t>(stream);
      if (topk) log_probs<T, true>(x, rows, cols, stride, temperature, o, d_workspace, st);
      else log_probs<T, false>(x, rows, cols, stride, temperature, o, d_workspace, st);
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
    const Weights g{d_stats, d_entropy, d_targets, d_g_target ? targets_per_row : 0, d_top_ids, d_g_top ? topk : 0,
                    d_g_target, d_g_entropy, d_g_lse, d_g_top};
    const OnDevice on(device);
    auto go = [&](auto* x) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
      log_probs_grad<T>(x, rows, cols, stride, temperature, g, static_cast<T*>(d_grad), grad_stride,
                        static_cast<hipStream_t>(stream));
    };
    if (type == QV_FLOAT) go(static_cast<const float*>(d_logits));
    else if (type == QV_BFLOAT16) go(static_cast<const bf16*>(d_logits));
    else go(static_cast<const f16*>(d_logits));
  });
}

}  // extern "C"
