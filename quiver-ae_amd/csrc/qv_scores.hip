// qv_scores.hip -- rows to 8 bits with a scale each, and the integer product of two
// such matrices.
#include <algorithm>
#include <atomic>

#include "qv_dense.hpp"
#include "qv_device.hpp"

using namespace qv;
using namespace qv::dev;
using namespace qv::dense;

namespace {

// ---- rows to 8 bits --------------------------------------------------------------
//
// A row is read once, by a group of G lanes that hold it in registers (E loads of 16
// bytes each) between the search for its largest magnitude and the rounding; R rows
// per group at once keep more loads in flight.  Bound by memory: one read, a quarter
// (of 16-bit values half) of it written; 1M x 128 floats take 125 us, 5.15 TB/s (a large
// copy runs at 4.9), 352 us with a wave per row and the row read twice.  Magnitudes are
// compared as whole numbers, whose order is theirs, with infinities and NaN above all.

constexpr uint32_t kTinyBits = 0x04000000u;  // 2^-119: below it 127 / a comes near the largest float
constexpr uint32_t kHugeBits = 0x7e800000u;  // 2^126: above it 1 / a is subnormal and keeps fewer bits
constexpr uint32_t kInfBits = 0x7f800000u;

// Largest value over the group of G lanes (a power of two) that the lane is in.
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  if constexpr (G >= 2) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
  if constexpr (G >= 4) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
  if constexpr (G >= 8) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));  // row_half_mirror
  if constexpr (G >= 16) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true));  // row_ror:8
  if constexpr (G >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(p[0], p[1]);
  }
  if constexpr (G >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(p[0], p[1]);
  }
  return v;
}

struct RowScale {
  float inv, scale;
};
__device__ __forceinline__ RowScale scale_of(uint32_t top) {
  const float a = __uint_as_float(top);
  if (top >= kInfBits) return {0.f, __builtin_nanf("")};
  if (top < kTinyBits) return {0.f, 0.f};
  const float h = top >= kHugeBits ? 0x1p-8f : 1.f;  // both products with it are exact
  return {1.f / (a * h) * (127.f * h), a / 127.f};
}

// x 127 / a to the nearest whole number, halves to even, in the low byte: adding 1.5 2^23
// rounds to it (|x| 127 / a <= 127 and a little).  inv 0 gives 0 for every x, infinities and NaN too.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return inv != 0.f ? __float_as_uint(x * inv + 12582912.f) : 0u;
}

template <class T>
__device__ __forceinline__ void store_codes(int8_t* row, int64_t j, int64_t dim, const float* v, float inv) {
  uint32_t word[kVec<T> / 4];
#pragma unroll
  for (int w = 0; w < kVec<T> / 4; w++) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = code_of(v[4 * w + i], inv);
    // bytes 0 of four words into one
    const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0c);
    word[w] = lo | hi;
  }
  if (j + kVec<T> <= dim) {
    __builtin_memcpy(row + j, word, kVec<T>);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; i++)
      if (j + i < dim) row[j + i] = (int8_t)(word[i / 4] >> (8 * (i % 4)));
  }
}

template <class T, int G, int E, int R>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t n, int64_t dim, int64_t stride,
                                                       int8_t* __restrict__ codes, int64_t code_stride,
                                                       float* __restrict__ scales, int64_t first_block) {
  constexpr int kGroups = 256 / G;
  const int lane = threadIdx.x % G;
  const int64_t first = (first_block + blockIdx.x) * kGroups * R + threadIdx.x / G;
  float v[R][E * kVec<T>];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int64_t row = min(first + r * kGroups, n - 1);
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int64_t j = (int64_t)(e * G + lane) * kVec<T>;
      load_tail(x + row * stride + j, dim - j, 0.f, v[r] + e * kVec<T>);
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int64_t row = first + r * kGroups;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < E * kVec<T>; i++) top = max(top, __float_as_uint(v[r][i]) & 0x7fffffffu);
    const RowScale s = scale_of(group_max<G>(top));
    if (row >= n) continue;
#pragma unroll
    for (int e = 0; e < E; e++)
      store_codes<T>(codes + row * code_stride, (int64_t)(e * G + lane) * kVec<T>, dim, v[r] + e * kVec<T>, s.inv);
    if (lane == 0) scales[row] = s.scale;
  }
}

// Rows longer than a wave holds: one workgroup per row, which is read again (from the
// caches) for the rounding.
template <class T>
__global__ __launch_bounds__(256) void quantize_long_kernel(const T* __restrict__ x, int64_t dim, int64_t stride,
                                                            int8_t* __restrict__ codes, int64_t code_stride,
                                                            float* __restrict__ scales, int64_t first_block) {
  __shared__ uint32_t tops[4];
  const int64_t row = first_block + blockIdx.x;
  const T* src = x + row * stride;
  uint32_t top = 0;
  for (int64_t j = (int64_t)threadIdx.x * kVec<T>; j < dim; j += 256 * kVec<T>) {
    float v[kVec<T>];
    load_tail(src + j, dim - j, 0.f, v);
#pragma unroll
    for (int i = 0; i < kVec<T>; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  top = group_max<64>(top);
  if (lane_id() == 0) tops[wave_id()] = top;
  __syncthreads();
  const RowScale s = scale_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
  for (int64_t j = (int64_t)threadIdx.x * kVec<T>; j < dim; j += 256 * kVec<T>) {
    float v[kVec<T>];
    load_tail(src + j, dim - j, 0.f, v);
    store_codes<T>(codes + row * code_stride, j, dim, v, s.inv);
  }
  if (threadIdx.x == 0) scales[row] = s.scale;
}

// ---- product -------------------------------------------------------------------
//
// Sums of int8 products on the matrix cores (v_mfma_i32_32x32x32_i8, exact in
// int32).  The rows of b are the instruction's rows and the rows of a its columns,
// so a lane ends with four consecutive columns j of one output row i.
//
// k goes in stages of 128 bytes of each row, eight pieces of 16.  The last piece of
// a row whose length is no multiple of 16 is its last 16 bytes; what it repeats is
// zeroed in a, so every load is a whole one inside the row and b needs no mask.
// Rows past the end repeat the last row; what they give is not stored.
//
// Five kernels, by what bounds the product (product() below has the rule): up to 32 rows
// reading b; short rows writing the result; long rows the matrix cores, with tiles
// straight to LDS where their rows are aligned and through registers where not; and a
// plain one for rows shorter than a piece.  All sum in int32 and scale in the order of
// the definition, so they give the same bits.

typedef int32_t i4 __attribute__((ext_vector_type(4)));
typedef int32_t i16v __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef i4 i4_any __attribute__((aligned(1), may_alias));
typedef f4 f4_any __attribute__((aligned(4), may_alias));

constexpr int kLoadsDone = 0x0f70;  // s_waitcnt vmcnt(0)
constexpr int kStage = 128;         // bytes of k per stage
constexpr int64_t kFar = 1 << 23;   // operands' row strides from here on: 256 rows' offsets pass 31 bits

template <class O>
struct Product {
  const int8_t* a;
  int64_t a_stride;
  const float* a_scales;
  int64_t m;
  const int8_t* b;
  int64_t b_stride;
  const float* b_scales;
  const float* bias;
  int64_t n, k;
  O* out;
  int64_t out_stride;
};

// What a piece starting `over` bytes before its place repeats, zeroed.
__device__ __forceinline__ i4 without_first(i4 v, int over) {
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const int cut = over - 4 * w;
    v[w] = cut <= 0 ? v[w] : cut >= 4 ? 0 : (int32_t)((uint32_t)v[w] & (~0u << (8 * cut)));
  }
  return v;
}

__device__ __forceinline__ i16v mfma(i4 x, i4 y, i16v acc) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(x, y, acc, 0, 0, 0);
}

// Puts an instruction's result, 32 columns j of 32 rows i, into a wave's tile [32][stride] in LDS.
__device__ __forceinline__ void put_sums(int32_t* tile, int stride, const i16v& acc) {
  const int lane = lane_id();
#pragma unroll
  for (int g = 0; g < 4; g++) {
    i4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = acc[4 * g + e];
    *reinterpret_cast<i4*>(tile + (lane % 32) * stride + 8 * g + 4 * (lane / 32)) = v;
  }
}

// Two values in the output's 16 bits, halves to even.  By instruction: the compiler takes the bfloat16 one apart, and
// joins float16 to the product before it, whose rounding to fp32 is then left out.
template <class O>
__device__ __forceinline__ uint32_t two_of(float x, float y) {
  uint32_t both;
  if constexpr (std::is_same<O, bf16>::value) asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(both) : "v"(x), "v"(y));
  else asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(both) : "v"(x), "v"(y));
  return both;
}

// Of P pieces of 16 bytes in each of P lanes, the lane's own one of every lane: the P x P transposed.
template <int P>
__device__ __forceinline__ void swap_pieces(i4 (&u)[P]) {
  auto stage = [&](auto distance, auto control) {
    constexpr int D = decltype(distance)::value, kControl = decltype(control)::value;
    const bool up = lane_id() & D;
#pragma unroll
    for (int q = 0; q < P; q++) {
      if (q & D) continue;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const int lo = u[q][w], hi = u[q | D][w];
        const int other_lo = __builtin_amdgcn_mov_dpp(lo, kControl, 0xF, 0xF, true);
        const int other_hi = __builtin_amdgcn_mov_dpp(hi, kControl, 0xF, 0xF, true);
        u[q][w] = up ? other_hi : lo;
        u[q | D][w] = up ? hi : other_lo;
      }
    }
  };
  stage(std::integral_constant<int, 1>(), std::integral_constant<int, 0xB1>());                          // quad_perm [1,0,3,2]
  if constexpr (P == 4) stage(std::integral_constant<int, 2>(), std::integral_constant<int, 0x4E>());  // quad_perm [2,3,0,1]
}

// Scales the results of R instructions, 32 R columns from j of the rows around the lane's row i, and stores them from
// the registers, whole lines of 8 rows at once (half lines of 16 rows with 32 columns of 16 bits).  Of the four columns
// that a lane has of every eight, those of 16 bits pass to the other half of the wave and back, eight for a lane; then
// groups of lanes swap rows for pieces of one row.  (Pieces stored as they are, 32 bytes of 32 rows at once, take 5.0
// for 5.35 TB/s in aligned rows, 2 for 3.8 in others.)  `sb`, `add`: the columns' scales and biases in LDS.  WHOLE:
// all of it lies in the output.
template <bool WHOLE, int R, class O>
__device__ __forceinline__ void store_sums(const i16v* const (&acc)[R], float sa, const float* sb, const float* add,
                                           int64_t i, int64_t j, const Product<O>& p) {
  constexpr int V = 16 / (int)sizeof(O), N = 16 / V, P = R * N;  // columns of a piece, pieces of a result, of all
  const int half = lane_id() / 32, c = lane_id() % P;
  i4 u[P];
#pragma unroll
  for (int y = 0; y < R; y++) {
    float v[16];
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int at = 32 * y + 8 * g + 4 * half;
      const f4 s = *reinterpret_cast<const f4*>(sb + at), t = *reinterpret_cast<const f4*>(add + at);
#pragma unroll
      for (int e = 0; e < 4; e++) v[4 * g + e] = ((float)(*acc[y])[4 * g + e] * sa) * s[e] + t[e];
    }
#pragma unroll
    for (int q = 0; q < N; q++) {
      if constexpr (sizeof(O) == 4) {
#pragma unroll
        for (int e = 0; e < 4; e++) u[N * y + q][e] = __float_as_int(v[4 * q + e]);
      } else {
#pragma unroll
        for (int d = 0; d < 2; d++) {
          const auto both = __builtin_amdgcn_permlane32_swap(two_of<O>(v[8 * q + 2 * d], v[8 * q + 2 * d + 1]),
                                                             two_of<O>(v[8 * q + 4 + 2 * d], v[8 * q + 5 + 2 * d]), false, false);
          u[N * y + q][d] = (int)both[0];
          u[N * y + q][2 + d] = (int)both[1];
        }
      }
    }
  }
  swap_pieces(u);
  i -= c;
  j += 2 * V * c + V * half;
  O* to = p.out + (i * p.out_stride + j);
  if (WHOLE || j + V <= p.n) {
#pragma unroll
    for (int r = 0; r < P; r++)
      if (WHOLE || i + r < p.m) *reinterpret_cast<i4_any*>(to + r * p.out_stride) = u[r];
  } else {
#pragma unroll
    for (int r = 0; r < P; r++) {
      union {
        i4 raw;
        O o[V];
      } piece;
      piece.raw = u[r];
#pragma unroll
      for (int e = 0; e < V; e++)
        if (i + r < p.m && j + e < p.n) to[r * p.out_stride + e] = piece.o[e];
    }
  }
}

// The scales and biases of the 16 bytes of a row, of J columns from j0, that a lane stores.
template <int J, class O>
struct Columns {
  static constexpr int V = 16 / (int)sizeof(O), L = J / V, R = kWave / L;  // columns per lane, lanes per row, rows at once
  float scale[V], add[V];
  int64_t j;
  bool whole;

  __device__ __forceinline__ Columns(int64_t j0, const Product<O>& p) : j(j0 + lane_id() % L * V), whole(j + V <= p.n) {
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      if (whole) {
        const f4 s = *reinterpret_cast<const f4_any*>(p.b_scales + j + v);
        const f4 t = p.bias ? (f4)*reinterpret_cast<const f4_any*>(p.bias + j + v) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; e++) scale[v + e] = s[e], add[v + e] = t[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int64_t q = min(j + v + e, p.n - 1);
          scale[v + e] = p.b_scales[q];
          add[v + e] = p.bias ? p.bias[q] : 0.f;
        }
      }
    }
  }
};

// Scales and stores a wave's tile of 32 rows, whose scales `sa` gives, and J columns: 16 bytes of a row per lane.
template <int J, class O, class F>
__device__ __forceinline__ void store_tile(const int32_t* tile, int stride, int64_t i0, const Columns<J, O>& c, F sa,
                                           const Product<O>& p) {
  using C = Columns<J, O>;
  if (c.j >= p.n) return;
  const int lane = lane_id(), jl = lane % C::L * C::V;
#pragma unroll
  for (int t = 0; t < 32 / C::R; t++) {
    const int r = t * C::R + lane / C::L;
    const int64_t i = i0 + r;
    if (i >= p.m) break;
    const float scale = sa(t, r);
    union {
      O o[C::V];
      i4 raw;
    } u;
#pragma unroll
    for (int v = 0; v < C::V; v += 4) {
      const i4 sums = *reinterpret_cast<const i4*>(tile + r * stride + jl + v);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float x = ((float)sums[e] * scale) * c.scale[v + e];
        u.o[v + e] = (O)(p.bias ? x + c.add[v + e] : x);
      }
    }
    O* dst = p.out + i * p.out_stride + c.j;
    if (c.whole) {
      *reinterpret_cast<i4_any*>(dst) = u.raw;
    } else {
#pragma unroll
      for (int v = 0; v < C::V; v++)
        if (c.j + v < p.n) dst[v] = u.o[v];
    }
  }
}

// A tile's scales of BM rows and BN columns, and the columns' biases (-0, which changes no sum, without), in LDS, put
// there by T threads.
template <int BM, int BN, int T>
struct TileScales {
  static constexpr int kBytes = (BM + 2 * BN) * 4;
  float* sa;

  __device__ __forceinline__ explicit TileScales(char* at) : sa(reinterpret_cast<float*>(at)) {}
  template <class O>
  __device__ __forceinline__ TileScales(char* at, int64_t i0, int64_t j0, const Product<O>& p) : sa(reinterpret_cast<float*>(at)) {
    for (int r = threadIdx.x; r < BM; r += T) sa[r] = p.a_scales[min(i0 + r, p.m - 1)];
    for (int r = threadIdx.x; r < BN; r += T) {
      sa[BM + r] = p.b_scales[min(j0 + r, p.n - 1)];
      sa[BM + BN + r] = p.bias ? p.bias[min(j0 + r, p.n - 1)] : -0.f;
    }
  }
  // A wave's results, from row i and column j of the tile at (i0, j0) on.
  template <bool WHOLE, int TM, int TN, class O>
  __device__ __forceinline__ void store_all(i16v (&acc)[TM][TN], int i, int j, int64_t i0, int64_t j0, const Product<O>& p) const {
    constexpr int R = sizeof(O) == 2 && TN % 2 == 0 ? 2 : 1;
    const float *sb = sa + BM + j, *add = sb + BN;
    i += lane_id() % 32;
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y += R) {
        const i16v* from[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
          asm volatile("" : "+a"(acc[x][y + r]) : : "memory");  // in turn: none leaves its accumulators before
          from[r] = &acc[x][y + r];
        }
        store_sums<WHOLE>(from, sa[i + 32 * x], sb + 32 * y, add + 32 * y, i0 + i + 32 * x, j0 + j + 32 * y, p);
      }
  }
  template <int TM, int TN, class O>
  __device__ __forceinline__ void store(i16v (&acc)[TM][TN], int i, int j, int64_t i0, int64_t j0, const Product<O>& p) const {
    if (i0 + BM <= p.m && j0 + BN <= p.n) store_all<true>(acc, i, j, i0, j0, p);
    else store_all<false>(acc, i, j, i0, j0, p);
  }
};

// Workgroups go round the eight XCDs: each XCD gets a run of consecutive tiles.
__device__ __forceinline__ int64_t tile_of_block(int64_t block, int64_t tiles) {
  const int64_t xcd = block % 8, per = tiles / 8, more = tiles % 8;
  return xcd * per + min(xcd, more) + block / 8;
}

// A tile of BM x BN outputs per workgroup, WM x WN waves of 32 TM x 32 TN each.  Both
// operands' stages go through registers into LDS, the next one in flight while the
// matrix cores work on this one; piece q of row r lies at q ^ (r / 2 mod 8), so that the
// 16 rows that are read at once (64 banks, 256 bytes) lie in 16 different places.  For
// rows of any alignment and length; 2,048 x 4,096 x 4,096 to bfloat16: 44 us, 1.6 POP/s;
// rows of 4,080: 47 us, of 4,095, which begin at any byte: 63 us.
template <int BM, int BN, int WM, int WN, class O>
__global__ __launch_bounds__(64 * WM * WN, 1) void product_tile_kernel(Product<O> p, int64_t tiles_m, int64_t tiles_n,
                                                                       int64_t group) {
  constexpr int T = 64 * WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int LA = BM * 8 / T, LB = BN * 8 / T, kRows = T / 8;
  constexpr int kBuffer = (BM + BN) * kStage;  // two of them, then the scales
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, wave = wave_id(), lane = lane_id();
  const int wm = wave / WN, wn = wave % WN;
  // tiles in groups of `group` rows of tiles, down the rows first
  const int64_t t = tile_of_block(blockIdx.x, tiles_m * tiles_n);
  const int64_t g = t / (group * tiles_n), gm = min(group, tiles_m - g * group), in = t - g * group * tiles_n;
  const int64_t i0 = (g * group + in % gm) * BM, j0 = in / gm * BN;

  const int piece = tid % 8, r0 = tid / 8;
  const int8_t *a = p.a + i0 * p.a_stride, *b = p.b + j0 * p.b_stride;
  uint32_t at_a[LA], at_b[LB];
#pragma unroll
  for (int q = 0; q < LA; q++) at_a[q] = (uint32_t)(min((int64_t)(r0 + q * kRows), p.m - 1 - i0) * p.a_stride);
#pragma unroll
  for (int q = 0; q < LB; q++) at_b[q] = (uint32_t)(min((int64_t)(r0 + q * kRows), p.n - 1 - j0) * p.b_stride);
  const int k = (int)p.k, stages = (k + kStage - 1) / kStage;
  i4 ra[LA], rb[LB];
  auto load = [&](int s) {
    const int place = s * kStage + piece * 16, from = min(place, k - 16);
#pragma unroll
    for (int q = 0; q < LA; q++) ra[q] = *reinterpret_cast<const i4_any*>(a + (at_a[q] + (uint32_t)from));
#pragma unroll
    for (int q = 0; q < LB; q++) rb[q] = *reinterpret_cast<const i4_any*>(b + (at_b[q] + (uint32_t)from));
  };
  auto keep = [&](int s) {
    char* to = lds + (s & 1) * kBuffer + r0 * kStage + (piece ^ (r0 / 2 & 7)) * 16;
    if ((s + 1) * kStage > k) {
      const int over = max(0, s * kStage + piece * 16 - (k - 16));
#pragma unroll
      for (int q = 0; q < LA; q++) ra[q] = without_first(ra[q], over);
    }
#pragma unroll
    for (int q = 0; q < LA; q++) *reinterpret_cast<i4*>(to + q * kRows * kStage) = ra[q];
#pragma unroll
    for (int q = 0; q < LB; q++) *reinterpret_cast<i4*>(to + BM * kStage + q * kRows * kStage) = rb[q];
  };
  i16v acc[TM][TN];
#pragma unroll
  for (int x = 0; x < TM; x++)
#pragma unroll
    for (int y = 0; y < TN; y++) acc[x][y] = i16v{};
  const int row = lane % 32, half = lane / 32;
  i4 fa[2][TM], fb[2][TN];
  auto read = [&](int s, int q) {  // a step's operands: 32 bytes of k
    const char* from = lds + (s & 1) * kBuffer + ((2 * q + half) ^ (row / 2 & 7)) * 16 + row * kStage;
#pragma unroll
    for (int x = 0; x < TM; x++) fa[q & 1][x] = *reinterpret_cast<const i4*>(from + (wm * TM + x) * 32 * kStage);
#pragma unroll
    for (int y = 0; y < TN; y++)
      fb[q & 1][y] = *reinterpret_cast<const i4*>(from + BM * kStage + (wn * TN + y) * 32 * kStage);
  };
  load(0);
  keep(0);
  const TileScales<BM, BN, T> scales(lds + 2 * kBuffer, i0, j0, p);
  __syncthreads();
  for (int s = 0; s < stages; s++) {
    const bool more = s + 1 < stages;
    if (more) load(s + 1);
    read(s, 0);
#pragma unroll
    for (int q = 0; q < 4; q++) {
      if (q < 3) read(s, q + 1);
      if (q == 3 && more) keep(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < TM; x++)
#pragma unroll
        for (int y = 0; y < TN; y++) acc[x][y] = mfma(fb[q & 1][y], fa[q & 1][x], acc[x][y]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
  }
  scales.store(acc, wm * TM * 32, wn * TN * 32, i0, j0, p);
}

// The same tiles where the matrix cores are what bounds the product: stages of 64 bytes
// of k go straight from memory to LDS (no registers, no LDS writes to issue), NB of
// them at a time, so NB - 1 are on their way while one is used.  A stage is two steps
// of 32 bytes; the second step's operands are read while the first one's products run,
// and the next stage's first operands while the second one's do, so the one barrier
// per stage, between the two, finds the operands of what follows it in registers.
// Needs 16-byte aligned rows and k a multiple of 64.
// MANY: one workgroup per CU walks over tiles, and the stages run on from tile to tile:
// the next tile's first ones are on their way, and its first operands in registers, while
// the results are stored (10,000 x 50,048 x 512: 457 to 490 us, with a workgroup per tile
// 519 when it took 457).
// 4,096^3 to bfloat16: 67 to 71 us among other work, 2.0 POP/s (a library's int8 product
// with a 32-bit result: 69), 74 one after the other: then power holds the clock down.
// 8,192 x 8,192 x 4,096: 252 to 263 us (with the results through LDS and a tile per workgroup
// 273); 8,192^3 of zeros 349 us, 3.1 POP/s, of codes over the whole range 545 us at 1.5
// GHz (the matrix instruction alone reaches 4.5 and 3.3 POP/s).  Loads and LDS reads in
// runs of their own instead of between the products: a fifth more.
//
// The schedule's next N x (P matrix instructions, one of the given kind): a matrix
// instruction takes 32 cycles, in which a wave can issue a few others; in a run of
// their own they would leave the matrix pipe idle.
constexpr int kMfma = 0x008, kVmem = 0x010, kDsRead = 0x100;
template <int N, int KIND, int P>
__device__ __forceinline__ void between() {
#pragma unroll
  for (int i = 0; i < N; i++) {
    __builtin_amdgcn_sched_group_barrier(kMfma, P, 0);
    __builtin_amdgcn_sched_group_barrier(KIND, 1, 0);
  }
}

constexpr int kReadsDone = 0xc07f;  // s_waitcnt lgkmcnt(0)
template <int N>
constexpr int kWaitFor = (N & 15) | (N >> 4 << 14) | 0x0070;  // s_waitcnt vmcnt(N) lgkmcnt(0)

template <int BM, int BN, int WM, int WN, int NB, bool MANY, class O>
__global__ __launch_bounds__(64 * WM * WN, 1) void product_deep_kernel(Product<O> p, int64_t tiles_m, int64_t tiles_n,
                                                                       int64_t group) {
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32, kRow = 64;
  using Scales = TileScales<BM, BN, 64 * WM * WN>;
  constexpr int I = (BM + BN) / 16 / (WM * WN);  // loads of 16 rows per wave and stage
  static_assert(I % 2 == 0, "issued in halves");
  constexpr int kBuffer = (BM + BN) * kRow;
  extern __shared__ __align__(16) char lds[];
  const int wave = wave_id(), lane = lane_id(), wm = wave / WN, wn = wave % WN;
  const uint32_t stages = (uint32_t)p.k / kRow;  // NB at least
  const uint32_t tiles = (uint32_t)(tiles_m * tiles_n), tn = (uint32_t)tiles_n, rows = (uint32_t)group;
  int64_t i0, j0, next_i0, next_j0;
  auto place_next = [&](uint32_t turn) {
    const uint32_t t = (uint32_t)tile_of_block(turn, tiles), g = t / (rows * tn), in = t - g * rows * tn;
    const uint32_t gm = min(rows, (uint32_t)tiles_m - g * rows);
    next_i0 = (int64_t)(g * rows + in % gm) * BM;
    next_j0 = (int64_t)(in / gm) * BN;
  };

  // piece q of row r lies at q ^ (r / 4 mod 4): the lanes of a load write 1 KB in a row, so what they load is
  // permuted instead
  const int piece = (lane % 4) ^ (lane / 16);
  const int8_t* src[I];
  char* scales_at = lds + NB * kBuffer;  // of this tile and the next one
  // the next tile's rows, and its scales on their way
  auto turn_to_next = [&](int buffer) {
#pragma unroll
    for (int q = 0; q < I; q++) {
      const int r = (wave * I + q) * 16 + lane / 4;
      src[q] = (r < BM ? p.a + min(next_i0 + r, p.m - 1) * p.a_stride : p.b + min(next_j0 + r - BM, p.n - 1) * p.b_stride) + piece * 16;
    }
    float* to = reinterpret_cast<float*>(scales_at + buffer * Scales::kBytes);
    for (int r = wave * kWave; r < BM + (p.bias ? 2 : 1) * BN; r += kWave * WM * WN) {
      const float* from = r < BM        ? p.a_scales + min(next_i0 + r + lane, p.m - 1)
                          : r < BM + BN ? p.b_scales + min(next_j0 + r - BM + lane, p.n - 1)
                                        : p.bias + min(next_j0 + r - BM - BN + lane, p.n - 1);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                       (__attribute__((address_space(3))) void*)(to + r), 4, 0, 0);
    }
  };
  // a half of a stage's loads (with one tile, stages past the last one repeat it: as many loads as the waits count)
  auto issue = [&](uint32_t s, int part) {
    char* to = lds + s % NB * kBuffer + wave * I * 1024;
    const uint32_t from = MANY ? 0 : min(s, stages - 1) * kRow;
#pragma unroll
    for (int q = part * I / 2; q < (part + 1) * I / 2; q++) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[q] + from),
                                       (__attribute__((address_space(3))) void*)(to + q * 1024), 16, 0, 0);
      if (MANY) src[q] += kRow;
    }
  };
  i16v acc[TM][TN];
  const int row = lane % 32, half = lane / 32;
  i4 fa[2][TM], fb[2][TN];
  auto read = [&](uint32_t s, int q) {
    const char* from = lds + s % NB * kBuffer + ((2 * q + half) ^ (row / 4 % 4)) * 16 + row * kRow;
#pragma unroll
    for (int x = 0; x < TM; x++) fa[q][x] = *reinterpret_cast<const i4*>(from + (wm * TM + x) * 32 * kRow);
#pragma unroll
    for (int y = 0; y < TN; y++) fb[q][y] = *reinterpret_cast<const i4*>(from + (BM + (wn * TN + y) * 32) * kRow);
  };
  auto products = [&](int q) {
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y++) acc[x][y] = mfma(fb[q][y], fa[q][x], acc[x][y]);
  };
  auto meet = [] {  // nothing of a stage moves over it
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  if (!p.bias) {
    for (int r = threadIdx.x; r < BN; r += 64 * WM * WN)
#pragma unroll
      for (int buffer = 0; buffer < 2; buffer++) Scales(scales_at + buffer * Scales::kBytes).sa[BM + BN + r] = -0.f;
  }
  uint32_t turn = blockIdx.x;
  place_next(turn);
  turn_to_next(0);
#pragma unroll
  for (int s = 0; s < NB; s++) {
    issue(s, 0);
    if (s + 1 < NB) issue(s, 1);
  }
  __builtin_amdgcn_s_waitcnt(kWaitFor<(NB - 1) * I - I / 2>);
  meet();
  read(0, 0);
  __builtin_amdgcn_s_waitcnt(kReadsDone);
  uint32_t s = 0, buffer = 0;
  do {
    i0 = next_i0;
    j0 = next_j0;
    turn += gridDim.x;
    if (MANY) place_next(min(turn, tiles - 1));  // (after the last tile some tile's first stages, which nobody reads)
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y++) {
        acc[x][y] = i16v{};
        asm volatile("" : "+a"(acc[x][y]));
      }
    for (uint32_t left = stages; left > 0; left--, s++) {
      read(s, 1);
      issue(s + NB - 1, 1);
      products(0);
      between<TM + TN, kDsRead, 1>();
      between<I / 2, kVmem, 2>();
      __builtin_amdgcn_sched_barrier(0);
      // stage s + 1 is there and every wave has read stage s
      __builtin_amdgcn_s_waitcnt(kWaitFor<(NB - 2) * I>);
      meet();
      if (MANY && left == NB) turn_to_next(buffer ^ 1);
      read(s + 1, 0);
      issue(s + NB, 0);
      products(1);
      between<TM + TN, kDsRead, 1>();
      between<I / 2, kVmem, 2>();
      __builtin_amdgcn_s_waitcnt(kReadsDone);  // long since: said for the compiler, which else waits at the loop's top
      __builtin_amdgcn_sched_barrier(0);
    }
    Scales(scales_at + buffer * Scales::kBytes).store(acc, wm * TM * 32, wn * TN * 32, i0, j0, p);
    buffer ^= 1;
  } while (MANY && turn < tiles);
  __builtin_amdgcn_s_waitcnt(kWaitFor<0>);  // no load into LDS outlives the wave
}

// Short rows, k <= 32 KS, whose product is mostly writing: 32 rows of a stay in a wave's
// registers while its workgroup (128 rows) walks over tiles of 64 rows of b, through
// LDS with the next two tiles on their way.
//
// Memory takes whole aligned lines of 128 bytes at 5.4 TB/s and rows cut elsewhere at
// 3.3 to 3.8, and rows of an odd length begin anywhere.  So a wave keeps, per row, a
// ring of two lines in LDS in which an element's place follows its address: a line is
// written whole as soon as its last column is there, and only the first and the last
// one of a walk are written in parts.
// 10,000 x 50,001 x 128 to bfloat16: 255 us call after call into the same scores, 4.0 TB/s,
// 264 into others each time (tiles with unaligned stores: 503), to float 4.5 TB/s;
// without its stores the kernel takes 171 us.
template <int KS, bool BIAS, class O>
__global__ __launch_bounds__(256, KS == 4 ? 3 : 2) void product_panel_kernel(Product<O> p, int64_t panels, int64_t tiles_n,
                                                               int64_t slices) {
  constexpr int PC = 2 * KS, kRow = 32 * KS, L = 64 * PC / 256, kRows = 256 / PC;
  constexpr int S = (int)sizeof(O), E = 128 / S, V = 16 / S;   // elements of a line, of 16 bytes
  constexpr int kRing = 256, Y = E / 32;  // bytes of a row's ring; 32-column results to a line
  __shared__ __align__(16) char lds[2][64 * kRow];
  __shared__ __align__(256) char rings[4][32 * kRing];
  __shared__ __align__(16) float sa[128];
  __shared__ float sb[2][BIAS ? 2 : 1][64];  // a tile's scales and biases
  const int tid = threadIdx.x, wave = wave_id(), lane = lane_id(), row = lane % 32, half = lane / 32;
  const int64_t t = tile_of_block(blockIdx.x, panels * slices), slice = t / panels, i0 = (t - slice * panels) * 128;
  const int64_t first = tiles_n * slice / slices, end = tiles_n * (slice + 1) / slices;
  const int k = (int)p.k, piece = tid % PC, r0 = tid / PC, from = min(piece * 16, k - 16);
  auto swap = [](int r) { return KS == 4 ? r / 2 & 7 : r & 15; };  // as in the tiles, for rows of 128 or 256 bytes
  i4 rb[L];
  float rs = 0.f;
  const bool scales = tid < (BIAS ? 128 : 64);
  const float* scale_of = !BIAS || tid < 64 ? p.b_scales : p.bias;
  auto load = [&](int64_t tile) {
    const int8_t* b = p.b + tile * 64 * p.b_stride;
    const int last = (int)min(p.n - 1 - tile * 64, (int64_t)63);
#pragma unroll
    for (int q = 0; q < L; q++) rb[q] = *reinterpret_cast<const i4_any*>(b + (uint32_t)(min(r0 + q * kRows, last) * (int)p.b_stride + from));
    if (scales) rs = scale_of[tile * 64 + min(tid % 64, last)];
  };
  auto keep = [&](int buffer) {
#pragma unroll
    for (int q = 0; q < L; q++) {
      const int r = r0 + q * kRows;
      *reinterpret_cast<i4*>(lds[buffer] + r * kRow + (piece ^ swap(r)) * 16) = rb[q];
    }
    if (scales) sb[buffer][tid / 64][tid % 64] = rs;
  };
  load(first);
  const int64_t it = i0 + wave * 32;  // the wave's rows
  const int rows = (int)min(p.m - it, (int64_t)32);
  i4 fa[KS];
  {
    const int8_t* a = p.a + min(it + row, p.m - 1) * p.a_stride;
#pragma unroll
    for (int q = 0; q < KS; q++) {
      const int place = (2 * q + half) * 16, at = min(place, k - 16);
      fa[q] = without_first(*reinterpret_cast<const i4_any*>(a + at), place - at);
    }
  }
  if (tid < 128) sa[tid] = p.a_scales[min(i0 + tid, p.m - 1)];
  // elements of its line before a row's first one
  auto shift = [&](int r) { return (int)(reinterpret_cast<uintptr_t>(p.out + (it + r) * p.out_stride) % 128) / S; };
  char* ring = rings[wave];
  // where the columns of a line go in the ring, register 4 g + e of result y; those of the next line
  // half a ring on
  uint32_t place[Y][16];
  typedef __attribute__((address_space(3))) O lds_o;
#pragma unroll
  for (int g = 0; g < 4; g++)
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
      for (int y = 0; y < Y; y++) {
        const int at = (int)(first & 1) * 64 + 32 * y + row + shift(8 * g + 4 * half + e);
        place[y][4 * g + e] = lds_addr(ring) + 4 * half * kRing + (at * S & (kRing - 1));
      }
  // lines as they leave: 8 lanes a line, 8 rows at once
  constexpr int G = 4;
  const int c = lane % 8;
  char* line_to[G];
  int rel[G];
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int r = 8 * g + lane / 8, sh = shift(r);
    rel[g] = c * V - sh;
    line_to[g] = reinterpret_cast<char*>(p.out + (it + r) * p.out_stride + (first * 64 + rel[g]));
  }
  // line number `line` (the E elements from column line E - shift on) of every row, columns [lo, hi) of it
  const int64_t lo = first * 64;
  auto leave = [&](int64_t line, int64_t hi, int64_t step) {
    const int least = (int)max(lo - line * E, (int64_t)-1024), most = (int)min(hi - line * E, (int64_t)1024);
    const char* from = ring + (int)(line & 1) * 128 + c * 16;
    if (rows == 32 && least <= 1 - E && most >= E) {  // whole lines of all rows
#pragma unroll
      for (int g = 0; g < G; g++) {
        *reinterpret_cast<i4*>(line_to[g]) = *reinterpret_cast<const i4*>(from + (8 * g + lane / 8) * kRing);
        line_to[g] += step;
      }
      return;
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int r = 8 * g + lane / 8;
      union {
        i4 raw;
        O o[V];
      } u;
      u.raw = *reinterpret_cast<const i4*>(from + r * kRing);
      if (r < rows) {
        if (rel[g] >= least && rel[g] + V <= most) {
          *reinterpret_cast<i4*>(line_to[g]) = u.raw;
        } else {
#pragma unroll
          for (int v = 0; v < V; v++)
            if (rel[g] + v >= least && rel[g] + v < most) reinterpret_cast<O*>(line_to[g])[v] = u.o[v];
        }
      }
      line_to[g] += step;
    }
    // every store of this way is done: a later wait for loads then need not count them, and on the other way
    // waits for the loads before its four stores only
    __builtin_amdgcn_s_waitcnt(kLoadsDone);
  };
  keep(0);
  if (first + 1 < end) load(first + 1);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < KS; q++) asm volatile("" : "+v"(fa[q]));  // these are there: the loop's waits count its own
#pragma unroll
  for (int q = 0; q < L; q++) asm volatile("" : "+v"(rb[q]));
  asm volatile("" : "+v"(rs));
  for (int64_t tile = first; tile < end; tile++) {
    const int buffer = (int)(tile - first) & 1;
    const char* b = lds[buffer] + row * kRow;
    i16v acc[2] = {i16v{}, i16v{}};
#pragma unroll
    for (int q = 0; q < KS; q++)
#pragma unroll
      for (int y = 0; y < 2; y++)
        acc[y] = mfma(fa[q], *reinterpret_cast<const i4*>(b + y * 32 * kRow + ((2 * q + half) ^ swap(row)) * 16), acc[y]);
    if (tile + 1 < end) keep(buffer ^ 1);
    if (tile + 2 < end) load(tile + 2);
#pragma unroll
    for (int l = 0; l < 2 / Y; l++) {
      float scale[Y], add[Y];
#pragma unroll
      for (int y = 0; y < Y; y++) {
        const int j = (l * Y + y) * 32 + row;
        scale[y] = sb[buffer][0][j];
        add[y] = BIAS ? sb[buffer][BIAS][j] : 0.f;
      }
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const f4 s = *reinterpret_cast<const f4*>(sa + wave * 32 + 8 * g + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; e += 2)
#pragma unroll
          for (int y = 0; y < Y; y++) {
            typedef O o2 __attribute__((ext_vector_type(2)));
            float x[2];
#pragma unroll
            for (int d = 0; d < 2; d++) {
              x[d] = ((float)acc[l * Y + y][4 * g + e + d] * s[e + d]) * scale[y];
              if constexpr (BIAS) x[d] = x[d] + add[y];
            }
            o2 out;
            if constexpr (sizeof(O) == 2) out = __builtin_bit_cast(o2, two_of<O>(x[0], x[1]));
            else out = o2{x[0], x[1]};
#pragma unroll
            for (int d = 0; d < 2; d++) {
              uint32_t& at = place[y][4 * g + e + d];
              ((lds_o*)(uintptr_t)at)[(8 * g + e + d) * kRing / S] = out[d];
              at ^= 128;
            }
          }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      leave(tile * (2 / Y) + l, p.n, 128);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
  }
  leave(end * (2 / Y), min(end * 64, p.n), 0);
}

// Up to 32 rows of a against strips of 32 rows of b, one strip per wave at a time (WK =
// 1), or a strip's k cut over the WK waves of its workgroup.  A wave's stage of b goes
// through registers into an LDS area of its own, so no barrier holds it; the next one
// is in flight meanwhile.  a's operands come from the caches, once for all strips
// while k is a single stage.  Bound by reading b: 1 x 1M x 128 in 29.5 us, 4.6 TB/s (24
// us over and over, part of b being cached), 8 x 100,000 x 1,024 in 19 us, 5.3 TB/s.
template <int WK, class O>
__global__ __launch_bounds__(256) void product_strip_kernel(Product<O> p, int64_t strips, int64_t step) {
  constexpr int kTile = 32 + 4;
  __shared__ __align__(16) char lds[4][32 * kTile * 4];  // a stage of b, then the strip's sums
  const int wave = wave_id(), lane = lane_id();
  const int row = lane % 32, half = lane / 32;
  const int k = (int)p.k, stages = (k + kStage - 1) / kStage;
  const int r0 = lane / 8, piece = lane % 8;
  const int8_t* a_row = p.a + min((int64_t)row, p.m - 1) * p.a_stride;
  char* area = lds[wave];
  i4 fa[4], rb[4];
  auto load_a = [&](int s) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int place = s * kStage + (2 * q + half) * 16, from = min(place, k - 16);
      fa[q] = without_first(*reinterpret_cast<const i4_any*>(a_row + from), place - from);
    }
  };
  auto load_b = [&](int64_t strip, int s) {
    const int from = min(s * kStage + piece * 16, k - 16);
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int64_t r = min(strip * 32 + r0 + 8 * q, p.n - 1);
      rb[q] = *reinterpret_cast<const i4_any*>(p.b + r * p.b_stride + from);
    }
  };
  using C = Columns<32, O>;
  float sa[32 / C::R];  // of the rows that the lane stores
#pragma unroll
  for (int t = 0; t < 32 / C::R; t++) sa[t] = p.a_scales[min((int64_t)(t * C::R + lane / C::L), p.m - 1)];
  auto scale = [&](int t, int) { return sa[t]; };
  const int s0 = WK == 1 ? 0 : wave;
  int64_t strip = WK == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  if (WK == 1 && strip >= strips) return;
  if (s0 < stages) load_b(strip, s0);
  if (stages == 1 && s0 < stages) load_a(0);
  for (; strip < strips; strip += step) {
    i16v acc{};
    for (int s = s0; s < stages; s += WK) {
      if (stages > 1) load_a(s);
#pragma unroll
      for (int q = 0; q < 4; q++)
        *reinterpret_cast<i4*>(area + (r0 + 8 * q) * kStage + (piece ^ ((r0 + 8 * q) / 2 & 7)) * 16) = rb[q];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (s + WK < stages) load_b(strip, s + WK);
      else if (strip + step < strips) load_b(strip + step, s0);
      const char* from = area + row * kStage;
#pragma unroll
      for (int q = 0; q < 4; q++)
        acc = mfma(*reinterpret_cast<const i4*>(from + ((2 * q + half) ^ (row / 2 & 7)) * 16), fa[q], acc);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    int32_t* tile = reinterpret_cast<int32_t*>(area);
    put_sums(tile, kTile, acc);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if constexpr (WK > 1) {
      __syncthreads();
      // every thread adds up its elements of the tiles into wave 0's, and wave 0 stores it
      int32_t* sum = reinterpret_cast<int32_t*>(lds[0]);
      for (int e = threadIdx.x; e < 32 * kTile; e += 256) {
        int32_t v = sum[e];
#pragma unroll
        for (int w = 1; w < WK; w++) v += reinterpret_cast<const int32_t*>(lds[w])[e];
        sum[e] = v;
      }
      __syncthreads();
      if (wave == 0) store_tile(sum, kTile, 0, C(strip * 32, p), scale, p);
      __syncthreads();
    } else {
      store_tile(tile, kTile, 0, C(strip * 32, p), scale, p);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// Rows shorter than one piece (16 bytes), or more than 32 rows further apart than 32-bit offsets reach:
// a 16 x 16 tile of the output per workgroup, one thread per element, both operands'
// rows staged 64 bytes at a time.
template <class O>
__global__ __launch_bounds__(256) void product_small_kernel(Product<O> p, int64_t tiles_n, int64_t first_block) {
  __shared__ int8_t sa[16][68], sb[16][68];
  const int tid = threadIdx.x, r = tid / 16, c = tid % 16;
  const int64_t tile = first_block + blockIdx.x, i0 = tile / tiles_n * 16, j0 = tile % tiles_n * 16;
  int32_t acc = 0;
  for (int64_t k0 = 0; k0 < p.k; k0 += 64) {
    for (int u = tid; u < 16 * 64; u += 256) {
      const int64_t row = u / 64, at = k0 + u % 64;
      sa[row][u % 64] = i0 + row < p.m && at < p.k ? p.a[(i0 + row) * p.a_stride + at] : (int8_t)0;
      sb[row][u % 64] = j0 + row < p.n && at < p.k ? p.b[(j0 + row) * p.b_stride + at] : (int8_t)0;
    }
    __syncthreads();
    for (int u = 0; u < 64; u++) acc += (int32_t)sa[r][u] * (int32_t)sb[c][u];
    __syncthreads();
  }
  if (i0 + r < p.m && j0 + c < p.n) {
    float v = ((float)acc * p.a_scales[i0 + r]) * p.b_scales[j0 + c];
    if (p.bias) v = v + p.bias[j0 + c];
    p.out[(i0 + r) * p.out_stride + j0 + c] = (O)v;
  }
}

template <class T>
void quantize(const void* x, int64_t n, int64_t dim, int64_t stride, int8_t* codes, int64_t code_stride, float* scales,
              hipStream_t st) {
  const T* in = static_cast<const T*>(x);
  auto go = [&](auto* kernel, int64_t rows) {
    in_launches((n + rows - 1) / rows, 256, [&](int64_t first, unsigned count) {
      hipLaunchKernelGGL(kernel, dim3(count), dim3(256), 0, st, in, n, dim, stride, codes, code_stride, scales, first);
    });
  };
  const int64_t vectors = (dim + kVec<T> - 1) / kVec<T>;
  if (vectors <= 8) go(quantize_kernel<T, 8, 1, 4>, 128);
  else if (vectors <= 16) go(quantize_kernel<T, 16, 1, 4>, 64);
  else if (vectors <= 32) go(quantize_kernel<T, 32, 1, 4>, 32);
  else if (vectors <= 64) go(quantize_kernel<T, 64, 1, 4>, 16);
  else if (vectors <= 128) go(quantize_kernel<T, 64, 2, 2>, 8);
  else if (vectors <= 256) go(quantize_kernel<T, 64, 4, 1>, 4);
  else if (vectors <= 512) go(quantize_kernel<T, 64, 8, 1>, 4);
  else
    in_launches(n, 256, [&](int64_t first, unsigned count) {
      hipLaunchKernelGGL(quantize_long_kernel<T>, dim3(count), dim3(256), 0, st, in, dim, stride, codes, code_stride,
                         scales, first);
    });
  HIP_OK(hipGetLastError());
}

// More than 64 KB of LDS is asked for once per kernel and device.
template <auto* KERNEL>
void allow_lds(int bytes) {
  static std::atomic<uint64_t> done{0};
  if (bytes <= 65536) return;
  int device = 0;
  HIP_OK(hipGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return;
  HIP_OK(hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
  done.fetch_or(bit, std::memory_order_relaxed);
}

template <int BM, int BN, int WM, int WN, class O>
void launch_tiles(const Product<O>& p, hipStream_t st) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  // down a group of tiles' rows first: as many as keep their rows of a within 2 MB of an XCD's L2, eight at least
  const int64_t group = std::min(tm, std::max<int64_t>(8, (2 << 20) / (BM * p.k)));
  constexpr int lds = 2 * (BM + BN) * kStage + TileScales<BM, BN, 64 * WM * WN>::kBytes;
  constexpr auto* kernel = &product_tile_kernel<BM, BN, WM, WN, O>;
  allow_lds<kernel>(lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(64 * WM * WN), lds, st, p, tm, tn, group);
  HIP_OK(hipGetLastError());
}

template <int BM, int BN, int WM, int WN, int NB, bool MANY, class O>
void launch_deep(const Product<O>& p, hipStream_t st) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  const int64_t group = std::min<int64_t>(tm, 8);
  const int lds = NB * (BM + BN) * 64 + 2 * TileScales<BM, BN, 64 * WM * WN>::kBytes;
  constexpr auto* kernel = &product_deep_kernel<BM, BN, WM, WN, NB, MANY, O>;
  allow_lds<kernel>(lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(MANY ? std::min<int64_t>(tm * tn, 256) : tm * tn)), dim3(64 * WM * WN), lds, st, p, tm, tn, group);
  HIP_OK(hipGetLastError());
}

template <int KS, class O>
void launch_panels(const Product<O>& p, hipStream_t st) {
  const int64_t panels = (p.m + 127) / 128, tiles_n = (p.n + 63) / 64;
  // as many workgroups as run at once, each with a like share of b's tiles
  const int64_t slices = std::min(tiles_n, std::max<int64_t>(1, 256 * (KS == 4 ? 3 : 2) / panels));
  auto* kernel = p.bias ? product_panel_kernel<KS, true, O> : product_panel_kernel<KS, false, O>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(panels * slices)), dim3(256), 0, st, p, panels, tiles_n, slices);
  HIP_OK(hipGetLastError());
}

template <class O>
void product(const Product<O>& p, hipStream_t st) {
  // (the strips' offsets, and all of the output's, have 64 bits)
  if (p.k < 16 || (p.m > 32 && (p.a_stride >= kFar || p.b_stride >= kFar))) {
    const int64_t tm = (p.m + 15) / 16, tn = (p.n + 15) / 16;
    in_launches(tm * tn, 256, [&](int64_t first, unsigned count) {
      hipLaunchKernelGGL(product_small_kernel<O>, dim3(count), dim3(256), 0, st, p, tn, first);
    });
    HIP_OK(hipGetLastError());
  } else if (p.m <= 32) {
    const int64_t strips = (p.n + 31) / 32;
    // a strip's stages over four waves where strips alone are too few (1 x 4,096 x 4,096: 11 us)
    if (strips < 2048 && p.k > kStage) {
      hipLaunchKernelGGL((product_strip_kernel<4, O>), dim3((unsigned)strips), dim3(256), 0, st, p, strips, strips);
    } else {
      const int64_t blocks = std::min<int64_t>((strips + 3) / 4, 256 * 6);
      hipLaunchKernelGGL((product_strip_kernel<1, O>), dim3((unsigned)blocks), dim3(256), 0, st, p, strips, blocks * 4);
    }
    HIP_OK(hipGetLastError());
  } else if (p.k <= 128) {
    launch_panels<4>(p, st);
  } else if (p.k <= 256) {
    launch_panels<8>(p, st);
  } else {
    // By how many tiles there are for the 256 CUs.  Measured to bfloat16, us, with tiles of 256, 128 and 64 straight
    // to LDS and of 128 through registers: 4,096^3: 71, 108, 156, 96; 2,048 x 4,096 x 4,096: 55, 51, 85, 44;
    // 1,024: 51, 24, 41, 31; 512: 49, 20, 19, 28; 64: 46, 18, 13, 27; 4,096 x 4,096 x 1,024: 34, 36, 46, 34;
    // 1,024 x 20,032 x 512: 40, 29, 36, 27; 10,000 x 50,048 x 512: 457, 510, 733, 583.  Tiles of 256 leave CUs without
    // one in the last turn, or rows of tiles empty: of 256 CUs' tiles, 4,096 x 20,032 x 768 fills 98 % in 5 turns: 97,
    // 119, 171, 106; 512 x 100,032 x 768 76 % in 4: 74, 77, 103, 63; 300 x 60,001 x 1,024 54 % in 2: 49, -, -, 42.
    auto tiles = [&](int64_t size) { return (p.m + size - 1) / size * ((p.n + size - 1) / size); };
    const bool direct = (reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) | p.a_stride | p.b_stride) % 16 == 0 &&
                        p.k % 64 == 0;
    const int64_t turns = (tiles(256) + 255) / 256;
    if (direct && (double)p.m * p.n >= 0.8 * 65536 * 256 * turns) launch_deep<256, 256, 2, 2, 4, true>(p, st);
    else if (direct && tiles(64) <= 512) launch_deep<64, 64, 2, 2, 4, false>(p, st);
    else if (direct && tiles(128) <= 256) launch_deep<128, 128, 2, 2, 4, false>(p, st);
    else if (tiles(64) <= 512) launch_tiles<64, 64, 2, 2>(p, st);
    else launch_tiles<128, 128, 2, 2>(p, st);
  }
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
    if (m > INT32_MAX || n > INT32_MAX || (m + 127) / 128 * ((n + 127) / 128) >= 1 << 24)
      qv::fail(QV_EUNSUPPORTED, "more tiles than one launch has");
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto go = [&](auto* o) {
      using O = std::remove_pointer_t<decltype(o)>;
      product(Product<O>{d_a, a_stride, d_a_scales, m, d_b, b_stride, d_b_scales, d_bias, n, k, o, out_stride}, st);
    };
    if (out_type == QV_FLOAT) go(static_cast<float*>(d_out));
    else if (out_type == QV_BFLOAT16) go(static_cast<bf16*>(d_out));
    else go(static_cast<f16*>(d_out));
  });
}

}  // extern "C"
