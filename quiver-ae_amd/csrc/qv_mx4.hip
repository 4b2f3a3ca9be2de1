// qv_mx4.hip -- rows in microscaled 4-bit floating point: to codes and back, and the
// product of two such matrices.
//
// A block of 32 values of a row shares a power of two 2^(s - 127), s one byte (255: the
// block is NaN); a code is a sign and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6; two codes to a
// byte, the lower half first.  A block's 16 bytes of codes are what a lane gives to a
// matrix instruction, which applies the scales itself.
#include <algorithm>

#include "qv_product.hpp"

using namespace qv;
using namespace qv::dev;
using namespace qv::dense;

namespace {

constexpr int kBlock = 32;  // values that share a scale

// ---- rows to 4 bits and back -------------------------------------------------------
//
// Four lanes hold a block, eight values each: its largest magnitude a, compared as a whole
// number, gives the scale, the least power of two of which a is 7 times at most (then no
// value is further than half a step of the codes from its own).  The scaled values are
// exact, and one instruction rounds two of them, halves to even, magnitudes over 6 to 6.
// Bound by memory.

constexpr uint32_t kInfBits = 0x7f800000u;

// Rows and blocks of a workgroup's run of blocks.
struct Places {
  int64_t row;    // of the workgroup's first block
  uint32_t rest;  // its number in the row
  uint32_t per_row, magic;
  __device__ __forceinline__ Places(int64_t first, uint32_t per_row, uint32_t magic)
      : row(first / per_row), rest((uint32_t)(first - row * per_row)), per_row(per_row), magic(magic) {}
  // of the one `u` (< 1024) further on
  __device__ __forceinline__ void at(uint32_t u, int64_t& r, uint32_t& b) const {
    const uint32_t v = rest + u;
    // v / per_row: by its reciprocal where that is exact (v per_row < 2^32), else v is less than twice per_row
    const uint32_t q = per_row == 1 ? v : per_row <= 32768 ? __umulhi(v, magic) : v >= per_row ? 1u : 0u;
    r = row + q;
    b = v - q * per_row;
  }
};

template <class T, int R>
__global__ __launch_bounds__(256) void to_mx4_kernel(const T* __restrict__ x, int64_t blocks, int64_t dim, int64_t stride,
                                                     uint8_t* __restrict__ codes, int64_t code_stride,
                                                     uint8_t* __restrict__ scales, int64_t scale_stride, uint32_t per_row,
                                                     uint32_t magic, int64_t first_group) {
  constexpr int kVecs = 8 / kVec<T>;  // loads of a lane's eight values
  const int quarter = threadIdx.x % 4;
  const int64_t first = (first_group + blockIdx.x) * (64 * R);
  const Places places(first, per_row, magic);
  float v[R][8];
  int64_t row[R];
  uint32_t block[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t u = (uint32_t)min((int64_t)(threadIdx.x / 4 + 64 * r), blocks - 1 - first);
    places.at(u, row[r], block[r]);
    const int64_t j = (int64_t)block[r] * kBlock + quarter * 8;
    const T* from = x + row[r] * stride + j;
#pragma unroll
    for (int e = 0; e < kVecs; e++) load_tail(from + e * kVec<T>, dim - j - e * kVec<T>, 0.f, v[r] + e * kVec<T>);
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[r][i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));
    top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));
    if (first + threadIdx.x / 4 + 64 * r >= blocks) continue;
    // a fraction above 1.75 carries into the exponent; a = 7 2^e has the exponent e + 2
    const int exponent = top >= kInfBits ? 255 : max((int)((top + 0x1fffffu) >> 23) - 2, 0);
    const float inv = __uint_as_float((uint32_t)(254 - exponent) << 23);
    uint32_t word = 0;
    if (exponent != 255) {
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[r][0] * inv, v[r][1] * inv, 1.f, 0);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[r][2] * inv, v[r][3] * inv, 1.f, 1);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[r][4] * inv, v[r][5] * inv, 1.f, 2);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[r][6] * inv, v[r][7] * inv, 1.f, 3);
    }
    const int64_t j = (int64_t)block[r] * kBlock + quarter * 8;
    uint8_t* to = codes + row[r] * code_stride + j / 2;
    if (j + 7 <= dim) {
      __builtin_memcpy(to, &word, 4);
    } else {
#pragma unroll
      for (int i = 0; i < 3; i++)
        if (j + 2 * i < dim) to[i] = (uint8_t)(word >> (8 * i));
    }
    if (quarter == 0) scales[row[r] * scale_stride + block[r]] = (uint8_t)exponent;
  }
}

__device__ __forceinline__ float scale_of(uint32_t s) {
  return s == 255 ? __builtin_nanf("") : __uint_as_float(s ? s << 23 : 1u << 22);
}

template <class T, int R>
__global__ __launch_bounds__(256) void from_mx4_kernel(const uint8_t* __restrict__ codes, int64_t blocks, int64_t dim,
                                                       int64_t code_stride, const uint8_t* __restrict__ scales,
                                                       int64_t scale_stride, T* __restrict__ out, int64_t stride,
                                                       uint32_t per_row, uint32_t magic, int64_t first_group) {
  const int quarter = threadIdx.x % 4;
  const int64_t first = (first_group + blockIdx.x) * (64 * R);
  const Places places(first, per_row, magic);
  uint32_t word[R], scale[R];
  int64_t row[R];
  uint32_t block[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t u = (uint32_t)min((int64_t)(threadIdx.x / 4 + 64 * r), blocks - 1 - first);
    places.at(u, row[r], block[r]);
    const int64_t j = (int64_t)block[r] * kBlock + quarter * 8;
    const uint8_t* from = codes + row[r] * code_stride + j / 2;
    word[r] = 0;
    if (j + 7 <= dim) {
      __builtin_memcpy(&word[r], from, 4);
    } else {
#pragma unroll
      for (int i = 0; i < 3; i++)
        if (j + 2 * i < dim) word[r] |= (uint32_t)from[i] << (8 * i);
    }
    scale[r] = scales[row[r] * scale_stride + block[r]];
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    if (first + threadIdx.x / 4 + 64 * r >= blocks) continue;
    const float s = scale_of(scale[r]);
    union {
      T t[8];
      raw4 raw[8 / kVec<T>];
    } u;
    auto two = [&](int i, auto v) {
      u.t[2 * i] = (T)(v[0] * s);
      u.t[2 * i + 1] = (T)(v[1] * s);
    };
    two(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 0));
    two(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 1));
    two(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 2));
    two(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 3));
    const int64_t j = (int64_t)block[r] * kBlock + quarter * 8;
    T* to = out + row[r] * stride + j;
    if (j + 8 <= dim) {
#pragma unroll
      for (int e = 0; e < 8 / kVec<T>; e++) *reinterpret_cast<raw4_any*>(to + e * kVec<T>) = u.raw[e];
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (j + i < dim) to[i] = u.t[i];
    }
  }
}

// ---- product -------------------------------------------------------------------
//
// Sums on the matrix cores (v_mfma_scale_f32_32x32x64_f8f6f4): the rows of b are the
// instruction's rows and the rows of a its columns, so a lane ends with four
// consecutive columns j of one output row i.  It gives 16 bytes of a row, one block, and
// that block's scale.  The products of two codes and their scales are exact, their sum is
// fp32.
//
// k goes in stages of 128 bytes of each row, eight pieces of 16.  The last piece of
// a row whose length is no multiple of 16 is its last 16 bytes; what it repeats is
// zeroed in a, so every load is a whole one inside the row and b needs no mask.
// Rows past the end repeat the last row; what they give is not stored.

typedef int32_t i8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

template <class O>
struct Product {
  const uint8_t* a;
  int64_t a_stride;
  const uint8_t* a_scales;
  int64_t as_stride, m;
  const uint8_t* b;
  int64_t b_stride;
  const uint8_t* b_scales;
  int64_t bs_stride;
  const float* bias;
  int64_t n, k;  // k: bytes of a row of codes
  int blocks;    // of a row
  O* out;
  int64_t out_stride;
};

// x: an instruction's rows, y: its columns; the scales are byte S of theirs.
template <int S>
__device__ __forceinline__ f16v mfma(i4 x, uint32_t scale_x, i4 y, uint32_t scale_y, f16v acc) {
  const i8v wx = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  const i8v wy = __builtin_shufflevector(y, y, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wx, wy, acc, 4, 4, S, (int)scale_x, S, (int)scale_y);
}

// Scales of the eight blocks from `at` on of a row of `blocks`; 0 past its end.
__device__ __forceinline__ uint64_t eight_scales(const uint8_t* row, int at, int blocks) {
  uint64_t v = 0;
  if (blocks >= 8) {
    const int from = min(at, blocks - 8);
    __builtin_memcpy(&v, row + from, 8);
    return at - from < 8 ? v >> (8 * (at - from)) : 0;
  }
  for (int i = at; i < blocks; i++) v |= (uint64_t)row[i] << (8 * (i - at));
  return v;
}

// 16 bytes of a row of fewer than that, zeros past its end.
__device__ __forceinline__ i4 short_row(const uint8_t* row, int k) {
  i4 v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; i++)
    if (i < k) v[i / 4] |= (int)row[i] << (8 * (i % 4));
  return v;
}

// A tile of BM x BN outputs per workgroup, WM x WN waves of 32 TM x 32 TN each.  Both
// operands' stages go through registers into LDS, the next one in flight while the
// matrix cores work on this one; piece q of row r lies at q ^ (r / 2 mod 8), so that the
// 16 rows that are read at once (64 banks, 256 bytes) lie in 16 different places.  For
// rows of any alignment, length and distance.
template <int BM, int BN, int WM, int WN, bool SHORT, class O>
__global__ __launch_bounds__(64 * WM * WN, 1) void product_tile_kernel(Product<O> p, int64_t tiles_m, int64_t tiles_n,
                                                                       int64_t group, int64_t first_block) {
  constexpr int T = 64 * WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int LA = BM * 8 / T, LB = BN * 8 / T, kRows = T / 8;
  constexpr int LS = (BM + BN + T - 1) / T;
  constexpr int kCodes = (BM + BN) * kStage, kBuffer = kCodes + (BM + BN) * 8;
  __shared__ __align__(16) char lds[2 * kBuffer + BN * 4];
  const int tid = threadIdx.x, wave = wave_id(), lane = lane_id();
  const int wm = wave / WN, wn = wave % WN;
  // tiles in groups of `group` rows of tiles, down the rows first
  const int64_t t = first_block + tile_of_block(blockIdx.x, gridDim.x);
  const int64_t g = t / (group * tiles_n), gm = min(group, tiles_m - g * group), in = t - g * group * tiles_n;
  const int64_t i0 = (g * group + in % gm) * BM, j0 = in / gm * BN;

  const int piece = tid % 8, r0 = tid / 8;
  const uint8_t *a[LA], *b[LB], *sc[LS];
#pragma unroll
  for (int q = 0; q < LA; q++) a[q] = p.a + min(i0 + r0 + q * kRows, p.m - 1) * p.a_stride;
#pragma unroll
  for (int q = 0; q < LB; q++) b[q] = p.b + min(j0 + r0 + q * kRows, p.n - 1) * p.b_stride;
#pragma unroll
  for (int q = 0; q < LS; q++) {
    const int r = min(tid + q * T, BM + BN - 1);
    sc[q] = r < BM ? p.a_scales + min(i0 + r, p.m - 1) * p.as_stride : p.b_scales + min(j0 + r - BM, p.n - 1) * p.bs_stride;
  }
  const int k = (int)p.k, stages = (k + kStage - 1) / kStage;
  i4 ra[LA], rb[LB];
  uint64_t rs[LS];
  auto load = [&](int s) {
    const int place = s * kStage + piece * 16, from = min(place, k - 16);
#pragma unroll
    for (int q = 0; q < LA; q++) {
      if constexpr (SHORT) ra[q] = short_row(a[q], piece == 0 ? k : 0);
      else ra[q] = *reinterpret_cast<const i4_any*>(a[q] + from);
    }
#pragma unroll
    for (int q = 0; q < LB; q++) {
      if constexpr (SHORT) rb[q] = short_row(b[q], piece == 0 ? k : 0);
      else rb[q] = *reinterpret_cast<const i4_any*>(b[q] + from);
    }
#pragma unroll
    for (int q = 0; q < LS; q++) rs[q] = eight_scales(sc[q], s * 8, p.blocks);
  };
  auto keep = [&](int s) {
    char* at = lds + (s & 1) * kBuffer;
    char* to = at + r0 * kStage + (piece ^ (r0 / 2 & 7)) * 16;
    if (!SHORT && (s + 1) * kStage > k) {
      const int over = max(0, s * kStage + piece * 16 - (k - 16));
#pragma unroll
      for (int q = 0; q < LA; q++) ra[q] = without_first(ra[q], over);
    }
#pragma unroll
    for (int q = 0; q < LA; q++) *reinterpret_cast<i4*>(to + q * kRows * kStage) = ra[q];
#pragma unroll
    for (int q = 0; q < LB; q++) *reinterpret_cast<i4*>(to + BM * kStage + q * kRows * kStage) = rb[q];
#pragma unroll
    for (int q = 0; q < LS; q++)
      if (tid + q * T < BM + BN) *reinterpret_cast<uint64_t*>(at + kCodes + (tid + q * T) * 8) = rs[q];
  };
  f16v acc[TM][TN];
#pragma unroll
  for (int x = 0; x < TM; x++)
#pragma unroll
    for (int y = 0; y < TN; y++) acc[x][y] = f16v{};
  const int row = lane % 32, half = lane / 32;
  // step q takes pieces q and 4 + q, so a lane's scales of a stage are four bytes in a row
  i4 fa[2][TM], fb[2][TN];
  uint32_t sa[TM], sb[TN];
  auto read = [&](int s, int q) {
    const char* from = lds + (s & 1) * kBuffer + ((q + 4 * half) ^ (row / 2 & 7)) * 16 + row * kStage;
#pragma unroll
    for (int x = 0; x < TM; x++) fa[q & 1][x] = *reinterpret_cast<const i4*>(from + (wm * TM + x) * 32 * kStage);
#pragma unroll
    for (int y = 0; y < TN; y++)
      fb[q & 1][y] = *reinterpret_cast<const i4*>(from + BM * kStage + (wn * TN + y) * 32 * kStage);
  };
  auto read_scales = [&](int s) {
    const char* from = lds + (s & 1) * kBuffer + kCodes + row * 8 + half * 4;
#pragma unroll
    for (int x = 0; x < TM; x++) sa[x] = *reinterpret_cast<const uint32_t*>(from + (wm * TM + x) * 32 * 8);
#pragma unroll
    for (int y = 0; y < TN; y++) sb[y] = *reinterpret_cast<const uint32_t*>(from + (BM + (wn * TN + y) * 32) * 8);
  };
  auto products = [&](auto step) {
    constexpr int Q = decltype(step)::value;
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y++) acc[x][y] = mfma<Q>(fb[Q & 1][y], sb[y], fa[Q & 1][x], sa[x], acc[x][y]);
  };
  if (stages > 0) {
    load(0);
    keep(0);
  }
  float* add = reinterpret_cast<float*>(lds + 2 * kBuffer);
  for (int r = tid; r < BN; r += T) add[r] = p.bias ? p.bias[min(j0 + r, p.n - 1)] : -0.f;
  __syncthreads();
  for (int s = 0; s < stages; s++) {
    const bool more = s + 1 < stages;
    if (more) load(s + 1);
    read_scales(s);
    read(s, 0);
    read(s, 1);
    __builtin_amdgcn_sched_barrier(0);
    products(std::integral_constant<int, 0>());
    __builtin_amdgcn_sched_barrier(0);
    read(s, 2);
    products(std::integral_constant<int, 1>());
    __builtin_amdgcn_sched_barrier(0);
    read(s, 3);
    products(std::integral_constant<int, 2>());
    __builtin_amdgcn_sched_barrier(0);
    if (more) keep(s + 1);
    products(std::integral_constant<int, 3>());
    __syncthreads();
  }
  const int64_t i = i0 + wm * TM * 32 + row, j = j0 + wn * TN * 32;
  constexpr int R = sizeof(O) == 2 && TN % 2 == 0 ? 2 : 1;
  auto store = [&](auto whole) {
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y += R)
        store_results<decltype(whole)::value, R>(
            [&](int r, int g) {
              const f4 t = *reinterpret_cast<const f4*>(add + wn * TN * 32 + 32 * (y + r) + 8 * g + 4 * half);
              f4 v;
#pragma unroll
              for (int e = 0; e < 4; e++) v[e] = acc[x][y + r][4 * g + e] + t[e];
              return v;
            },
            i + 32 * x, j + 32 * y, p.m, p.n, p.out, p.out_stride);
  };
  if (i0 + BM <= p.m && j0 + BN <= p.n) store(std::true_type());
  else store(std::false_type());
}

template <class F>
void in_runs(int64_t n, int64_t dim, int64_t run, F f) {
  const uint32_t per_row = (uint32_t)((dim + kBlock - 1) / kBlock);
  const uint32_t magic = (uint32_t)(((uint64_t{1} << 32) + per_row - 1) / per_row);
  const int64_t blocks = n * per_row;
  in_launches((blocks + run - 1) / run, 256, [&](int64_t first, unsigned count) { f(blocks, per_row, magic, first, count); });
  HIP_OK(hipGetLastError());
}

template <class T>
void to_mx4(const void* x, int64_t n, int64_t dim, int64_t stride, uint8_t* codes, int64_t code_stride, uint8_t* scales,
            int64_t scale_stride, hipStream_t st) {
  constexpr int R = 4;
  in_runs(n, dim, 64 * R, [&](int64_t blocks, uint32_t per_row, uint32_t magic, int64_t first, unsigned count) {
    hipLaunchKernelGGL((to_mx4_kernel<T, R>), dim3(count), dim3(256), 0, st, static_cast<const T*>(x), blocks, dim, stride,
                       codes, code_stride, scales, scale_stride, per_row, magic, first);
  });
}

template <class T>
void from_mx4(const uint8_t* codes, int64_t n, int64_t dim, int64_t code_stride, const uint8_t* scales, int64_t scale_stride,
              void* out, int64_t stride, hipStream_t st) {
  constexpr int R = 4;
  in_runs(n, dim, 64 * R, [&](int64_t blocks, uint32_t per_row, uint32_t magic, int64_t first, unsigned count) {
    hipLaunchKernelGGL((from_mx4_kernel<T, R>), dim3(count), dim3(256), 0, st, codes, blocks, dim, code_stride, scales,
                       scale_stride, static_cast<T*>(out), stride, per_row, magic, first);
  });
}

template <int BM, int BN, int WM, int WN, bool SHORT, class O>
void launch_tiles(const Product<O>& p, hipStream_t st) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  // down a group of tiles' rows first: as many as keep their rows of a within 2 MB of an XCD's L2, eight at least
  const int64_t group = std::min(tm, std::max<int64_t>(8, (2 << 20) / (BM * std::max<int64_t>(p.k, 16))));
  in_launches(tm * tn, 64 * WM * WN, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL((product_tile_kernel<BM, BN, WM, WN, SHORT, O>), dim3(count), dim3(64 * WM * WN), 0, st, p, tm, tn,
                       group, first);
  });
  HIP_OK(hipGetLastError());
}

template <class O>
void product(const Product<O>& p, hipStream_t st) {
  if (p.k < 16) launch_tiles<64, 64, 2, 2, true>(p, st);
  else launch_tiles<64, 64, 2, 2, false>(p, st);
}

// Codes and scales of n rows of dim values.
void check_rows(const char* codes_name, const char* scales_name, const void* codes, int64_t code_stride, const void* scales,
                int64_t scale_stride, int64_t n, int64_t dim) {
  check_matrix(codes_name, codes, n, dim / 2 + dim % 2, code_stride, 1);
  check_matrix(scales_name, scales, n, dim / kBlock + (dim % kBlock != 0), scale_stride, 1);
}

}  // namespace

extern "C" {

int qv_quantize_rows_mx4(const void* d_x, int32_t type, int64_t n, int64_t dim, int64_t x_stride, uint8_t* d_codes,
                         int64_t code_stride, uint8_t* d_scales, int64_t scale_stride, int device, void* stream) {
  return qv::guard([&] {
    check_matrix("x", d_x, n, dim, x_stride, value_size(type));
    check_rows("codes", "scales", d_codes, code_stride, d_scales, scale_stride, n, dim);
    if (n > INT32_MAX || dim > INT32_MAX) qv::fail(QV_EUNSUPPORTED, "more than 2^31 - 1 rows or columns");
    if (n == 0 || dim == 0) return;
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (type == QV_FLOAT) to_mx4<float>(d_x, n, dim, x_stride, d_codes, code_stride, d_scales, scale_stride, st);
    else if (type == QV_BFLOAT16) to_mx4<bf16>(d_x, n, dim, x_stride, d_codes, code_stride, d_scales, scale_stride, st);
    else to_mx4<f16>(d_x, n, dim, x_stride, d_codes, code_stride, d_scales, scale_stride, st);
  });
}

int qv_mx4_values(const uint8_t* d_codes, int64_t code_stride, const uint8_t* d_scales, int64_t scale_stride, int64_t n,
                  int64_t dim, void* d_out, int32_t out_type, int64_t out_stride, int device, void* stream) {
  return qv::guard([&] {
    check_matrix("out", d_out, n, dim, out_stride, value_size(out_type));
    check_rows("codes", "scales", d_codes, code_stride, d_scales, scale_stride, n, dim);
    if (n > INT32_MAX || dim > INT32_MAX) qv::fail(QV_EUNSUPPORTED, "more than 2^31 - 1 rows or columns");
    if (n == 0 || dim == 0) return;
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (out_type == QV_FLOAT) from_mx4<float>(d_codes, n, dim, code_stride, d_scales, scale_stride, d_out, out_stride, st);
    else if (out_type == QV_BFLOAT16) from_mx4<bf16>(d_codes, n, dim, code_stride, d_scales, scale_stride, d_out, out_stride, st);
    else from_mx4<f16>(d_codes, n, dim, code_stride, d_scales, scale_stride, d_out, out_stride, st);
  });
}

int qv_mx4_product(const uint8_t* d_a, int64_t a_stride, const uint8_t* d_a_scales, int64_t a_scale_stride, int64_t m,
                   const uint8_t* d_b, int64_t b_stride, const uint8_t* d_b_scales, int64_t b_scale_stride,
                   const float* d_bias, int64_t n, int64_t k, void* d_out, int32_t out_type, int64_t out_stride, int device,
                   void* stream) {
  return qv::guard([&] {
    if (m < 0 || n < 0 || k < 0) qv::fail(QV_EINVAL, "negative size");
    if (k % 2) qv::fail(QV_EINVAL, "k must be even: a row of an odd length ends with a zero code");
    const int size = value_size(out_type);
    if (m == 0 || n == 0) return;
    check_rows("a", "a_scales", d_a, a_stride, d_a_scales, a_scale_stride, m, k);
    check_rows("b", "b_scales", d_b, b_stride, d_b_scales, b_scale_stride, n, k);
    check_matrix("out", d_out, m, n, out_stride, size);
    if (d_bias) check_vector("bias", d_bias, n);
    if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX) qv::fail(QV_EUNSUPPORTED, "more than 2^31 - 1 rows or columns");
    const OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto go = [&](auto* o) {
      using O = std::remove_pointer_t<decltype(o)>;
      product(Product<O>{d_a, a_stride, d_a_scales, a_scale_stride, m, d_b, b_stride, d_b_scales, b_scale_stride, d_bias, n,
                         k / 2, (int)((k + kBlock - 1) / kBlock), o, out_stride},
              st);
    };
    if (out_type == QV_FLOAT) go(static_cast<float*>(d_out));
    else if (out_type == QV_BFLOAT16) go(static_cast<bf16*>(d_out));
    else go(static_cast<f16*>(d_out));
  });
}

}  // extern "C"
