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
// Bound by memory: 1M x 128 floats 104 to 109 us, 5.3 TB/s; 1M x 128 of 16 bits 63, 100,000 x 769 43.

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
    const T* from = x + row[r] * stride;
#pragma unroll
    for (int e = 0; e < kVecs; e++) {
      if (sizeof(T) == 2 && dim >= kVec<T>) load_near_end(from, j + e * kVec<T>, dim, v[r] + e * kVec<T>);
      else load_tail(from + j + e * kVec<T>, dim - j - e * kVec<T>, 0.f, v[r] + e * kVec<T>);
    }
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

// Back again, a lane writes 16 bytes of a row: 1M x 128 to float 81 us call after call, 7.2 TB/s, into one result
// or three in turn; behind the calls that make the codes 93 (lanes of 32 bytes, in two stores, and through the L2: 149).
template <class T, int R>
__global__ __launch_bounds__(256) void from_mx4_kernel(const uint8_t* __restrict__ codes, int64_t blocks, int64_t dim,
                                                       int64_t code_stride, const uint8_t* __restrict__ scales,
                                                       int64_t scale_stride, T* __restrict__ out, int64_t stride,
                                                       uint32_t per_row, uint32_t magic, int64_t first_group, bool stream) {
  constexpr int V = kVec<T>, kLanes = kBlock / V, kBlocks = 256 / kLanes;  // values of a lane, lanes of a block
  const int part = threadIdx.x % kLanes, number = threadIdx.x / kLanes;
  const int64_t first = (first_group + blockIdx.x) * (kBlocks * R);
  const Places places(first, per_row, magic);
  uint32_t word[R], scale[R];
  int64_t row[R];
  uint32_t block[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t u = (uint32_t)min((int64_t)(number + kBlocks * r), blocks - 1 - first);
    places.at(u, row[r], block[r]);
    const int64_t j = (int64_t)block[r] * kBlock + part * V;
    const uint8_t* from = codes + row[r] * code_stride + j / 2;
    word[r] = 0;
    if (j + V - 1 <= dim) {
      __builtin_memcpy(&word[r], from, V / 2);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2 - 1; i++)
        if (j + 2 * i < dim) word[r] |= (uint32_t)from[i] << (8 * i);
    }
    scale[r] = scales[row[r] * scale_stride + block[r]];
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    if (first + number + kBlocks * r >= blocks) continue;
    const float s = scale_of(scale[r]);
    union {
      T t[V];
      raw4 raw;
    } u;
    auto two = [&](int i, auto v) {
      u.t[2 * i] = (T)(v[0] * s);
      u.t[2 * i + 1] = (T)(v[1] * s);
    };
    two(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 0));
    two(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 1));
    if constexpr (V == 8) {
      two(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 2));
      two(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[r], 1.f, 3));
    }
    const int64_t j = (int64_t)block[r] * kBlock + part * V;
    T* to = out + row[r] * stride + j;
    if (j + V <= dim) {
      store_past(u.raw, reinterpret_cast<raw4_any*>(to), stream);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++)
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

constexpr int64_t kFar = 1 << 24;  // row strides from here on: 256 rows' offsets may pass 32 bits

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
  bool stream, stream_lines;  // results past the caches: where rows are whole lines, through lines
};

// x: an instruction's rows, y: its columns; the scales are byte S of theirs.
template <int S>
__device__ __forceinline__ f16v mfma(i4 x, uint32_t scale_x, i4 y, uint32_t scale_y, f16v acc) {
  const i8v wx = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  const i8v wy = __builtin_shufflevector(y, y, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wx, wy, acc, 4, 4, S, (int)scale_x, S, (int)scale_y);
}

// The same of 16 rows, 16 columns and four blocks of each; the scales are their lowest bytes.
__device__ __forceinline__ f4 mfma16(i4 x, uint32_t scale_x, i4 y, uint32_t scale_y, f4 acc) {
  const i8v wx = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  const i8v wy = __builtin_shufflevector(y, y, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wx, wy, acc, 4, 4, 0, (int)scale_x, 0, (int)scale_y);
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

// Stores a wave's results, from row i and column j of the BM x BN tile at (i0, j0) on; `bias`: the tile's columns', in LDS
// (-0, which changes no sum, without).
template <int BM, int BN, int TM, int TN, class O>
__device__ __forceinline__ void store_tile(f16v (&acc)[TM][TN], int i, int j, int64_t i0, int64_t j0, const float* bias,
                                           const Product<O>& p) {
  constexpr int R = sizeof(O) == 2 && TN % 2 == 0 ? 2 : 1;
  const int row = lane_id() % 32, half = lane_id() / 32;
  auto store = [&](auto whole, auto stream) {
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y += R) {
#pragma unroll
        for (int r = 0; r < R; r++) asm volatile("" : "+a"(acc[x][y + r]) : : "memory");  // in turn: none leaves its accumulators before
        store_results<decltype(whole)::value, decltype(stream)::value, R>(
            [&](int r, int g) {
              const f4 t = *reinterpret_cast<const f4*>(bias + j + 32 * (y + r) + 8 * g + 4 * half);
              f4 v;
#pragma unroll
              for (int e = 0; e < 4; e++) v[e] = acc[x][y + r][4 * g + e] + t[e];
              return v;
            },
            i0 + i + 32 * x + row, j0 + j + 32 * y, p.m, p.n, p.out, p.out_stride);
      }
  };
  if (i0 + BM > p.m || j0 + BN > p.n) store(std::false_type(), std::false_type());
  else if (p.stream) store(std::true_type(), std::true_type());
  else store(std::true_type(), std::false_type());
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
  store_tile<BM, BN, TM, TN>(acc, wm * TM * 32, wn * TN * 32, i0, j0, add, p);
}

// The same tiles where the matrix cores are what bounds the product: stages of 64 bytes
// of k go straight from memory to LDS (no registers, no LDS writes to issue), NB of
// them at a time, so NB - 1 are on their way while one is used.  A stage is two steps
// of 32 bytes; the second step's operands are read while the first one's products run,
// and the next stage's first operands while the second one's do, so the one barrier
// per stage, between the two, finds the operands of what follows it in registers.
// Needs 16-byte aligned rows, scales' rows of whole aligned words, k a multiple of 64.
// G: a load brings a row's scales of G stages, 16 bytes for four (k a multiple of 256 and rows
// of scales 16-byte aligned; then a group's stages are unrolled, with places that are
// constants), else a word of each, which fetches its line again for the next one where rows
// are long (4,096^3: 57 us, and 49 before the groups' stages were unrolled).
// MANY: one workgroup per CU walks over tiles, and the stages run on from tile to tile:
// the next tile's first ones are on their way, and its first operands in registers, while
// the results are stored.
// 4,096^3 to bfloat16: 42 us, 3.3 PFLOP/s, of zeros 36 (a library's 4-bit product with block scales: 70); 8,192^3: 277 us,
// 4.0 PFLOP/s, of zeros 218 (library: 359).  The matrix instruction alone runs at 6.5 PFLOP/s on varied codes, 8.9 on
// zeros: LDS (98 KB a stage, 784 of the 1,024 cycles of its products) and power hold it.
template <int BM, int BN, int WM, int WN, int NB, int G, bool MANY, class O>
__global__ __launch_bounds__(64 * WM * WN, 1) void product_deep_kernel(Product<O> p, int64_t tiles_m, int64_t tiles_n,
                                                                       int64_t group) {
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32, kRow = 64, kWaves = WM * WN;
  constexpr int I = (BM + BN) / 16 / kWaves;                               // loads of 16 rows per wave and stage
  constexpr int S = (BM + BN + kWave * kWaves - 1) / (kWave * kWaves);     // loads of 64 rows' scales
  constexpr int SE = G == 1 ? S : 0;  // of which every stage has as many (the waits count these only)
  static_assert(I % 2 == 0, "issued in halves");
  constexpr int kBuffer = (BM + BN) * kRow;
  constexpr int kScales = (BM + BN) * 4 * G, kSlots = G == 1 ? NB : 2;  // scales of G stages
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
  // a wave loads rows of one operand only: 16 I of them from `first`, and scales of 64 S from `first_scales`
  static_assert(BM == BN && kWaves == 4, "two waves for each operand");
  const int first = wave % 2 * 16 * I, first_scales = wave * S * kWave % BM;
  const bool of_a = wave < 2, scales_of_a = wave * S * kWave % (BM + BN) < BM;
  struct Tile {  // where its rows begin, and the lanes' rows from there
    const uint8_t *rows, *scales;
    uint32_t row[I], scale[S];
  } next;
  const uint8_t *rows_at[2], *scales_at_row;  // of the two halves of a stage's loads
  uint32_t row_at[I], scale_at[S];
  char* scales_at = lds + NB * kBuffer;
  char* bias_at = scales_at + kSlots * kScales;  // of three tiles in turn: other waves may still store the last one
  // the next tile's rows, and its biases on their way
  auto find_next = [&](int slot) {
    const int64_t begin = of_a ? next_i0 : next_j0, scales_begin = scales_of_a ? next_i0 : next_j0;
    const int64_t stride = of_a ? p.a_stride : p.b_stride, scales_stride = scales_of_a ? p.as_stride : p.bs_stride;
    const int most = (int)min((of_a ? p.m : p.n) - 1 - begin, (int64_t)BM - 1);
    const int scales_most = (int)min((scales_of_a ? p.m : p.n) - 1 - scales_begin, (int64_t)BM - 1);
    next.rows = (of_a ? p.a : p.b) + begin * stride;
    next.scales = (scales_of_a ? p.a_scales : p.b_scales) + scales_begin * scales_stride;
#pragma unroll
    for (int q = 0; q < I; q++) next.row[q] = (uint32_t)min(first + q * 16 + lane / 4, most) * (uint32_t)stride + piece * 16;
#pragma unroll
    for (int q = 0; q < S; q++) next.scale[q] = (uint32_t)min(first_scales + q * kWave + lane, scales_most) * (uint32_t)scales_stride;
    if (p.bias) {
      float* to = reinterpret_cast<float*>(bias_at) + slot * BN;
      const int bias_most = (int)min(p.n - 1 - next_j0, (int64_t)BN - 1);
      for (int r = wave * kWave; r < BN; r += kWave * kWaves)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p.bias + next_j0 + min(r + lane, bias_most)),
                                         (__attribute__((address_space(3))) void*)(to + r), 4, 0, 0);
    }
  };
  auto turn_to_next = [&](bool yes) {
    rows_at[0] = yes ? next.rows : rows_at[0];
    rows_at[1] = yes ? next.rows : rows_at[1];
    scales_at_row = yes ? next.scales : scales_at_row;
#pragma unroll
    for (int q = 0; q < I; q++) row_at[q] = yes ? next.row[q] : row_at[q];
#pragma unroll
    for (int q = 0; q < S; q++) scale_at[q] = yes ? next.scale[q] : scale_at[q];
  };
  // a half of a stage's loads, the scales of it and the next G - 1 with the first one (with one tile, stages past the last
  // one repeat it: as many loads as the waits count)
  auto issue = [&](uint32_t s, int part) {
    if (part == 0 && s % G == 0) {
      char* to = scales_at + s / G % kSlots * kScales;
      const uint8_t* from = scales_at_row + (MANY ? 0 : min(s, stages - G) * 4);
#pragma unroll
      for (int q = 0; q < S; q++) {
        const auto there = (__attribute__((address_space(3))) void*)(to + (wave * S + q) * kWave % (BM + BN) * 4 * G);
        if constexpr (G == 1) __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + scale_at[q]), there, 4, 0, 0);
        else __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + scale_at[q]), there, 16, 0, 0);
      }
      if (MANY) scales_at_row += 4 * G;
    }
    char* to = lds + s % NB * kBuffer + wave * I * 1024;
    const uint8_t* from = rows_at[part] + (MANY ? 0 : min(s, stages - 1) * kRow);
#pragma unroll
    for (int q = part * I / 2; q < (part + 1) * I / 2; q++)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + row_at[q]),
                                       (__attribute__((address_space(3))) void*)(to + q * 1024), 16, 0, 0);
    if (MANY) rows_at[part] += kRow;
  };
  f16v acc[TM][TN];
  const int row = lane % 32, half = lane / 32;
  // step q takes pieces q and 2 + q, so a lane's scales of a stage are two bytes in a row of the four
  i4 fa[2][TM], fb[2][TN];
  uint32_t sa[TM], sb[TN], next_sa[TM], next_sb[TN];
  auto read = [&](uint32_t s, int q) {
    const char* from = lds + s % NB * kBuffer + ((q + 2 * half) ^ (row / 4 % 4)) * 16 + row * kRow;
#pragma unroll
    for (int x = 0; x < TM; x++) fa[q][x] = *reinterpret_cast<const i4*>(from + (wm * TM + x) * 32 * kRow);
#pragma unroll
    for (int y = 0; y < TN; y++) fb[q][y] = *reinterpret_cast<const i4*>(from + (BM + (wn * TN + y) * 32) * kRow);
  };
  auto read_scales = [&](uint32_t s) {
    const char* from = scales_at + s / G % kSlots * kScales + row * 4 * G + s % G * 4;
#pragma unroll
    for (int x = 0; x < TM; x++) next_sa[x] = *reinterpret_cast<const uint32_t*>(from + (wm * TM + x) * 32 * 4 * G);
#pragma unroll
    for (int y = 0; y < TN; y++) next_sb[y] = *reinterpret_cast<const uint32_t*>(from + (BM + (wn * TN + y) * 32) * 4 * G);
  };
  auto turn_scales = [&] {
#pragma unroll
    for (int x = 0; x < TM; x++) sa[x] = next_sa[x] >> (16 * half);
#pragma unroll
    for (int y = 0; y < TN; y++) sb[y] = next_sb[y] >> (16 * half);
  };
  auto products = [&](auto step) {
    constexpr int Q = decltype(step)::value;
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y++) acc[x][y] = mfma<Q>(fb[Q][y], sb[y], fa[Q][x], sa[x], acc[x][y]);
  };
  auto meet = [] {  // nothing of a stage moves over it
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  if (!p.bias)
    for (int r = threadIdx.x; r < 3 * BN; r += kWave * kWaves) reinterpret_cast<float*>(bias_at)[r] = -0.f;
  uint32_t turn = blockIdx.x, slot = 0;
  place_next(turn);
  find_next(0);
  rows_at[0] = rows_at[1] = scales_at_row = nullptr;
  turn_to_next(true);
#pragma unroll
  for (int s = 0; s < NB; s++) {
    issue(s, 0);
    if (s + 1 < NB) issue(s, 1);
  }
  __builtin_amdgcn_s_waitcnt(kWaitFor<(NB - 2) * (I + SE) + I / 2 + SE>);
  meet();
  read(0, 0);
  read_scales(0);
  __builtin_amdgcn_s_waitcnt(kReadsDone);
  // stage s, `last` of its tile of which loads are still to be asked for
  auto one_stage = [&](uint32_t s, bool last) {
    turn_scales();
    read(s, 1);
    issue(s + NB - 1, 1);
    products(std::integral_constant<int, 0>());
    between<TM + TN, kDsRead, 1>();
    between<I / 2, kVmem, 2>();
    __builtin_amdgcn_sched_barrier(0);
    // stage s + 1 is there and every wave has read stage s
    __builtin_amdgcn_s_waitcnt(kWaitFor<(NB - 2) * (I + SE)>);
    meet();
    if (MANY) turn_to_next(last);
    read(s + 1, 0);
    read_scales(s + 1);
    issue(s + NB, 0);
    products(std::integral_constant<int, 1>());
    between<TM + TN, kDsRead, 1>();
    between<I / 2, kVmem, 1>();
    __builtin_amdgcn_s_waitcnt(kReadsDone);  // long since: said for the compiler, which else waits at the loop's top
    __builtin_amdgcn_sched_barrier(0);
  };
  uint32_t turns = 0;  // groups of G stages so far
  do {
    i0 = next_i0;
    j0 = next_j0;
    turn += gridDim.x;
    if (MANY) {  // (after the last tile some tile's first stages, which nobody reads)
      place_next(min(turn, tiles - 1));
      find_next(slot == 2 ? 0 : slot + 1);
    }
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y++) {
        acc[x][y] = f16v{};
        asm volatile("" : "+a"(acc[x][y]));
      }
    uint32_t left = stages;
    do {
      static_assert(G == 1 || G == 4 && NB == 4, "the stages of a group have places of their own");
#pragma unroll
      for (int i = 0; i < G; i++) one_stage(turns * G + i, i == 0 && left == NB);
      turns++;
      left -= G;
    } while (left > 0);
    store_tile<BM, BN, TM, TN>(acc, wm * TM * 32, wn * TN * 32, i0, j0, reinterpret_cast<float*>(bias_at) + slot * BN, p);
    slot = slot == 2 ? 0 : slot + 1;
  } while (MANY && turn < tiles);
  __builtin_amdgcn_s_waitcnt(kWaitFor<0>);  // no load into LDS outlives the wave
}

// U strips of 16 rows of b: which of its 16 U rows strip u's are, so that a lane's 4 U results are of columns in a row.
template <int U>
__device__ __forceinline__ int strip_row(int u, int row) {
  return row / 4 * (4 * U) + u * 4 + row % 4;
}

// The biases of a lane's columns, from j on; -0, which changes no sum, without.
template <int U, class O>
__device__ __forceinline__ void load_biases(f4 (&add)[U], int64_t j, const Product<O>& p) {
#pragma unroll
  for (int u = 0; u < U; u++, j += 4) {
    add[u] = f4{-0.f, -0.f, -0.f, -0.f};
    if (!p.bias) continue;
    if (j + 4 <= p.n) {
      add[u] = *reinterpret_cast<const f4_any*>(p.bias + j);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) add[u][e] = p.bias[min(j + e, p.n - 1)];
    }
  }
}

// Stores a lane's columns, from j on of row i, where they lie in the output.  32 bytes of them: lanes of two rows exchange
// halves first, and each store writes 128 bytes in a row of eight rows.
template <int U, class O>
__device__ __forceinline__ void store_columns(f4 (&v)[U], const f4 (&add)[U], int64_t i, int64_t j, const Product<O>& p) {
  constexpr int N = 4 * U, V = kVec<O>;
  constexpr bool kTwo = N == 2 * V;
#pragma unroll
  for (int u = 0; u < U; u++) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[u][e] += add[u][e];
    asm volatile("" : "+v"(v[u]));  // here: a matrix instruction that the compiler moves behind the branch has not all lanes' scales
  }
  O o[N];
#pragma unroll
  for (int e = 0; e < N; e++) o[e] = (O)v[e / 4][e % 4];
  raw4 own[2] = {}, other[2] = {};
  if constexpr (kTwo) {
    __builtin_memcpy(own, o, sizeof(o));
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) other[u][e] = (uint32_t)__builtin_amdgcn_mov_dpp((int)own[u][e], 0xB1, 0xF, 0xF, true);
  }
  if (j + N <= p.n) {
    if constexpr (kTwo) {
      const bool odd = i & 1;
      O* to = p.out + (i - odd) * p.out_stride + j + (odd ? V : 0);
      if (i - odd < p.m) store_past(odd ? other[1] : own[0], reinterpret_cast<raw4_any*>(to), p.stream);
      if (i - odd + 1 < p.m) store_past(odd ? own[1] : other[0], reinterpret_cast<raw4_any*>(to + p.out_stride), p.stream);
    } else if (i < p.m) {
      O* to = p.out + i * p.out_stride + j;
      if constexpr (N == V) store_past(__builtin_bit_cast(raw4, o), reinterpret_cast<raw4_any*>(to), p.stream);
      else __builtin_memcpy(to, o, sizeof(o));
    }
  } else if (i < p.m) {
    O* to = p.out + i * p.out_stride + j;
#pragma unroll
    for (int e = 0; e < N - 1; e++)
      if (j + e < p.n) to[e] = o[e];
  }
}

// Short rows of b, of up to four blocks for each of K matrix instructions, stay in a wave's registers: U strips of 16 of them
// (v_mfma_scale_f32_16x16x128_f8f6f4: what 64 lanes load of 16 rows of 128 values is 1 KB in a row), with their biases, while 16 TM
// rows of a at a time go by, the next ones on their way.  Bound by reading b and writing: 1 x 1M x 128 to float 12.5 us, 5.8
// TB/s (with biases that each are asked for when their result is there: 19); 32 x 900,000 x 128 28 us, 6.3 TB/s (with stores of 64
// bytes in a row through the L2: 62); 64 x 600,000 x 128 to 16 bits 21 us (with 64 bytes in a row: 25).
template <int U, int TM, int K, class O>
__global__ __launch_bounds__(256) void product_row_kernel(Product<O> p, int64_t groups, int64_t first_block, int64_t rows) {
  const int lane = lane_id(), row = lane % 16, quarter = lane / 16;
  const int64_t group = (first_block + blockIdx.x) * 4 + wave_id();
  if (group >= groups) return;
  const int k = (int)p.k;
  int at[K], over[K], block[K];  // of a lane's piece of each step: where it begins, what is of the one before, its block
#pragma unroll
  for (int q = 0; q < K; q++) {
    const int place = q * 64 + quarter * 16;
    at[q] = min(place, k - 16);
    over[q] = place - at[q];
    block[q] = min(q * 4 + quarter, p.blocks - 1);
  }
  i4 fa[TM][K], fb[U][K];
  uint32_t sa[TM][K], sb[U][K];
  const int64_t j0 = group * (16 * U);
  f4 add[U];  // asked for with the rows
  load_biases<U>(add, j0 + quarter * (4 * U), p);
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int64_t j = min(j0 + strip_row<U>(u, row), p.n - 1);
#pragma unroll
    for (int q = 0; q < K; q++) {
      fb[u][q] = *reinterpret_cast<const i4_any*>(p.b + j * p.b_stride + at[q]);
      sb[u][q] = p.b_scales[j * p.bs_stride + block[q]];
    }
  }
  int64_t i0 = blockIdx.y * rows;
  const int64_t end = min(p.m, i0 + rows);
  auto load = [&] {
#pragma unroll
    for (int x = 0; x < TM; x++) {
      const int64_t i = min(i0 + 16 * x + row, p.m - 1);
#pragma unroll
      for (int q = 0; q < K; q++) {
        fa[x][q] = *reinterpret_cast<const i4_any*>(p.a + i * p.a_stride + at[q]);
        sa[x][q] = p.a_scales[i * p.as_stride + block[q]];
      }
    }
  };
  load();
  for (;;) {
    i4 a[TM][K];
    uint32_t scale[TM][K];
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int q = 0; q < K; q++) {
        a[x][q] = without_first(fa[x][q], over[q]);
        scale[x][q] = sa[x][q];
      }
    const int64_t here = i0;
    i0 += 16 * TM;
    if (i0 < end) load();
#pragma unroll
    for (int x = 0; x < TM; x++) {
      f4 v[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        v[u] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < K; q++) v[u] = mfma16(fb[u][q], sb[u][q], a[x][q], scale[x][q], v[u]);
      }
      store_columns<U>(v, add, here + 16 * x + row, j0 + quarter * (4 * U), p);
    }
    if (i0 >= end) return;
  }
}

// Few longer rows, up to 16 TM: b goes to the registers one turn ahead, U strips of V = 4 / U steps of four blocks.  A lane loads one word of scales, those of
// one row and step; two exchanges between the quarters of the wave give every lane the word of each.  a and its scales
// lie in LDS in the order of the lanes.  WK > 1: a strip's blocks are cut over the workgroup's WK waves.
template <int U, int TM, int WK, class O>
__global__ __launch_bounds__(WK == 1 ? 256 : 64 * WK) void product_strip_kernel(Product<O> p, int64_t groups) {
  constexpr int V = 4 / U, kWaves = WK == 1 ? 4 : WK;
  extern __shared__ __align__(16) char lds[];
  const int wave = wave_id(), lane = lane_id(), row = lane % 16, quarter = lane / 16;
  const int k = (int)p.k, blocks = p.blocks, steps = (blocks + 3) / 4, turns = (steps + V - 1) / V;
  const int64_t step = (int64_t)gridDim.x * (WK == 1 ? 4 : 1);
  int64_t group = WK == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  const int first = WK == 1 ? 0 : wave;
  const int64_t scales_end = (p.n - 1) * p.bs_stride + blocks;

  i4 next_b[U][V];
  uint32_t next_scales = 0;
  auto load = [&](int64_t group, int turn) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint8_t* from = p.b + min(group * (16 * U) + strip_row<U>(u, row), p.n - 1) * p.b_stride;
#pragma unroll
      for (int v = 0; v < V; v++)
        next_b[u][v] = *reinterpret_cast<const i4_any*>(from + min(((turn * V + v) * 4 + quarter) * 16, k - 16));
    }
    // the word of this row and step; bytes past the row's end are 0
    const int block = (turn * V + quarter % V) * 4;
    const int64_t at = min(group * (16 * U) + strip_row<U>(quarter / V, row), p.n - 1) * p.bs_stride + min(block, blocks - 1);
    const int64_t from = min(at, scales_end - 4);
    uint32_t word;
    __builtin_memcpy(&word, p.b_scales + from, 4);
    const int valid = blocks - block;
    next_scales = valid <= 0 ? 0 : word >> (8 * (int)(at - from)) & (valid >= 4 ? ~0u : (1u << 8 * valid) - 1);
  };
  if (group < groups && first < turns) load(group, first);

  // a in LDS: piece q of step s and tile x at ((s TM + x) 64 + 16 q + row) 16, its scale behind them
  char* sa = lds + steps * TM * 1024;
  const int pieces = (int)p.m * steps * 4;
  for (int e = threadIdx.x; e < pieces; e += 4 * 64 * kWaves) {
    i4 v[4];
    int at[4];
    char scale[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int n = min(e + q * 64 * kWaves, pieces - 1);
      const int i = n / (steps * 4), block = n - i * (steps * 4), place = block * 16, from = min(place, k - 16);
      at[q] = (block / 4 * TM + i / 16) * 64 + block % 4 * 16 + i % 16;
      v[q] = without_first(*reinterpret_cast<const i4_any*>(p.a + i * p.a_stride + from), place - from);
      scale[q] = block < blocks ? (char)p.a_scales[i * p.as_stride + min(block, blocks - 1)] : 0;
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {
      *reinterpret_cast<i4*>(lds + at[q] * 16) = v[q];
      sa[at[q]] = scale[q];
    }
  }
  __syncthreads();

  for (; group < groups; group += step) {
    f4 acc[TM][U], add[U];
    load_biases<U>(add, group * (16 * U) + quarter * (4 * U), p);
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int u = 0; u < U; u++) acc[x][u] = f4{0.f, 0.f, 0.f, 0.f};
    for (int turn = first; turn < turns; turn += WK) {
      i4 b[U][V];
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < V; v++) b[u][v] = next_b[u][v];
      const uint32_t word = next_scales;
      if (turn + WK < turns) load(group, turn + WK);
      else if (group + step < groups) load(group + step, first);
      // words[q]: that of quarter q's rows, in every lane
      uint32_t words[4];
      {
        const auto h = __builtin_amdgcn_permlane32_swap(word, word, false, false);
        const auto lo = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
        words[0] = lo[0], words[1] = lo[1], words[2] = hi[0], words[3] = hi[1];
      }
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int s = turn * V + v;
        if (V > 1 && s >= steps) break;
#pragma unroll
        for (int x = 0; x < TM; x++) {
          const i4 a = *reinterpret_cast<const i4*>(lds + ((s * TM + x) * 64 + lane) * 16);
          const uint32_t scale = *reinterpret_cast<const uint8_t*>(sa + (s * TM + x) * 64 + lane);
#pragma unroll
          for (int u = 0; u < U; u++) acc[x][u] = mfma16(b[u][v], words[u * V + v] >> (8 * quarter), a, scale, acc[x][u]);
        }
      }
    }
    if constexpr (WK > 1) {
      f4* parts = reinterpret_cast<f4*>(lds + steps * TM * 1088);
#pragma unroll
      for (int x = 0; x < TM; x++)
#pragma unroll
        for (int u = 0; u < U; u++) parts[(wave * TM * U + x * U + u) * 64 + lane] = acc[x][u];
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int x = 0; x < TM; x++)
#pragma unroll
          for (int u = 0; u < U; u++)
#pragma unroll
            for (int w = 1; w < WK; w++) acc[x][u] += parts[(w * TM * U + x * U + u) * 64 + lane];
      }
      __syncthreads();
      if (wave) continue;
    }
#pragma unroll
    for (int x = 0; x < TM; x++) store_columns<U>(acc[x], add, 16 * x + row, group * (16 * U) + quarter * (4 * U), p);
  }
}

// Short rows, k <= 32 KS bytes, whose product is mostly writing: 32 rows of a stay in a wave's
// registers while its workgroup (128 rows) walks over tiles of 64 rows of b, through
// LDS with the next two tiles on their way.  Results leave in whole lines (LineRing).  (KS = 4 to floats spills two of its 168
// registers, 12 bytes of a lane.)
template <int KS, class O>
__global__ __launch_bounds__(256, KS == 8 ? 2 : 3) void product_panel_kernel(Product<O> p, int64_t panels, int64_t tiles_n,
                                                                             int64_t slices) {
  constexpr int PC = 2 * KS, kRow = 32 * KS, L = 64 * PC / 256, kRows = 256 / PC, Y = LineRing<O>::Y;
  constexpr int kWords = (KS + 3) / 4;  // of a lane's scales
  __shared__ __align__(16) char lds[2][64 * kRow];
  __shared__ __align__(256) char rings[4][LineRing<O>::kBytes];
  __shared__ __align__(16) uint8_t sc[2][64 * PC];  // a tile's scales
  __shared__ float sb[2][64];                       // and biases (-0, which changes no sum, without)
  const int tid = threadIdx.x, wave = wave_id(), lane = lane_id(), row = lane % 32, half = lane / 32;
  const int64_t t = tile_of_block(blockIdx.x, panels * slices), slice = t / panels, i0 = (t - slice * panels) * 128;
  const int64_t first = tiles_n * slice / slices, end = tiles_n * (slice + 1) / slices;
  const int k = (int)p.k, piece = tid % PC, r0 = tid / PC, from = min(piece * 16, k - 16);
  auto swap = [](int r) { return KS == 2 ? r / 4 & 3 : KS == 4 ? r / 2 & 7 : r & 15; };  // as in the tiles, by the row's bytes
  i4 rb[L];
  uint32_t rs = 0;  // KS / 2 bytes of a row's scales
  float bias = -0.f;
  auto load = [&](int64_t tile) {
    const uint8_t* b = p.b + tile * 64 * p.b_stride;
    const int last = (int)min(p.n - 1 - tile * 64, (int64_t)63);
#pragma unroll
    for (int q = 0; q < L; q++) rb[q] = *reinterpret_cast<const i4_any*>(b + ((uint32_t)min(r0 + q * kRows, last) * (uint32_t)p.b_stride + from));
    const uint8_t* s = p.b_scales + tile * 64 * p.bs_stride + (uint32_t)min(tid / 4, last) * (uint32_t)p.bs_stride;
    rs = 0;
#pragma unroll
    for (int u = 0; u < KS / 2; u++) {
      const int block = tid % 4 * (KS / 2) + u;
      if (block < p.blocks) rs |= (uint32_t)s[block] << (8 * u);
    }
    if (p.bias && tid < 64) bias = p.bias[tile * 64 + min(tid, last)];
  };
  auto keep = [&](int buffer) {
#pragma unroll
    for (int q = 0; q < L; q++) {
      const int r = r0 + q * kRows;
      *reinterpret_cast<i4*>(lds[buffer] + r * kRow + (piece ^ swap(r)) * 16) = rb[q];
    }
    __builtin_memcpy(sc[buffer] + tid * (KS / 2), &rs, KS / 2);
    if (tid < 64) sb[buffer][tid] = bias;
  };
  load(first);
  const int64_t it = i0 + wave * 32;  // the wave's rows
  const int rows = (int)min(p.m - it, (int64_t)32);
  // step q takes pieces q and KS + q, so a lane's scales are KS bytes in a row
  i4 fa[KS];
  uint32_t sa[kWords] = {};
  {
    const uint8_t* a = p.a + min(it + row, p.m - 1) * p.a_stride;
    const uint8_t* s = p.a_scales + min(it + row, p.m - 1) * p.as_stride;
#pragma unroll
    for (int q = 0; q < KS; q++) {
      const int block = q + KS * half, at = min(block * 16, k - 16);
      fa[q] = without_first(*reinterpret_cast<const i4_any*>(a + at), block * 16 - at);
      if (block < p.blocks) sa[q / 4] |= (uint32_t)s[block] << (8 * (q % 4));
    }
  }
  LineRing<O> ring(rings[wave], p.out, p.out_stride, it, rows, first, p.stream_lines);
  keep(0);
  if (first + 1 < end) load(first + 1);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < KS; q++) asm volatile("" : "+v"(fa[q]));  // these are there: the loop's waits count its own
#pragma unroll
  for (int q = 0; q < L; q++) asm volatile("" : "+v"(rb[q]));
  asm volatile("" : "+v"(rs), "+v"(bias));
  for (int64_t tile = first; tile < end; tile++) {
    const int buffer = (int)(tile - first) & 1;
    const char* b = lds[buffer] + row * kRow;
    f16v acc[2] = {f16v{}, f16v{}};
    uint32_t s[2][kWords];
#pragma unroll
    for (int y = 0; y < 2; y++) {
      const uint8_t* at = sc[buffer] + (32 * y + row) * PC + half * KS;
      if constexpr (KS == 2) s[y][0] = *reinterpret_cast<const uint16_t*>(at);
      else __builtin_memcpy(s[y], __builtin_assume_aligned(at, KS), KS);
    }
    auto step = [&](auto number) {
      constexpr int Q = decltype(number)::value;
      if constexpr (Q < KS) {
#pragma unroll
        for (int y = 0; y < 2; y++)
          acc[y] = mfma<Q % 4>(fa[Q], sa[Q / 4], *reinterpret_cast<const i4*>(b + y * 32 * kRow + ((Q + KS * half) ^ swap(row)) * 16),
                               s[y][Q / 4], acc[y]);
      }
    };
    step(std::integral_constant<int, 0>());
    step(std::integral_constant<int, 1>());
    step(std::integral_constant<int, 2>());
    step(std::integral_constant<int, 3>());
    step(std::integral_constant<int, 4>());
    step(std::integral_constant<int, 5>());
    step(std::integral_constant<int, 6>());
    step(std::integral_constant<int, 7>());
    if (tile + 1 < end) keep(buffer ^ 1);
    if (tile + 2 < end) load(tile + 2);
#pragma unroll
    for (int l = 0; l < 2 / Y; l++) {
#pragma unroll
      for (int y = 0; y < Y; y++) {
        const float add = sb[buffer][(l * Y + y) * 32 + row];
#pragma unroll
        for (int r = 0; r < 16; r += 2) ring.put(y, r, acc[l * Y + y][r] + add, acc[l * Y + y][r + 1] + add);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      ring.leave(tile * (2 / Y) + l, p.n, 128);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
  }
  ring.leave(end * (2 / Y), min(end * 64, p.n), 0);
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

// Whether values go past the L2 (kStreamBytes), us, past it and through it; into three results in turn.  Rows of whole lines or
// halves of them: 1M x 128 floats 81, 106; 500,000 x 128 of 16 bits every 160 26, 38.  Rows one behind the other, whose ends'
// lines meet: of whole 16 bytes, up to 256 of them, 1M x 104 of 16 bits 41, 47, 1M x 52 floats 35, 37 (but 300,000 x 264 of 16 bits
// 36, 32); results that the last cache does not keep beside the codes, 1.2M x 100 of 16 bits (240 MB) 57, 111, 1M x 99 floats
// 97, 130, 1M x 100 of 16 bits (200 MB) 48, 54 (with 120 MB 31, 32; longer rows 250,000 x 1,001 of 16 bits 154, 134, 50,000 x
// 1,004 floats 53, 44; floats that leave only part of a lane's four out of a block 3M x 31 207, 144, 1.5M x 63 150, 124).  Rows
// apart: 1M x 100 floats every 132 144, 173; but at odd places 300,000 x 96 of 16 bits every 128 35, 15, 1M x 33 of 16 bits
// every 40 53, 24, 200,000 x 255 of 16 bits every 300 42, 39; 1M x 100 floats every 131 168, 192.
template <class T>
bool values_past_the_l2(const T* out, int64_t n, int64_t dim, int64_t stride) {
  const int64_t row = dim * (int64_t)sizeof(T), bytes = n * row;
  const int64_t bits = reinterpret_cast<uintptr_t>(out) | stride * (int64_t)sizeof(T) | row;
  if (bytes < kStreamBytes) return false;
  if (bits % 64 == 0) return true;
  if (row > 1040) return false;
  if (stride > dim) return bits % 16 == 0 && bytes >= int64_t{256} << 20;
  if (bytes < int64_t{180} << 20) return bits % 16 == 0 && row <= 256;
  return sizeof(T) == 2 || dim % kBlock <= kBlock - 4;
}

template <class T>
void from_mx4(const uint8_t* codes, int64_t n, int64_t dim, int64_t code_stride, const uint8_t* scales, int64_t scale_stride,
              void* out, int64_t stride, hipStream_t st) {
  constexpr int R = 4;
  const bool past = values_past_the_l2(static_cast<const T*>(out), n, dim, stride);
  in_runs(n, dim, 8 * kVec<T> * R, [&](int64_t blocks, uint32_t per_row, uint32_t magic, int64_t first, unsigned count) {
    hipLaunchKernelGGL((from_mx4_kernel<T, R>), dim3(count), dim3(256), 0, st, codes, blocks, dim, code_stride, scales,
                       scale_stride, static_cast<T*>(out), stride, per_row, magic, first, past);
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

template <int BM, int BN, int WM, int WN, int NB, int G, bool MANY, class O>
void launch_deep(const Product<O>& p, hipStream_t st) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  const int64_t group = std::min<int64_t>(tm, 8);
  constexpr int lds = NB * (BM + BN) * 64 + (G == 1 ? NB : 2) * (BM + BN) * 4 * G + 3 * BN * 4;
  constexpr auto* kernel = &product_deep_kernel<BM, BN, WM, WN, NB, G, MANY, O>;
  allow_lds<kernel>(lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(MANY ? std::min<int64_t>(tm * tn, 256) : tm * tn)), dim3(64 * WM * WN), lds, st, p, tm, tn, group);
  HIP_OK(hipGetLastError());
}

template <int KS, class O>
void launch_panels(const Product<O>& p, hipStream_t st) {
  const int64_t panels = (p.m + 127) / 128, tiles_n = (p.n + 63) / 64;
  // as many workgroups as run at once, each with a like share of b's tiles
  const int64_t slices = std::min(tiles_n, std::max<int64_t>(1, 256 * (KS == 8 ? 2 : 3) / panels));
  hipLaunchKernelGGL((product_panel_kernel<KS, O>), dim3((unsigned)(panels * slices)), dim3(256), 0, st, p, panels, tiles_n, slices);
  HIP_OK(hipGetLastError());
}

// In 64 bits: rows may have 2^26 blocks.
int64_t strip_lds(int64_t blocks, int u, int tm, int wk) {
  return (blocks + 3) / 4 * tm * 1088 + (wk > 1 ? wk * tm * u * 1024 : 0);
}

template <int U, int TM, int WK, class O>
void launch_strips(const Product<O>& p, hipStream_t st) {
  const int64_t groups = (p.n + 16 * U - 1) / (16 * U);
  const int64_t need = strip_lds(p.blocks, U, TM, WK);
  if (need > 160 * 1024) qv::fail(QV_EUNSUPPORTED, "rows too long for strips");
  const int lds = (int)need;
  constexpr int kThreads = WK == 1 ? 256 : 64 * WK;
  // as many workgroups as run at once
  const int64_t most = 256 * std::min(2048 / kThreads, 160 * 1024 / std::max(lds, 1));
  const int64_t blocks = std::min(most, WK == 1 ? (groups + 3) / 4 : groups);
  constexpr auto* kernel = &product_strip_kernel<U, TM, WK, O>;
  allow_lds<kernel>(lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), lds, st, p, groups);
  HIP_OK(hipGetLastError());
}

template <int U, int TM, int K, class O>
void launch_rows(const Product<O>& p, hipStream_t st) {
  const int64_t groups = (p.n + 16 * U - 1) / (16 * U), blocks = (groups + 3) / 4;
  // a's rows cut over workgroups too where b's alone are too few
  const int64_t chunks = (p.m + 16 * TM - 1) / (16 * TM), slices = std::min(chunks, std::max<int64_t>(1, 1024 / blocks));
  const int64_t rows = (chunks + slices - 1) / slices * (16 * TM);
  in_launches(blocks, 256, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL((product_row_kernel<U, TM, K, O>), dim3(count, (unsigned)((p.m + rows - 1) / rows)), dim3(256), 0, st, p,
                       groups, first, rows);
  });
  HIP_OK(hipGetLastError());
}

// Which kernel: rows of up to 128 values, and few of up to 256, stay in registers; large results of short rows leave in
// whole lines; few longer rows read b; others keep the matrix cores busy.
template <class O>
void product(const Product<O>& p, hipStream_t st) {
  const int64_t scale_bits = reinterpret_cast<uintptr_t>(p.a_scales) | reinterpret_cast<uintptr_t>(p.b_scales) | p.as_stride | p.bs_stride;
  const int64_t code_bits = reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) | p.a_stride | p.b_stride;
  const bool near = std::max({p.a_stride, p.b_stride, p.as_stride, p.bs_stride}) < kFar;
  const bool direct = near && code_bits % 16 == 0 && scale_bits % 4 == 0 && p.k % 64 == 0 && p.k > 256;
  const bool four = direct && scale_bits % 16 == 0 && p.k % 256 == 0;
  auto tiles = [&](int64_t size) { return (p.m + size - 1) / size * ((p.n + size - 1) / size); };
  // Large results of short rows leave through lines.  Measured, us, panels and what else there is.  Rows of b in registers, from 96
  // MB on: 1,000 x 50,001 x 100 of 16 bits (100 MB) 28, 31; 10,000 x 50,001 x 128 220, 438; 1,000 x 20,001 x 64 floats (80 MB) 20,
  // 19; 64 x 600,001 x 128 of 16 bits (77 MB) 27, 24; but rows that are whole lines leave the registers so: 10,000 x 50,048 x 128 219, 209.
  // Tiles, from 72 MB on, past 64 rows: 100 x 368,912 x 200 of 16 bits (74 MB) 25, 34; 200 x 200,000 x 256 (80 MB) 25, 29; 1,000 x 20,001 x 256
  // floats (80 MB) 23, 19; 128 x 300,000 x 384 of 16 bits (77 MB) 35, 41; 4,000 x 10,001 x 512 floats (160 MB) 40, 58; 128 x 130,000 x 512
  // (67 MB) 26, 20; 500 x 40,001 x 256 of 16 bits (40 MB) 18, 16; 64 x 600,000 x 384 (77 MB) 58, 46.
  const double bytes = (double)p.m * p.n * sizeof(O);
  const bool lines = near && p.m < 1 << 30;  // (a launch has less than 2^32 threads)
  const bool panels = lines && bytes >= 72e6 && p.m > 64;
  constexpr int U = sizeof(O) == 2 ? 4 : 2;  // strips of 32 bytes of a result's row
  if (p.k < 16) {
    launch_tiles<64, 64, 2, 2, true>(p, st);
  } else if (p.blocks <= 4) {
    if (p.m <= 16) launch_rows<U, 1, 1>(p, st);
    else if (lines && bytes >= 96e6 && !p.stream) launch_panels<2>(p, st);
    else if (p.m <= 32) launch_rows<U, 2, 1>(p, st);
    else launch_rows<U, 4, 1>(p, st);
  } else if (p.blocks <= 8 && p.m <= 32) {
    // (strips: 16 x 300,000 x 200 to 16 bits 13.9 us, here 9.1; tiles: 32 x 300,000 x 200 20, here 11; 64 x 144,162 x 256 11, here 15)
    if (p.m <= 16) launch_rows<U, 1, 2>(p, st);
    else launch_rows<U, 2, 2>(p, st);
  } else if (p.blocks <= 16 && p.m <= 16) {
    // (tiles: 16 x 500,000 x 384 34 us, here 24; of 32 rows they take 9.7 for 100,000 x 512, strips 12.3)
    launch_strips<2, 1, 1>(p, st);
  } else if (p.m <= 32 && direct && tiles(64) < 1 << 23) {
    // (strips and tiles through registers, us: 1 x 100,000 x 1,024: 14.0, 14.0, here 12.1; 1 x 16,384 x 16,384: 42, 70, here 37)
    if (four) launch_deep<64, 64, 2, 2, 4, 4, false>(p, st);
    else launch_deep<64, 64, 2, 2, 4, 1, false>(p, st);
  } else if (p.m <= 32 && p.n <= 8192 && strip_lds(p.blocks, 1, 2, 4) <= 150 * 1024) {
    // A strip's blocks over four waves where tiles are too few.  Measured, us, with tiles and so: 32 x 4,000 x 4,001: 16.7, 12.7; 2,001: 9.4,
    // 8.0; 32 x 20,000 x 1,001: 7.3, 11.9.
    if (p.m <= 16) launch_strips<1, 1, 4>(p, st);
    else launch_strips<1, 2, 4>(p, st);
  } else if (panels && p.k <= 128) {
    launch_panels<4>(p, st);
  } else if (panels && p.k <= 256) {
    launch_panels<8>(p, st);
  } else {
    // By how many tiles there are for the 256 CUs.  Measured to bfloat16, us, with tiles of 256, 128 and 64 straight to LDS
    // and of 128 and 64 through registers: 4,096^3: 45, 60, 101, 62, 93; 2,048 x 4,096 x 4,096: 35, 30, 45, 30, 42; 1,024:
    // 31, 16, 24, 25, 23; 512: 28, 13, 12, 21, 14; 64: 28, 11, 7, 19, 12; 10,000 x 50,048 x 1,024: 399, 468, -, 489, -.
    // Where scales come a word at a time (k no multiple of 512) and rows are long, each word's line is fetched again for
    // the next: 4,096 x 4,096 x 4,224: 55, 83, 148, 65, -; 2,048: -, 45, 76, 35, 57; 1,024: -, 25, 40, 29, 34; 512: -, 18,
    // 21, 24, 18; 64: -, 13, 9, 20, 12; 1,024 x 4,096 x 1,152: -, 8.7, 11.2, 10.9, 10.1.
    // Up to 64 rows, tiles of 64 (64 x 50,000 x 768: 8.3, with tiles of 128 10.5; 64 x 300,000 x 1,024: 48, 56).
    // Tiles of 256 where they are filled to 80 % and fill the CUs' turns so (as for 8-bit rows).
    const bool narrow = std::min(p.m, p.n) <= 64;
    const int64_t turns = (tiles(256) + 255) / 256;
    const bool fill = (double)p.m * p.n >= 0.8 * 65536 * 256 * turns && tiles(256) < int64_t{1} << 31;
    if (four && fill) launch_deep<256, 256, 2, 2, 4, 4, true>(p, st);
    else if (direct && fill) launch_deep<256, 256, 2, 2, 4, 1, true>(p, st);
    else if (four && tiles(64) <= 512) launch_deep<64, 64, 2, 2, 4, 4, false>(p, st);
    else if (four && !narrow && tiles(128) < 1 << 23) launch_deep<128, 128, 2, 2, 4, 4, false>(p, st);
    else if (direct && tiles(64) <= 128) launch_deep<64, 64, 2, 2, 4, 1, false>(p, st);
    else if (direct && !narrow && tiles(128) <= 256) launch_deep<128, 128, 2, 2, 4, 1, false>(p, st);
    else if (narrow || tiles(64) <= 512) launch_tiles<64, 64, 2, 2, false>(p, st);
    else launch_tiles<128, 128, 2, 2, false>(p, st);
  }
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
      const bool stream = (double)m * n * size >= kStreamBytes;
      const bool lines = (reinterpret_cast<uintptr_t>(d_out) | out_stride * size) % 128 == 0;
      product(Product<O>{d_a, a_stride, d_a_scales, a_scale_stride, m, d_b, b_stride, d_b_scales, b_scale_stride, d_bias, n,
                         k / 2, (int)((k + kBlock - 1) / kBlock), o, out_stride, stream && lines, stream},
              st);
    };
    if (out_type == QV_FLOAT) go(static_cast<float*>(d_out));
    else if (out_type == QV_BFLOAT16) go(static_cast<bf16*>(d_out));
    else go(static_cast<f16*>(d_out));
  });
}

}  // extern "C"
