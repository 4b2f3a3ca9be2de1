// qv_product.hpp -- what the matrix products (8-bit and microscaled 4-bit) share: pieces
// of 16 bytes, waits and their schedule, tiles over the XCDs, results from registers to rows.
#pragma once

#include <atomic>

#include "qv_dense.hpp"
#include "qv_device.hpp"

namespace qv {
namespace dense {

typedef int32_t i4 __attribute__((ext_vector_type(4)));
typedef int32_t i16v __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef i4 i4_any __attribute__((aligned(1), may_alias));
typedef f4 f4_any __attribute__((aligned(4), may_alias));

constexpr int kLoadsDone = 0x0f70;  // s_waitcnt vmcnt(0)
constexpr int kStage = 128;         // bytes of k per stage

// What a piece starting `over` bytes before its place repeats, zeroed.
__device__ __forceinline__ i4 without_first(i4 v, int over) {
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const int cut = over - 4 * w;
    v[w] = cut <= 0 ? v[w] : cut >= 4 ? 0 : (int32_t)((uint32_t)v[w] & (~0u << (8 * cut)));
  }
  return v;
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
    const bool up = dev::lane_id() & D;
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

// Stores the results of R instructions from the registers: 32 R columns from j of the rows around the lane's row i,
// whole lines of 8 rows at once (half lines of 16 rows with 32 columns of 16 bits).  Of the four columns that a lane
// has of every eight, those of 16 bits pass to the other half of the wave and back, eight for a lane; then groups of
// lanes swap rows for pieces of one row.  (Pieces stored as they are, 32 bytes of 32 rows at once, take 5.0 for 5.35
// TB/s in aligned rows, 2 for 3.8 in others.)  four(y, g): the lane's four results of columns 32 y + 8 g + 4 half on.
// m, n, out, out_stride: the whole output.  WHOLE: all of it lies in the output.
template <bool WHOLE, int R, class O, class F>
__device__ __forceinline__ void store_results(F four, int64_t i, int64_t j, int64_t m, int64_t n, O* out, int64_t out_stride) {
  constexpr int V = 16 / (int)sizeof(O), N = 16 / V, P = R * N;  // columns of a piece, pieces of a result, of all
  const int half = dev::lane_id() / 32, c = dev::lane_id() % P;
  i4 u[P];
#pragma unroll
  for (int y = 0; y < R; y++) {
    float v[16];
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const f4 w = four(y, g);
#pragma unroll
      for (int e = 0; e < 4; e++) v[4 * g + e] = w[e];
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
  O* to = out + (i * out_stride + j);
  if (WHOLE || j + V <= n) {
#pragma unroll
    for (int r = 0; r < P; r++)
      if (WHOLE || i + r < m) *reinterpret_cast<i4_any*>(to + r * out_stride) = u[r];
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
        if (i + r < m && j + e < n) to[r * out_stride + e] = piece.o[e];
    }
  }
}

// Workgroups go round the eight XCDs: each XCD gets a run of consecutive tiles.
__device__ __forceinline__ int64_t tile_of_block(int64_t block, int64_t tiles) {
  const int64_t xcd = block % 8, per = tiles / 8, more = tiles % 8;
  return xcd * per + min(xcd, more) + block / 8;
}

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

}  // namespace dense
}  // namespace qv
