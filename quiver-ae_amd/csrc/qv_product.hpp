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
// (So neither value is a matrix instruction's result itself: the compiler would not wait for it.)
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
// m, n, out, out_stride: the whole output.  WHOLE: all of it lies in the output.  STREAM: past the caches (kStreamBytes).
template <bool WHOLE, bool STREAM, int R, class O, class F>
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
      if (WHOLE || i + r < m) {
        if constexpr (STREAM) __builtin_nontemporal_store(u[r], reinterpret_cast<i4_any*>(to + r * out_stride));
        else *reinterpret_cast<i4_any*>(to + r * out_stride) = u[r];
      }
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

// Results of a wave's 32 rows on their way to memory, 64 columns at a time, in whole lines.
//
// Memory takes whole aligned lines of 128 bytes at 5.4 TB/s and rows cut elsewhere at
// 3.3 to 3.8, and rows of an odd length begin anywhere.  So a wave keeps, per row, a
// ring of two lines in LDS in which an element's place follows its address: a line is
// written whole as soon as its last column is there, and only the first and the last
// one of a walk over columns are written in parts.
template <class O>
struct LineRing {
  static constexpr int S = (int)sizeof(O), E = 128 / S, V = 16 / S;  // elements of a line, of 16 bytes
  static constexpr int kRing = 256, Y = E / 32;                      // bytes of a row's ring; 32-column results to a line
  static constexpr int kBytes = 32 * kRing;                          // of a wave, aligned to kRing
  static constexpr int G = 4;                                        // lines leave by 8 lanes each, 8 rows at once
  char* ring;
  uint32_t place[Y][16];  // where the lane's columns of a line go in the ring, register 4 g + e of result y; those of the
                          // next line half a ring on
  char* line_to[G];
  int rel[G], rows;
  int64_t lo;
  bool stream;

  // rows [it, it + rows) of `out`, columns from 64 first on; stream: past the caches (kStreamBytes)
  __device__ __forceinline__ LineRing(char* ring, O* out, int64_t out_stride, int64_t it, int rows, int64_t first, bool stream)
      : ring(ring), rows(rows), lo(first * 64), stream(stream) {
    const int lane = dev::lane_id(), row = lane % 32, half = lane / 32, c = lane % 8;
    // elements of its line before a row's first one
    auto shift = [&](int r) { return (int)(reinterpret_cast<uintptr_t>(out + (it + r) * out_stride) % 128) / S; };
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int y = 0; y < Y; y++) {
          const int at = (int)(first & 1) * 64 + 32 * y + row + shift(8 * g + 4 * half + e);
          place[y][4 * g + e] = dev::lds_addr(ring) + 4 * half * kRing + (at * S & (kRing - 1));
        }
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int r = 8 * g + lane / 8, sh = shift(r);
      rel[g] = c * V - sh;
      line_to[g] = reinterpret_cast<char*>(out + (it + r) * out_stride + (first * 64 + rel[g]));
    }
  }
  // registers r and r + 1 of the 32 columns' result y of the line to come (two_of's condition holds here too)
  __device__ __forceinline__ void put(int y, int r, float v0, float v1) {
    typedef O o2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) O lds_o;
    o2 out;
    if constexpr (sizeof(O) == 2) out = __builtin_bit_cast(o2, two_of<O>(v0, v1));
    else out = o2{v0, v1};
#pragma unroll
    for (int d = 0; d < 2; d++) {
      uint32_t& at = place[y][r + d];
      ((lds_o*)(uintptr_t)at)[(r / 4 * 8 + r % 4 + d) * kRing / S] = out[d];
      at ^= 128;
    }
  }
  // line number `line` (the E elements from column line E - shift on) of every row, columns [lo, hi) of it
  __device__ __forceinline__ void leave(int64_t line, int64_t hi, int64_t step) {
    const int lane = dev::lane_id(), c = lane % 8;
    const int least = (int)max(lo - line * E, (int64_t)-1024), most = (int)min(hi - line * E, (int64_t)1024);
    const char* from = ring + (int)(line & 1) * 128 + c * 16;
    if (rows == 32 && least <= 1 - E && most >= E) {  // whole lines of all rows
      i4 u[G];
#pragma unroll
      for (int g = 0; g < G; g++) u[g] = *reinterpret_cast<const i4*>(from + (8 * g + lane / 8) * kRing);
#pragma unroll
      for (int g = 0; g < G; g++) {
        store_past(u[g], reinterpret_cast<i4*>(line_to[g]), stream);
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
  }
};

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
