// nls_attend.h -- what the attention kernels share: element types as matrix
// operands, the parts an fp32 number is split into, a row's place and its keys.
#pragma once
#include <hip/hip_runtime.h>

#include "nls_paged.h"

namespace nls {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float minus_inf() { return -__builtin_inff(); }

// x, computed no earlier than here: keeps what a rare path derives from it out
// of the registers of the loop around it
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <typename TC>
struct Elem;
template <>
struct Elem<_Float16> {
  typedef h8 vec;
  static constexpr int kKeys = 32;  // keys per step of a wave: the depth of one product
  // fp32 as two halves, 22 bits; the weights are up to 2^14, so that small
  // ones stay clear of fp16's denormal range (2^-24 is 2^-38 of the largest)
  static constexpr int kParts = 2;
  static constexpr float kShift = 14.f;
};
template <>
struct Elem<__bf16> {
  typedef b8 vec;
  static constexpr int kKeys = 32;
  static constexpr int kParts = 3;  // fp32 as three times 8 bits, exactly
  static constexpr float kShift = 0.f;
};
template <>
struct Elem<float> {
  typedef f4 vec;
  static constexpr int kKeys = 16;
  static constexpr int kParts = 1;
  static constexpr float kShift = 0.f;
};
// 16-bit queries: the weights are rounded to the cache's type for the products.
// The values are then divided by the sum of the rounded weights, which takes the
// common part of the roundings out (all of it where one key has all the
// weight); lse goes by the sum of the weights themselves.
template <typename T, typename TC>
constexpr bool rounds_weights() {
  return sizeof(T) == 2;
}
template <typename T, typename TC>
constexpr int parts_of() {
  return sizeof(T) == 4 ? Elem<TC>::kParts : 1;
}

__device__ __forceinline__ f4 mma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma16(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// four elements of the depth per lane, one product each
__device__ __forceinline__ f4 mma16(f4 a, f4 b, f4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// x as N parts of the cache's type, largest first, into element j of p[0 .. N)
template <int N>
__device__ __forceinline__ void split(float x, h8* p, int j) {
  const _Float16 hi = (_Float16)x;
  p[0][j] = hi;
  if constexpr (N > 1) p[1][j] = (_Float16)(x - (float)hi);
}
template <int N>
__device__ __forceinline__ void split(float x, b8* p, int j) {
  if constexpr (N == 1) {
    p[0][j] = (__bf16)x;
  } else {
    // the upper 16 bits, cut: what is left is exact
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
      p[i][j] = __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(x) >> 16));
      x -= hi;
    }
  }
}
template <int N>
__device__ __forceinline__ void split(float x, f4* p, int j) {
  p[0][j] = x;
}

// fp32 queries over fp16: the exponent of the power of two that a row is divided
// by, from its largest element.  That comes into [2^13, 2^14): its lower part
// keeps 11 bits too.  (The power is a normal number: rows of denormals stay
// below, at 2^-23 or more.)
__device__ __forceinline__ int query_exponent(float top) {
  const int e = top > 0.f && top < __builtin_inff() ? ilogbf(top) - 13 : 0;
  return e < -126 ? -126 : e;
}

// c plus the elements of x, two products with 1 at a time
__device__ __forceinline__ float plus_all(h8 x, float c) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 8; j += 2) c = __builtin_amdgcn_fdot2(h2{x[j], x[j + 1]}, h2{1, 1}, c, false);
  return c;
}
__device__ __forceinline__ float plus_all(b8 x, float c) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 8; j += 2) c = __builtin_amdgcn_fdot2_f32_bf16(b2{x[j], x[j + 1]}, b2{1.f, 1.f}, c, false);
  return c;
}

// Which keys a sequence's tokens see: row r of kv head's group is token r /
// group at position p, keys [low(p), p].
struct Sees {
  int64_t lo, p0;  // the first key of all; token 0's position
  int window;
  int64_t len;
  __device__ int64_t low(int64_t p) const {
    const int64_t w = p + 1 - window;
    return window > 0 && w > lo ? w : lo;
  }
};
__device__ __forceinline__ Sees sees_of(const AttendArgs& a, const Chunk& c) {
  Sees s;
  s.p0 = position_of(a.p, c, 0);
  s.lo = a.first && c.slot >= 0 ? a.first[c.slot] : 0;
  if (s.lo < 0) s.lo = 0;
  s.window = a.window;
  s.len = c.len;
  return s;
}

// A position or key as an int: what is beyond the ints is beyond every key.
__device__ __forceinline__ int as_int(int64_t x) { return x < -1 ? -1 : x > 0x7fffffff ? 0x7fffffff : (int)x; }

// The keys that tokens t0 .. t1 see between them, from a multiple of 32 on, and
// the parts of `keys` keys that they fall into (the last one takes the rest).
struct Span {
  int lo, hi, parts;
  __device__ int begin(int part, int keys) const { return lo + part * keys; }
  __device__ int end(int part, int keys) const { return part + 1 == parts ? hi : lo + (part + 1) * keys; }
};
__device__ __forceinline__ Span span_of(const Sees& s, int t0, int t1, int keys, int most) {
  Span r;
  const int64_t end = s.p0 + t1 + 1 < s.len ? s.p0 + t1 + 1 : s.len;
  r.hi = as_int(end < 0 ? 0 : end);
  r.lo = as_int(s.low(s.p0 + t0)) & ~31;
  if (r.lo > r.hi) r.lo = r.hi;  // no key: no step begins behind the last one
  const uint32_t n = r.hi > r.lo ? ((uint32_t)(r.hi - r.lo) + (uint32_t)keys - 1) / (uint32_t)keys : 1;
  r.parts = n < (uint32_t)most ? (int)n : most < 1 ? 1 : most;
  return r;
}

// Where the parts of rows that are split over workgroups wait to be joined
// (rows: few_rows' 16 of each task, chunk_rows' token times heads + head):
// fp32 sums [part][row][D] relative to the part's largest score, and that
// score (times log2 e) with the sum of the weights, and of the weights as the
// products took them.
struct Parts {
  float* o;
  f4* ml;
  int64_t rows;   // of one part
  int keys;       // of one part
  int most;       // parts at most; 1 or 0: none are used
};

constexpr int kChunkTile = 128;  // rows of a workgroup of the chunk kernel
// log2 of the weight of a row's largest score: room for weights 2^8 larger
template <typename TC>
constexpr float chunk_shift() {
  return __is_same(TC, _Float16) ? 7.f : 0.f;
}
// Where few rows and chunks share a launch: where registers for as many waves
// suit both (one SIMD takes two of either, or one).
template <typename TC, int D>
constexpr bool together() {
  return D == 256 || (D == 128 && sizeof(TC) == 2);
}
// few: the parts of the sequences of few rows, which the launch takes too where
// they go together; NULL: those are chunks as well
hipError_t launch_chunk(const AttendArgs& a, int type, int cache_type, const Parts& parts, int64_t tiles,
                        const Parts* few, int few_tiles, hipStream_t s);

// How a call's rows are dealt out.
struct AttendPlan {
  bool few, chunk;        // which kernels run
  int few_tiles;          // of 16 rows per sequence and kv head (single tokens of wide groups: several)
  int64_t chunk_tiles;
  Parts few_parts, chunk_parts;  // (pointers unset)
  size_t few_bytes, chunk_bytes;
};

}  // namespace nls
