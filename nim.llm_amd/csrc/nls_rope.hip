// nls_rope.hip -- rotary positions, and the new tokens' way into the cache.
//
// A pair (a, b) of a head at position p turns by p f_j:
//   a' = s (a cos - b sin),  b' = s (b cos + a sin).
// Both kernels are bound by the bytes they pass on.  One workgroup takes one
// token: its dim / 2 sines and cosines are computed once, into LDS, and serve
// all of its heads.  The angle p f_j is float64 and reduced there to [-pi, pi]
// (at position 10^6 an fp32 angle is off by 0.03), its sine and cosine are fp32,
// each to a few units of its own last place.
// 8191 tokens of 32 heads of 128, bf16 (134 MB): 24.6 us, 5.4 TB/s.
#include "nls_paged.h"
#include "nls_quant.h"

namespace nls {
namespace {

constexpr int kTurnThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {  // one rounding, to nearest even
  return (T)x;
}

template <typename T, int N>
struct Pack {  // (a vector, so that it is loaded and stored whole)
  T v __attribute__((ext_vector_type(N)));
  static constexpr int kAlign = sizeof(T) * N < 16 ? sizeof(T) * N : 16;
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> x;
  __builtin_memcpy(&x, __builtin_assume_aligned(p, Pack<T, N>::kAlign), sizeof(T) * N);
  return x;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) {
  __builtin_memcpy(__builtin_assume_aligned(p, Pack<T, N>::kAlign), &x, sizeof(T) * N);
}

// sin and cos of each pair at position `pos`, times the amplitude
__device__ void turn_table(const TurnArgs& t, int64_t pos, float2* cs) {
  for (int j = threadIdx.x; j < t.rot / 2; j += kTurnThreads) {
    const double angle = (double)pos * t.freqs[j];
    const double n = __builtin_rint(angle * 0.15915494309189535);
    // 2 pi as the sum of two float64
    const double r = __builtin_fma(-n, 2.4492935982947064e-16, __builtin_fma(-n, 6.283185307179586, angle));
    // of its first 24 bits, then turned by the rest, which counts where either is
    // next to 0
    const float hi = (float)r, lo = (float)(r - (double)hi);
    float s0, c0;
    sincosf(hi, &s0, &c0);
    const float s = __builtin_fmaf(lo, c0, s0), c = __builtin_fmaf(-lo, s0, c0);
    cs[j] = make_float2(c * t.amplitude, s * (t.amplitude * t.sign));
  }
}

// The work of one head, in units: first the units of N pairs each, then those
// of N elements behind the turned ones.  N pairs are N elements of either half,
// or 2 N neighbours when interleaved.
template <typename T, int N>
struct Unit {
  Pack<T, N> a, b;
};
template <typename T, int N, bool kInterleaved>
__device__ __forceinline__ Unit<T, N> load_unit(const T* x, int u, int rot) {
  const int pairs = rot / (2 * N);
  Unit<T, N> r;
  if (u < pairs) {
    r.a = load_pack<T, N>(x + (kInterleaved ? 2 * u * N : u * N));
    r.b = load_pack<T, N>(x + (kInterleaved ? 2 * u * N + N : u * N + rot / 2));
  } else {
    r.a = load_pack<T, N>(x + rot + (u - pairs) * N);
  }
  return r;
}

template <typename T, typename TO, int N, bool kInterleaved>
__device__ __forceinline__ void store_unit(const Unit<T, N>& x, TO* y, int u, int rot, const float2* cs) {
  const int pairs = rot / (2 * N);
  if (u < pairs) {
    const int j = u * N;
    const int ia = kInterleaved ? 2 * j : j, ib = kInterleaved ? 2 * j + N : j + rot / 2;
    const Pack<T, N>&p = x.a, &q = x.b;
    Pack<TO, N> r, w;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kInterleaved && N == 1) {
        const float a = to_f(p.v[0]), b = to_f(q.v[0]);
        r.v[0] = from_f<TO>(a * cs[j].x - b * cs[j].y);
        w.v[0] = from_f<TO>(b * cs[j].x + a * cs[j].y);
      } else if constexpr (kInterleaved) {
        if (i & 1) continue;
        const float2 c0 = cs[j + i / 2], c1 = cs[j + N / 2 + i / 2];
        const float a0 = to_f(p.v[i]), b0 = to_f(p.v[i + 1]), a1 = to_f(q.v[i]), b1 = to_f(q.v[i + 1]);
        r.v[i] = from_f<TO>(a0 * c0.x - b0 * c0.y);
        r.v[i + 1] = from_f<TO>(b0 * c0.x + a0 * c0.y);
        w.v[i] = from_f<TO>(a1 * c1.x - b1 * c1.y);
        w.v[i + 1] = from_f<TO>(b1 * c1.x + a1 * c1.y);
      } else {
        const float2 c = cs[j + i];
        const float a = to_f(p.v[i]), b = to_f(q.v[i]);
        r.v[i] = from_f<TO>(a * c.x - b * c.y);
        w.v[i] = from_f<TO>(b * c.x + a * c.y);
      }
    }
    store_pack(y + ia, r);
    store_pack(y + ib, w);
    return;
  }
  if constexpr (__is_same(T, TO)) {
    store_pack(y + rot + (u - pairs) * N, x.a);
  } else {
    Pack<TO, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = from_f<TO>(to_f(x.a.v[i]));
    store_pack(y + rot + (u - pairs) * N, r);
  }
}

template <typename T, int N, bool kInterleaved>
__global__ __launch_bounds__(kTurnThreads) void rope_kernel(TurnArgs t) {
  __shared__ float2 cs[kMaxHeadDim / 2];
  const int token = blockIdx.x;
  const bool in_place = t.x.d == t.y.d;
  const int units = in_place ? t.rot / (2 * N) : t.rot / (2 * N) + (t.dim - t.rot) / N, all = units * t.heads;
  const T* x = static_cast<const T*>(t.x.d) + token * t.x.token_stride;
  T* y = static_cast<T*>(t.y.d) + token * t.y.token_stride;
  auto load = [&](int w) { return load_unit<T, N, kInterleaved>(x + w / units * t.x.head_stride, w % units, t.rot); };
  auto store = [&](const Unit<T, N>& d, int w) {
    store_unit<T, T, N, kInterleaved>(d, y + w / units * t.y.head_stride, w % units, t.rot, cs);
  };
  turn_table(t, t.positions[token], cs);
  __syncthreads();
  for (int w = threadIdx.x; w < all; w += kTurnThreads) store(load(w), w);
}

template <typename T, typename TC, int N, bool kInterleaved>
__global__ __launch_bounds__(kTurnThreads) void append_kernel(TurnArgs t, PagedArgs a) {
  __shared__ float2 cs[kMaxHeadDim / 2];
  const int token = blockIdx.x;
  // The rows in units: q's, k's, v's.  A thread's first is requested before the
  // look-ups that say where the token belongs, a chain of loads that takes as
  // long (prompts of 6100 tokens in 48 heads of 128, bf16, 150 MB: 43.8 us when
  // all are requested behind it, 30.8 us so, 4.9 TB/s; two ahead: 31.0).
  const int rot = t.freqs ? t.rot : 0;
  const int pairs = rot / (2 * N), units = pairs + (t.dim - rot) / N, per = t.dim / N;
  const int qu = t.heads ? (t.x.d == t.y.d ? pairs : units) : 0;  // in place, what is not turned stays
  const int nq = qu * t.heads, nk = units * a.kv_heads, all = nq + nk + per * a.kv_heads;
  const T* x = static_cast<const T*>(t.x.d) + token * t.x.token_stride;
  T* y = static_cast<T*>(t.y.d) + token * t.y.token_stride;
  const T* k = static_cast<const T*>(t.k.d) + token * t.k.token_stride;
  const T* v = static_cast<const T*>(t.v.d) + token * t.v.token_stride;
  auto load = [&](int w) {
    if (w < nq) return load_unit<T, N, kInterleaved>(x + w / qu * t.x.head_stride, w % qu, rot);
    w -= nq;
    if (w < nk) return load_unit<T, N, kInterleaved>(k + w / units * t.k.head_stride, w % units, rot);
    w -= nk;
    return load_unit<T, N, kInterleaved>(v + w / per * t.v.head_stride, w % per, 0);
  };
  Unit<T, N> first;
  if ((int)threadIdx.x < all) first = load(threadIdx.x);

  // the token's sequence: the starts not behind it, less one (64 at a time)
  const int lane = threadIdx.x & 63;
  int seq = -1;
  for (int s0 = 0; s0 < a.seqs + 1; s0 += 64) {
    const int s = s0 + lane;
    const int n = __popcll(__ballot(s <= a.seqs && a.starts[s <= a.seqs ? s : a.seqs] <= token));
    seq += n;
    if (n < 64) break;
  }
  if (seq < 0 || seq >= a.seqs) return;  // a row of no sequence
  const Chunk c = chunk_of(a, seq);
  const int64_t pos = position_of(a, c, token - c.begin);
  const int page = page_of(a, c.slot, pos);
  if (t.freqs) turn_table(t, pos, cs);
  __syncthreads();
  TC* row = static_cast<TC*>(a.kv) + (page < 0 ? 0 : token_offset(a, page, pos));
  auto store = [&](const Unit<T, N>& d, int w) {
    if (w < nq) {
      store_unit<T, T, N, kInterleaved>(d, y + w / qu * t.y.head_stride, w % qu, rot, cs);
      return;
    }
    if (page < 0) return;
    w -= nq;
    if (w < nk) {
      store_unit<T, TC, N, kInterleaved>(d, row + w / units * a.head_stride, w % units, rot, cs);
      return;
    }
    w -= nk;
    store_unit<T, TC, N, kInterleaved>(d, row + a.value_offset + w / per * a.head_stride, w % per, 0, cs);
  };
  if ((int)threadIdx.x < all) store(first, threadIdx.x);
  for (int w = threadIdx.x + kTurnThreads; w < all; w += kTurnThreads) store(load(w), w);
}

template <typename T, int N>
hipError_t rope_of(const TurnArgs& t, hipStream_t s) {
  if (t.interleaved)
    rope_kernel<T, N, true><<<t.tokens, kTurnThreads, 0, s>>>(t);
  else
    rope_kernel<T, N, false><<<t.tokens, kTurnThreads, 0, s>>>(t);
  return hipGetLastError();
}

template <typename T, typename TC, int N>
hipError_t append_of(const TurnArgs& t, const PagedArgs& a, hipStream_t s) {
  if (t.interleaved)
    append_kernel<T, TC, N, true><<<t.tokens, kTurnThreads, 0, s>>>(t, a);
  else
    append_kernel<T, TC, N, false><<<t.tokens, kTurnThreads, 0, s>>>(t, a);
  return hipGetLastError();
}

template <typename T, typename TC>
hipError_t append_width(const TurnArgs& t, const PagedArgs& a, bool wide, hipStream_t s) {
  return wide ? append_of<T, TC, 8>(t, a, s) : append_of<T, TC, 1>(t, a, s);
}

// ---------------------------------------------------------------- pages of blocks

// The largest and least of a block's elements, and whether one is not finite: of
// 8 in each of 4 neighbouring lanes.
__device__ __forceinline__ void over_block(const float* x, float& hi, float& lo, int& odd) {
  hi = lo = x[0];
  odd = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hi = fmaxf(hi, x[j]);
    lo = fminf(lo, x[j]);
    odd |= !(fabsf(x[j]) < __builtin_inff());
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    hi = fmaxf(hi, __shfl_xor(hi, d));
    lo = fminf(lo, __shfl_xor(lo, d));
    odd |= __shfl_xor(odd, d);
  }
}

// A block's factor, and what its elements are multiplied by.
template <int kBits>
__device__ __forceinline__ _Float16 factor_of(float hi, float lo, int odd, float* step) {
  const float t = kBits == 8 ? fmaxf(hi, -lo) * 0.007874015718698502f : fmaxf(hi * 0.1428571492433548f, lo * -0.125f);
  const _Float16 d = (_Float16)fminf(t, kBits == 8 ? 515.5f : 8188.f);  // (so that fp16 holds d c)
  *step = (float)d > 0.f ? 1.f / (float)d : 0.f;
  return odd ? (_Float16)__builtin_nanf("") : d;
}

// The element's code as it is held.
template <int kBits>
__device__ __forceinline__ uint32_t code_of(float x, float step) {
  constexpr float kLow = kBits == 8 ? -127.f : -8.f, kHigh = kBits == 8 ? 127.f : 7.f;
  const float c = __builtin_rintf(x * step);
  return (uint32_t)((int)fminf(fmaxf(c, kLow), kHigh) + (kBits == 8 ? 128 : 8));  // (NaN: the lowest)
}

// 8 neighbouring elements of a row from d on, turned.
enum Turn { kNoTurn, kNeighbours, kHalves };
template <typename T, bool kWide, Turn kTurn>
__device__ __forceinline__ void turned8(const T* row, int d, int rot, const float2* cs, float (&x)[8]) {
  if constexpr (kWide) {
    const Pack<T, 8> p = load_pack<T, 8>(row + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f(p.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f(row[d + e]);
  }
  if constexpr (kTurn == kNeighbours) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if (d + e >= rot) break;
      const float2 c = cs[(d + e) / 2];
      const float a = x[e], b = x[e + 1];
      x[e] = a * c.x - b * c.y;
      x[e + 1] = b * c.x + a * c.y;
    }
  }
  if constexpr (kTurn == kHalves) {
    const int half = rot / 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (d + e >= rot) break;
      const bool low = d + e < half;
      const int j = low ? d + e : d + e - half;
      const float2 c = cs[j];
      const float other = to_f(row[low ? d + e + half : j]);
      x[e] = low ? x[e] * c.x - other * c.y : x[e] * c.x + other * c.y;
    }
  }
}

// Tokens' k and v into pages of blocks, and their q turned.  A block is four
// lanes of 8 elements: a key's of neighbours, a value's of 4 neighbours in either
// half, whose codes are one piece of the row (nls_quant.h).  Factors and codes
// come of fp32 products alone, each rounded once, so that they are the same
// numbers wherever they are computed.
// Bound by the bytes: prompts of 6102 tokens, 8 heads of 128, bf16 to Q8_0
// (38 MB): 13 us, what the launch and two trips to memory cost included (a
// workgroup for each token 18).
template <typename T, int kBits, bool kWide, Turn kTurn>
__global__ __launch_bounds__(kTurnThreads) void append_quant_kernel(TurnArgs t, PagedArgs a, int tokens) {
  constexpr int N = kWide ? 8 : 1;
  constexpr bool kInterleaved = kTurn == kNeighbours;
  __shared__ float2 turns[kTurn == kNoTurn ? 1 : kTokensMost][kMaxHeadDim / 2];
  __shared__ TokenPlace places[kTokensMost];
  const int first = blockIdx.x * tokens, n = t.tokens - first < tokens ? t.tokens - first : tokens;
  const int rot = kTurn == kNoTurn ? 0 : t.rot;
  const int pairs = rot / (2 * N), units = pairs + (t.dim - rot) / N;
  const int qu = t.heads ? (t.x.d == t.y.d ? pairs : units) : 0;
  find_places(a, first, n, places);
  __syncthreads();
  if constexpr (kTurn != kNoTurn) {
    for (int j = 0; j < n; ++j)
      if (places[j].seq >= 0) turn_table(t, places[j].pos, turns[j]);
    __syncthreads();
  }
  if (qu) {
    const int per = qu * t.heads;
    for (int w = threadIdx.x; w < per * n; w += kTurnThreads) {
      const int j = w / per, u = w % per;
      if (places[j].seq < 0) continue;
      const T* x = static_cast<const T*>(t.x.d) + (first + j) * t.x.token_stride + u / qu * t.x.head_stride;
      T* y = static_cast<T*>(t.y.d) + (first + j) * t.y.token_stride + u / qu * t.y.head_stride;
      store_unit<T, T, N, kInterleaved>(load_unit<T, N, kInterleaved>(x, u % qu, rot), y, u % qu, rot,
                                        turns[kTurn == kNoTurn ? 0 : j]);
    }
  }
  const int size = 1 << a.page_shift;
  const QuantShape s = quant_shape(kBits == 8 ? kQ8_0 : kQ4_0, t.dim, size);
  const int planes = plane_count(s.groups);
  // keys of all tokens, then values: four lanes to a block (a plane)
  const int nk = 4 * s.groups * a.kv_heads, nv = 4 * planes * a.kv_heads;
  for (int w = threadIdx.x; w < (nk + nv) * n; w += kTurnThreads) {
    const bool key = w < nk * n;
    const int j = key ? w / nk : (w - nk * n) / nv, u = key ? w % nk : (w - nk * n) % nv;
    const TokenPlace p = places[j];
    if (p.page < 0) continue;
    const int place = (int)(p.pos & (size - 1)), g = u & 3;
    char* home = static_cast<char*>(a.kv) + (int64_t)p.page * a.page_stride;
    if (key) {
      const int head = u / (4 * s.groups), x = u % (4 * s.groups) >> 2;
      float e[8], hi, lo, step;
      int odd;
      turned8<T, kWide, kTurn>(static_cast<const T*>(t.k.d) + (first + j) * t.k.token_stride + head * t.k.head_stride,
                               32 * x + 8 * g, rot, turns[kTurn == kNoTurn ? 0 : j], e);
      over_block(e, hi, lo, odd);
      const _Float16 d = factor_of<kBits>(hi, lo, odd, &step);
      char* to = home + quant_base(s, head, 0);
      uint32_t r[kBits / 4] = {};
#pragma unroll
      for (int z = 0; z < 8; ++z)
        r[kBits == 8 ? z / 4 : 0] |= code_of<kBits>(e[z], step) << (kBits == 8 ? 8 * (z & 3) : 4 * nibble_of(z));
      __builtin_memcpy(__builtin_assume_aligned(to + place * s.row + key_at(s, x, g), kBits), r, kBits);
      if (g == 0) reinterpret_cast<_Float16*>(to + s.codes)[x * size + place] = d;
    } else {
      const int head = u / (4 * planes);
      const Plane plane = plane_of(s.groups, u % (4 * planes) >> 2);
      const T* row = static_cast<const T*>(t.v.d) + (first + j) * t.v.token_stride + head * t.v.head_stride +
                     32 * plane.first + 4 * g;
      char* to = home + quant_base(s, head, 1);
      by_width(plane.wide, [&](auto wide) {
        constexpr int W = wide;
        float e[W][8];
#pragma unroll
        for (int x = 0; x < W; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if constexpr (kWide) {
              const Pack<T, 4> four = load_pack<T, 4>(row + 32 * x + 16 * h);
#pragma unroll
              for (int z = 0; z < 4; ++z) e[x][4 * h + z] = to_f(four.v[z]);
            } else {
#pragma unroll
              for (int z = 0; z < 4; ++z) e[x][4 * h + z] = to_f(row[32 * x + 16 * h + z]);
            }
        uint32_t r[W * kBits / 4] = {};
#pragma unroll
        for (int x = 0; x < W; ++x) {
          float hi, lo, step;
          int odd;
          over_block(e[x], hi, lo, odd);
          const _Float16 d = factor_of<kBits>(hi, lo, odd, &step);
#pragma unroll
          for (int z = 0; z < 4; ++z) {  // lane 4 g + z of the operands
            const uint32_t low = code_of<kBits>(e[x][z], step), high = code_of<kBits>(e[x][4 + z], step);
            const int byte = (z * W + x) * (kBits / 4);
            r[byte / 4] |= (low | high << kBits) << (8 * (byte % 4));
          }
          if (g == 0) reinterpret_cast<_Float16*>(to + s.codes)[(plane.first + x) * size + place] = d;
        }
        constexpr int kBytes = W * kBits;
        __builtin_memcpy(__builtin_assume_aligned(to + place * s.row + value_at(s, plane, 4 * g), kBytes < 16 ? kBytes : 16), r,
                         kBytes);
      });
    }
  }
}

template <typename T, int kBits, bool kWide>
hipError_t append_quant_of(const TurnArgs& t, const PagedArgs& a, hipStream_t s) {
  const int per = tokens_of_group(t.tokens), groups = (t.tokens + per - 1) / per;
  if (!t.freqs)
    append_quant_kernel<T, kBits, kWide, kNoTurn><<<groups, kTurnThreads, 0, s>>>(t, a, per);
  else if (t.interleaved)
    append_quant_kernel<T, kBits, kWide, kNeighbours><<<groups, kTurnThreads, 0, s>>>(t, a, per);
  else
    append_quant_kernel<T, kBits, kWide, kHalves><<<groups, kTurnThreads, 0, s>>>(t, a, per);
  return hipGetLastError();
}
template <typename T>
hipError_t append_quant_type(const TurnArgs& t, const PagedArgs& a, int cache_type, bool wide, hipStream_t s) {
  if (cache_type == kQ8_0) return wide ? append_quant_of<T, 8, true>(t, a, s) : append_quant_of<T, 8, false>(t, a, s);
  return wide ? append_quant_of<T, 4, true>(t, a, s) : append_quant_of<T, 4, false>(t, a, s);
}

}  // namespace

hipError_t launch_append_quant(const TurnArgs& t, const PagedArgs& a, int type, int cache_type, bool wide, hipStream_t s) {
  switch (type) {
    case kF32: return append_quant_type<float>(t, a, cache_type, wide, s);
    case kF16: return append_quant_type<_Float16>(t, a, cache_type, wide, s);
    default: return append_quant_type<__bf16>(t, a, cache_type, wide, s);
  }
}

hipError_t launch_rope(const TurnArgs& t, int type, bool wide, hipStream_t s) {
  switch (type) {
    case kF32: return wide ? rope_of<float, 4>(t, s) : rope_of<float, 1>(t, s);
    case kF16: return wide ? rope_of<_Float16, 8>(t, s) : rope_of<_Float16, 1>(t, s);
    default: return wide ? rope_of<__bf16, 8>(t, s) : rope_of<__bf16, 1>(t, s);
  }
}

hipError_t launch_append(const TurnArgs& t, const PagedArgs& a, int type, int cache_type, bool wide, hipStream_t s) {
  if (type == kF32) {
    if (cache_type == kF32) return append_width<float, float>(t, a, wide, s);
    if (cache_type == kF16) return append_width<float, _Float16>(t, a, wide, s);
    return append_width<float, __bf16>(t, a, wide, s);
  }
  if (type == kF16) return append_width<_Float16, _Float16>(t, a, wide, s);
  return append_width<__bf16, __bf16>(t, a, wide, s);
}

}  // namespace nls
