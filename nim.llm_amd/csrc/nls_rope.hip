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

}  // namespace

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
