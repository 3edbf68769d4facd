// nls_quant.hip -- rows of a cache read back: the last tokens of each sequence
// as [tokens, kv_heads, head_dim], from pages of any type.
//
// Bound by the bytes: a row's elements are converted (blocks: one product with
// the factor, rounded once) as they pass.  16 contexts of up to 4000 tokens, 8
// heads of 128, Q4_0 to bf16 (220 MB): 54 us with two sets of rows in turn, 58 with six,
// 3.8 TB/s, four fifths of what a large copy reaches.  A workgroup for each token,
// whose look-ups are a wait of their own, 76; values stored in 8 bytes a lane 56 and
// 63; stores that pass the caches 60 and 71.
#include "nls_quant.h"

namespace nls {
namespace {

constexpr int kReadThreads = 256;

template <typename T, int N, bool kWide>
__device__ __forceinline__ void put(T* to, const float* x) {
  if constexpr (kWide) {
    typedef T vec __attribute__((ext_vector_type(N)));
    vec r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)x[i];
    __builtin_memcpy(__builtin_assume_aligned(to, sizeof(T) * N < 16 ? sizeof(T) * N : 16), &r, sizeof r);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = (T)x[i];
  }
}

// Tokens without a place read as zeros.
template <typename T, typename TC, bool kWide>
__global__ __launch_bounds__(kReadThreads) void read_kernel(ReadArgs r, int tokens) {
  __shared__ TokenPlace places[kTokensMost];
  const PagedArgs& a = r.p;
  const int first = blockIdx.x * tokens, n = a.tokens - first < tokens ? a.tokens - first : tokens;
  find_places(a, first, n, places);
  __syncthreads();
  const int per = a.dim / 8, all = 2 * per * a.kv_heads;
  for (int w = threadIdx.x; w < all * n; w += kReadThreads) {
    const int j = w / all, i = w % all, k = i >= per * a.kv_heads, u = k ? i - per * a.kv_heads : i;
    const int head = u / per, d = u % per * 8;
    const TokenPlace p = places[j];
    if (p.seq < 0) continue;
    const HeadsView& to = k ? r.v : r.k;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (p.page >= 0) {
      typedef TC vec __attribute__((ext_vector_type(8)));
      const TC* from = static_cast<const TC*>(a.kv) + token_offset(a, p.page, p.pos) + head * a.head_stride +
                       (k ? a.value_offset : 0) + d;
      vec y;
      __builtin_memcpy(&y, __builtin_assume_aligned(from, 16), sizeof y);
#pragma unroll
      for (int z = 0; z < 8; ++z) x[z] = (float)y[z];
    }
    put<T, 8, kWide>(static_cast<T*>(to.d) + (first + j) * to.token_stride + head * to.head_stride + d, x);
  }
}

// A thread takes 8 neighbouring elements of a key, or 4 neighbours of either half
// of each block of a value's plane, whose codes are one piece of the row.
template <typename T, int kBits, bool kWide>
__global__ __launch_bounds__(kReadThreads) void read_quant_kernel(ReadArgs r, int tokens) {
  __shared__ TokenPlace places[kTokensMost];
  const PagedArgs& a = r.p;
  const int first = blockIdx.x * tokens, n = a.tokens - first < tokens ? a.tokens - first : tokens;
  find_places(a, first, n, places);
  __syncthreads();
  const int size = 1 << a.page_shift;
  const QuantShape s = quant_shape(kBits == 8 ? kQ8_0 : kQ4_0, a.dim, size);
  const int planes = plane_count(s.groups);
  const int nk = 4 * s.groups * a.kv_heads, nv = 4 * planes * a.kv_heads;
  for (int w = threadIdx.x; w < (nk + nv) * n; w += kReadThreads) {
    const bool key = w < nk * n;
    const int j = key ? w / nk : (w - nk * n) / nv, u = key ? w % nk : (w - nk * n) % nv, g = u & 3;
    const TokenPlace p = places[j];
    if (p.seq < 0) continue;
    const int place = (int)(p.pos & (size - 1));
    const char* home = static_cast<const char*>(a.kv) + (int64_t)(p.page < 0 ? 0 : p.page) * a.page_stride;
    if (key) {
      const int head = u / (4 * s.groups), b = u % (4 * s.groups) >> 2;
      const char* from = home + quant_base(s, head, 0);
      const float d = (float)reinterpret_cast<const _Float16*>(from + s.codes)[b * size + place];
      uint32_t c[kBits / 4];
      __builtin_memcpy(c, __builtin_assume_aligned(from + place * s.row + key_at(s, b, g), kBits), kBits);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float code = kBits == 8 ? (float)(int)((c[e / 4 * (kBits / 8)] >> (8 * (e & 3))) & 255) - 128.f
                                      : (float)(int)((c[0] >> (4 * nibble_of(e))) & 15) - 8.f;
        x[e] = p.page < 0 ? 0.f : d * code;
      }
      put<T, 8, kWide>(static_cast<T*>(r.k.d) + (first + j) * r.k.token_stride + head * r.k.head_stride + 32 * b + 8 * g, x);
    } else {
      const int head = u / (4 * planes);
      const Plane plane = plane_of(s.groups, u % (4 * planes) >> 2);
      const char* from = home + quant_base(s, head, 1);
      T* to = static_cast<T*>(r.v.d) + (first + j) * r.v.token_stride + head * r.v.head_stride + 32 * plane.first + 4 * g;
      by_width(plane.wide, [&](auto wide) {
        constexpr int W = wide, kBytes = W * kBits;
        uint32_t c[kBytes / 4];
        __builtin_memcpy(c, __builtin_assume_aligned(from + place * s.row + value_at(s, plane, 4 * g), kBytes < 16 ? kBytes : 16),
                         kBytes);
        float d[W];
#pragma unroll
        for (int b = 0; b < W; ++b) d[b] = (float)reinterpret_cast<const _Float16*>(from + s.codes)[(plane.first + b) * size + place];
#pragma unroll
        for (int b = 0; b < W; ++b) {
          float x[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const int byte = (z * W + b) * (kBits / 4) + (kBits == 8 ? h : 0);
              const uint32_t code = c[byte / 4] >> (8 * (byte % 4) + (kBits == 8 ? 0 : 4 * h));
              x[h][z] = p.page < 0 ? 0.f : d[b] * ((float)(int)(code & (kBits == 8 ? 255 : 15)) - (kBits == 8 ? 128.f : 8.f));
            }
          if constexpr (kWide && sizeof(T) == 2) {
            // two lanes' 4 of either half become 8 of one half each
            uint32_t w[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              T r[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) r[z] = (T)x[h][z];
              __builtin_memcpy(w[h], r, sizeof r);
            }
            const int odd = g & 1;
            uint32_t q[4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const uint32_t got = __builtin_amdgcn_mov_dpp(odd ? w[0][n] : w[1][n], 0xb1, 0xf, 0xf, false);  // of lane ^ 1
              q[n] = odd ? got : w[0][n];
              q[2 + n] = odd ? w[1][n] : got;
            }
            __builtin_memcpy(__builtin_assume_aligned(to + 32 * b + (odd ? 12 : 0), 16), q, sizeof q);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) put<T, 4, kWide>(to + 32 * b + 16 * h, x[h]);
          }
        }
      });
    }
  }
}

template <typename T, bool kWide>
hipError_t read_of(const ReadArgs& a, int cache_type, hipStream_t s) {
  const int per = tokens_of_group(a.p.tokens), n = (a.p.tokens + per - 1) / per;
  switch (cache_type) {
    case kF32: read_kernel<T, float, kWide><<<n, kReadThreads, 0, s>>>(a, per); break;
    case kF16: read_kernel<T, _Float16, kWide><<<n, kReadThreads, 0, s>>>(a, per); break;
    case kBF16: read_kernel<T, __bf16, kWide><<<n, kReadThreads, 0, s>>>(a, per); break;
    case kQ8_0: read_quant_kernel<T, 8, kWide><<<n, kReadThreads, 0, s>>>(a, per); break;
    default: read_quant_kernel<T, 4, kWide><<<n, kReadThreads, 0, s>>>(a, per); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_read(const ReadArgs& a, int type, int cache_type, bool wide, hipStream_t s) {
  switch (type) {
    case kF32: return wide ? read_of<float, true>(a, cache_type, s) : read_of<float, false>(a, cache_type, s);
    case kF16: return wide ? read_of<_Float16, true>(a, cache_type, s) : read_of<_Float16, false>(a, cache_type, s);
    default: return wide ? read_of<__bf16, true>(a, cache_type, s) : read_of<__bf16, false>(a, cache_type, s);
  }
}

}  // namespace nls
