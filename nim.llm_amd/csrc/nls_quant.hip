// nls_quant.hip -- rows of a cache read back: the last tokens of each sequence
// as [tokens, kv_heads, head_dim], from pages of any type.
//
// Bound by the bytes: a row's elements are converted (blocks: one product with
// the factor, rounded once) as they pass.  One workgroup takes one token.
#include "nls_quant.h"

namespace nls {
namespace {

constexpr int kReadThreads = 256;

template <typename T, int N>
__device__ __forceinline__ void put(T* to, const float* x) {
  typedef T vec __attribute__((ext_vector_type(N)));
  vec r;
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = (T)x[i];
  __builtin_memcpy(__builtin_assume_aligned(to, sizeof(T) * N < 16 ? sizeof(T) * N : 16), &r, sizeof r);
}
template <typename T, bool kWide>
__device__ __forceinline__ void put8(T* to, const float (&x)[8]) {
  if constexpr (kWide) {
    put<T, 8>(to, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = (T)x[i];
  }
}

// Where a token's keys and values lie: its page's first byte (NULL: it has no
// place) and its place there.
struct Place {
  char* page;
  int place;
  bool row;  // it belongs to a sequence
};
__device__ __forceinline__ Place place_of(const PagedArgs& a, int token, int64_t page_bytes) {
  const int lane = threadIdx.x & 63;
  int seq = -1;
  for (int s0 = 0; s0 < a.seqs + 1; s0 += 64) {
    const int s = s0 + lane;
    const int n = __popcll(__ballot(s <= a.seqs && a.starts[s <= a.seqs ? s : a.seqs] <= token));
    seq += n;
    if (n < 64) break;
  }
  if (seq < 0 || seq >= a.seqs) return {nullptr, 0, false};
  const Chunk c = chunk_of(a, seq);
  const int64_t pos = position_of(a, c, token - c.begin);
  const int page = page_of(a, c.slot, pos);
  return {page < 0 ? nullptr : static_cast<char*>(a.kv) + (int64_t)page * page_bytes,
          (int)(pos & ((1 << a.page_shift) - 1)), true};
}

// A token without a place reads as zeros.
template <typename T, typename TC, bool kWide>
__global__ __launch_bounds__(kReadThreads) void read_kernel(ReadArgs r) {
  const PagedArgs& a = r.p;
  const int token = blockIdx.x;
  const Place at = place_of(a, token, a.page_stride * (int64_t)sizeof(TC));
  if (!at.row) return;
  const int per = a.dim / 8, all = 2 * per * a.kv_heads;
  for (int w = threadIdx.x; w < all; w += kReadThreads) {
    const int k = w >= per * a.kv_heads, u = k ? w - per * a.kv_heads : w, head = u / per, d = u % per * 8;
    const HeadsView& to = k ? r.v : r.k;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (at.page) {
      typedef TC vec __attribute__((ext_vector_type(8)));
      const TC* from = reinterpret_cast<const TC*>(at.page) + at.place * a.token_stride + head * a.head_stride +
                       (k ? a.value_offset : 0) + d;
      vec p;
      __builtin_memcpy(&p, __builtin_assume_aligned(from, 16), sizeof p);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
    }
    put8<T, kWide>(static_cast<T*>(to.d) + token * to.token_stride + head * to.head_stride + d, x);
  }
}

template <typename T, int kBits, bool kWide>
__global__ __launch_bounds__(kReadThreads) void read_quant_kernel(ReadArgs r) {
  const PagedArgs& a = r.p;
  const int token = blockIdx.x;
  const Place at = place_of(a, token, a.page_stride);
  if (!at.row) return;
  const int size = 1 << a.page_shift;
  const QuantShape s = quant_shape(kBits == 8 ? kQ8_0 : kQ4_0, a.dim, size);
  const int planes = plane_count(s.groups);
  const int nk = 4 * s.groups * a.kv_heads, all = nk + 16 * planes * a.kv_heads;
  for (int w = threadIdx.x; w < all; w += kReadThreads) {
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (w < nk) {
      const int head = w / (4 * s.groups), u = w % (4 * s.groups), b = u >> 2, g = u & 3;
      if (at.page) {
        const char* from = at.page + quant_base(s, head, 0);
        const float d = (float)reinterpret_cast<const _Float16*>(from + s.codes)[b * size + at.place];
        uint32_t c[kBits / 4];
        __builtin_memcpy(c, __builtin_assume_aligned(from + at.place * s.row + key_at(s, b, g), kBits), kBits);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = d * (kBits == 8 ? (float)(int)((c[e / 4 * (kBits / 8)] >> (8 * (e & 3))) & 255) - 128.f
                                 : (float)(int)((c[0] >> (4 * nibble_of(e))) & 15) - 8.f);
      }
      put8<T, kWide>(static_cast<T*>(r.k.d) + token * r.k.token_stride + head * r.k.head_stride + 32 * b + 8 * g, x);
    } else {
      const int n = (w - nk) >> 4, i = (w - nk) & 15, head = n / planes;
      const Plane p = plane_of(s.groups, n % planes);
      T* to = static_cast<T*>(r.v.d) + token * r.v.token_stride + head * r.v.head_stride + 32 * p.first + i;
      if (at.page) {
        const char* from = at.page + quant_base(s, head, 1);
        const char* row = from + at.place * s.row + value_at(s, p, i);
        const int bytes = p.wide * kBits / 4;
        uint32_t c[2] = {0, 0};
        if (bytes == 8)
          __builtin_memcpy(c, __builtin_assume_aligned(row, 8), 8);
        else
          c[0] = bytes == 4 ? *reinterpret_cast<const uint32_t*>(row)
                 : bytes == 2 ? *reinterpret_cast<const uint16_t*>(row) : *reinterpret_cast<const uint8_t*>(row);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (b >= p.wide) break;
          const float d = (float)reinterpret_cast<const _Float16*>(from + s.codes)[(p.first + b) * size + at.place];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            x[2 * b + h] = d * (kBits == 8 ? (float)(int)((c[b / 2] >> (16 * (b & 1) + 8 * h)) & 255) - 128.f
                                           : (float)(int)((c[0] >> (8 * b + 4 * h)) & 15) - 8.f);
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (b >= p.wide) break;
        to[32 * b] = (T)x[2 * b];
        to[32 * b + 16] = (T)x[2 * b + 1];
      }
    }
  }
}

template <typename T, bool kWide>
hipError_t read_of(const ReadArgs& a, int cache_type, hipStream_t s) {
  const int n = a.p.tokens;
  switch (cache_type) {
    case kF32: read_kernel<T, float, kWide><<<n, kReadThreads, 0, s>>>(a); break;
    case kF16: read_kernel<T, _Float16, kWide><<<n, kReadThreads, 0, s>>>(a); break;
    case kBF16: read_kernel<T, __bf16, kWide><<<n, kReadThreads, 0, s>>>(a); break;
    case kQ8_0: read_quant_kernel<T, 8, kWide><<<n, kReadThreads, 0, s>>>(a); break;
    default: read_quant_kernel<T, 4, kWide><<<n, kReadThreads, 0, s>>>(a); break;
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
