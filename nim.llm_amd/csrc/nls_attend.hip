// nls_attend.hip -- attention of chunks of new tokens over the paged cache.
//
// One wave per (token, head): each lane holds up to four of the head's
// elements, keys pass one at a time with the running maximum and sum of the
// softmax.
#include "nls_paged.h"

namespace nls {
namespace {

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

template <typename T, typename TC>
__global__ __launch_bounds__(64) void attend_kernel(AttendArgs a) {
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  int seq = -1;
  for (int s0 = 0; s0 < a.p.seqs + 1; s0 += 64) {
    const int s = s0 + lane;
    const int n = __popcll(__ballot(s <= a.p.seqs && a.p.starts[s <= a.p.seqs ? s : a.p.seqs] <= token));
    seq += n;
    if (n < 64) break;
  }
  if (seq < 0 || seq >= a.p.seqs) return;
  const Chunk c = chunk_of(a.p, seq);
  const int64_t pos = position_of(a.p, c, token - c.begin);
  int64_t lo = a.first && c.slot >= 0 ? a.first[c.slot] : 0, hi = pos + 1 < c.len ? pos + 1 : c.len;
  if (lo < 0) lo = 0;
  if (a.window > 0 && pos + 1 - a.window > lo) lo = pos + 1 - a.window;
  const T* q = static_cast<const T*>(a.q.d) + token * a.q.token_stride + head * a.q.head_stride;
  float x[4], o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = lane + 64 * i < a.p.dim ? (float)q[lane + 64 * i] : 0.f;
  float m = -__builtin_inff(), l = 0;
  for (int64_t j = lo; j < hi; ++j) {
    const int page = page_of(a.p, c.slot, j);
    if (page < 0) continue;
    const TC* k = static_cast<const TC*>(a.p.kv) + token_offset(a.p, page, j) + head / a.group * a.p.head_stride;
    const TC* v = k + a.p.value_offset;
    float s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.p.dim) s += x[i] * (float)k[lane + 64 * i];
    s = wave_sum(s) * a.scale;
    if (s == -__builtin_inff()) continue;
    const float top = fmaxf(m, s), f = expf(m - top), w = expf(s - top);
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.p.dim) o[i] = o[i] * f + w * (float)v[lane + 64 * i];
    m = top;
  }
  T* out = static_cast<T*>(a.out.d) + token * a.out.token_stride + head * a.out.head_stride;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.p.dim) out[lane + 64 * i] = (T)(l != 0 ? o[i] / l : 0.f);
  if (a.lse && lane == 0) a.lse[(int64_t)token * a.heads + head] = l != 0 ? m + logf(l) : -__builtin_inff();
}

template <typename T, typename TC>
hipError_t attend_of(const AttendArgs& a, hipStream_t s) {
  attend_kernel<T, TC><<<dim3(a.p.tokens, a.heads), 64, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

size_t attend_workspace(const AttendArgs&, int, int64_t) { return 0; }

hipError_t launch_attend(const AttendArgs& a, int type, int cache_type, int, int64_t, void*, hipStream_t s) {
  if (type == kF32) {
    if (cache_type == kF32) return attend_of<float, float>(a, s);
    if (cache_type == kF16) return attend_of<float, _Float16>(a, s);
    return attend_of<float, __bf16>(a, s);
  }
  if (type == kF16) return attend_of<_Float16, _Float16>(a, s);
  return attend_of<__bf16, __bf16>(a, s);
}

}  // namespace nls
