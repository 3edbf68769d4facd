// nls_beam.hip -- beam search's selection over the beams of a group and the
// vocabulary.
//
//   c(r, v) = s_r + (l_rv - max_r) - ln sum_v exp(l_rv - max_r)
//
// Bound by one read of the logits.  Only a row's `beams` largest logits can be
// among its group's best candidates, so one pass takes everything from a row:
// a workgroup holds 8192 logits in registers (32 KB in flight), takes their
// maximum, the sum of exponentials and the largest ones.  A bound for those
// comes of the lanes' own maxima: the beams-th largest of a wave's 64 is
// reached by that many logits, and few others reach it.  The second launch, a
// workgroup per group, joins the slices' sums in float64 and merges their
// lists in the same way.
#include "nls_beam.h"
#include "nls_primitives.h"
#include "nls_rowsplit.h"

namespace nls {
namespace {

constexpr int kNT = kBeamThreads, kWaves = kNT / kWave;
constexpr int kPer = kBeamSlice / kNT;  // logits of a thread
constexpr int kList = 512;              // logits of a slice that reach the bound, at most
constexpr int kMerge = 1024;            // candidates of a group likewise

typedef float f4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bool takes_part(const BeamArgs& a, int row) {
  return a.scores[row] > -__builtin_inff() && !(a.ended && a.ended[row]);
}

__global__ __launch_bounds__(kNT, 4) void beam_slice_kernel(BeamArgs a) {
  __shared__ float sh_max[kWaves], sh_sum[kWaves];
  __shared__ uint32_t sh_bound[kWaves];
  __shared__ int count;
  __shared__ BeamEntry list[kList];
  __shared__ BeamEntry best[kWaves];
  const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  if (!takes_part(a, row)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float none = -__builtin_inff();
  const float* x = a.logits + (int64_t)row * a.vocab + (int64_t)slice * kBeamSlice;
  const int n = (int)(a.vocab - (int64_t)slice * kBeamSlice < kBeamSlice ? a.vocab - (int64_t)slice * kBeamSlice : kBeamSlice);
  float l[kPer];  // element (k, e) of a thread: logit (k 256 + thread) 4 + e of the slice
#pragma unroll
  for (int k = 0; k < kPer / 4; ++k) {
    const int at = (k * kNT + (int)threadIdx.x) * 4;
    if (n == kBeamSlice || at + 4 <= n) {
      f4v v;
      __builtin_memcpy(&v, x + at, 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) l[4 * k + e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) l[4 * k + e] = at + e < n ? x[at + e] : none;
    }
  }
  float top = none;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    l[j] = fmaxf(l[j], none);  // (NaN: -infinity)
    top = fmaxf(top, l[j]);
  }
  const uint32_t key = top == none ? 0u : f2key(top);
  const uint32_t wave_top = wave_max_u32(key), wave_bound = wave_kth_largest(key, a.beams);
  if (lane == 0) {
    sh_max[wave] = wave_top ? key2f(wave_top) : none;
    sh_bound[wave] = wave_bound;
  }
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  float mx = sh_max[0];
  uint32_t bound = sh_bound[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    mx = fmaxf(mx, sh_max[w]);
    bound = max(bound, sh_bound[w]);
  }
  float sum = 0.f;
  if (mx == __builtin_inff()) {  // those of +infinity, each as much
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += l[j] == mx ? 1.f : 0.f;
  } else if (mx > none) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += expf_estimate(l[j] - mx);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) sh_sum[wave] = sum;
  const float least = bound ? key2f(bound) : none;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (l[j] >= least && l[j] > none) {
      const int at = atomicAdd(&count, 1);
      if (at < kList) list[at] = {l[j], (int32_t)(slice * kBeamSlice + ((j >> 2) * kNT + threadIdx.x) * 4 + (j & 3))};
    }
  __syncthreads();
  const int64_t part = blockIdx.x;
  BeamEntry* out = a.entries + part * a.beams;
  if (threadIdx.x == 0) a.parts[part] = {mx, sh_sum[0] + sh_sum[1] + sh_sum[2] + sh_sum[3]};
  const int m = count;
  if (m <= kList) {
    // a place for each by the number of those before it
    for (int i = threadIdx.x; i < m; i += kNT) {
      const BeamEntry e = list[i];
      int rank = 0;
      for (int j = 0; j < m; ++j) {
        const BeamEntry o = list[j];
        rank += o.l > e.l || (o.l == e.l && o.v < e.v);
      }
      if (rank < a.beams) out[rank] = e;
    }
    for (int i = m + threadIdx.x; i < a.beams; i += kNT) out[i] = {none, -1};
    return;
  }
  // Too many reach the bound (equal ones): one after another, each the first
  // behind the one before it.
  BeamEntry last{__builtin_inff(), -1};
  for (int r = 0; r < a.beams; ++r) {
    BeamEntry e{none, 0x7fffffff};
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int v = slice * kBeamSlice + ((j >> 2) * kNT + threadIdx.x) * 4 + (j & 3);
      const bool behind = l[j] < last.l || (l[j] == last.l && v > last.v);
      if (behind && l[j] > none) argmax_merge(e.l, e.v, l[j], v);
    }
    wave_argmax(e.l, e.v);
    if (lane == 0) best[wave] = e;
    __syncthreads();
    last = best[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) argmax_merge(last.l, last.v, best[w].l, best[w].v);
    if (threadIdx.x == 0) out[r] = last;  // (more than kList of them: there is one each time)
    __syncthreads();
  }
}

// A candidate of a group: what it is worth and beam * 2^32 + v + 1.
struct Candidate {
  double c;
  int64_t at;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  return a.c > b.c || (a.c == b.c && a.at < b.at);
}

__global__ __launch_bounds__(kNT) void beam_merge_kernel(BeamArgs a) {
  __shared__ float s_score[kMaxBeams], s_max[kMaxBeams];
  __shared__ double s_lse[kMaxBeams];
  __shared__ int s_kind[kMaxBeams];  // 0 no candidates, 1 the row's, 2 itself
  __shared__ Candidate s_top[kNT];
  __shared__ Candidate s_bound, s_wave[kWaves];
  __shared__ Candidate list[kMerge];
  __shared__ int count, s_found;
  const int g = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double none = -__builtin_inf();
  for (int b = wave; b < a.beams; b += kWaves) {
    const int row = g * a.beams + b;
    const float score = a.scores[row];
    const bool live = score > -__builtin_inff(), ended = a.ended && a.ended[row];
    float mx = -__builtin_inff();
    double sum = 0.0;
    if (live && !ended) {
      const BeamPart* p = a.parts + (int64_t)row * a.slices;
      for (int s = lane; s < a.slices; s += kWave) mx = fmaxf(mx, p[s].max);
#pragma unroll
      for (int d = 32; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
      if (mx > -__builtin_inff())
        for (int s = lane; s < a.slices; s += kWave) {
          const BeamPart q = p[s];
          sum += q.max == mx ? (double)q.sum : (double)q.sum * exp((double)q.max - (double)mx);
        }
#pragma unroll
      for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    }
    if (lane == 0) {
      s_score[b] = score;
      s_max[b] = mx;
      s_lse[b] = log(sum);
      s_kind[b] = !live ? 0 : ended ? 2 : mx > -__builtin_inff() ? 1 : 0;
    }
  }
  if (threadIdx.x == 0) {
    count = 0;
    s_found = 0;
  }
  __syncthreads();
  const int lists = a.beams * a.slices;
  // entry i of a list, or none
  auto candidate = [&](int which, int i) {
    const int b = which / a.slices, s = which - b * a.slices, kind = s_kind[b];
    if (kind == 1) {
      const BeamEntry e = a.entries[((int64_t)g * lists + which) * a.beams + i];
      if (e.v < 0) return Candidate{none, 0};
      const double x = e.l == s_max[b] ? 0.0 : (double)e.l - (double)s_max[b];
      return Candidate{(x - s_lse[b]) + (double)s_score[b], (int64_t)b << 32 | (uint32_t)(e.v + 1)};
    }
    if (kind == 2 && s == 0 && i == 0) return Candidate{(double)s_score[b], (int64_t)b << 32};
    return Candidate{none, 0};
  };
  // The bound: the beams-th of the threads' best, each of another list or more.
  Candidate mine{none, 0};
  for (int i = threadIdx.x; i < lists; i += kNT) {
    const Candidate c = candidate(i, 0);
    if (c.c > none && (mine.c == none || before(c, mine))) mine = c;
  }
  s_top[threadIdx.x] = mine;
  __syncthreads();
  if (mine.c > none) {
    int rank = 0;
    for (int j = 0; j < kNT; ++j) rank += s_top[j].c > none && before(s_top[j], mine);
    if (rank == a.beams - 1) {
      s_bound = mine;
      s_found = 1;
    }
  }
  __syncthreads();
  const bool bounded = s_found;
  const Candidate bound = s_bound;
  for (int i = threadIdx.x; i < lists; i += kNT)
    for (int k = 0; k < a.beams; ++k) {
      const Candidate c = candidate(i, k);
      if (!(c.c > none) || (bounded && before(bound, c))) break;
      const int at = atomicAdd(&count, 1);
      if (at < kMerge) list[at] = c;
    }
  __syncthreads();
  const int n = count, row0 = g * a.beams;
  auto put = [&](int place, const Candidate& c) {
    const int b = (int)(c.at >> 32), v = (int)(uint32_t)c.at - 1;
    a.parents[row0 + place] = row0 + b;
    a.tokens[row0 + place] = v;
    a.out_scores[row0 + place] = (float)c.c;
    if (a.out_ended) {
      int over = s_kind[b] == 2;
      for (int i = 0; i < a.n_eog; ++i) over |= v >= 0 && v == a.eog[i];
      a.out_ended[row0 + place] = over;
    }
  };
  auto put_none = [&](int place) {
    a.parents[row0 + place] = row0 + place;
    a.tokens[row0 + place] = -1;
    a.out_scores[row0 + place] = -__builtin_inff();
    if (a.out_ended) a.out_ended[row0 + place] = 0;
  };
  if (n <= kMerge) {
    for (int i = threadIdx.x; i < n; i += kNT) {
      const Candidate c = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += before(list[j], c);
      if (rank < a.beams) put(rank, c);
    }
    for (int i = n + threadIdx.x; i < a.beams; i += kNT) put_none(i);
    return;
  }
  // More than the list holds: one after another.
  Candidate last{__builtin_inf(), -1};
  for (int r = 0; r < a.beams; ++r) {
    Candidate c{none, 0};
    for (int i = threadIdx.x; i < lists; i += kNT)
      for (int k = 0; k < a.beams; ++k) {
        const Candidate o = candidate(i, k);
        if (!(o.c > none)) break;
        if (!before(last, o)) continue;
        if (c.c == none || before(o, c)) c = o;
        break;  // (a list is in order)
      }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const Candidate o{__shfl_xor(c.c, d), __shfl_xor(c.at, d)};
      if (o.c > none && (c.c == none || before(o, c))) c = o;
    }
    if (lane == 0) s_wave[wave] = c;
    __syncthreads();
    last = s_wave[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
      if (s_wave[w].c > none && (last.c == none || before(s_wave[w], last))) last = s_wave[w];
    if (threadIdx.x == 0) put(r, last);  // (more than kMerge of them: there is one each time)
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_beam(const BeamArgs& a, hipStream_t s) {
  beam_slice_kernel<<<a.groups * a.beams * a.slices, kNT, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  beam_merge_kernel<<<a.groups, kNT, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace nls
