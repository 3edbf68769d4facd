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
// lists in the same way.  64 groups of 8 beams over 128256, a fifth of them ended
// (210 MB): 44 us, 4.8 TB/s, and 7 for the second launch (whose bound by ballots and
// lists requested ahead, with fewer instructions a logit in the first, took both from
// 80 to 51).  That is what up to 16 beams cost (16 groups of 16 over 128256: 54 us for
// both).  With more the lists grow long, and are ranked by counting, or pass what LDS
// holds and are taken one after another: 16 groups of 32 272 us, 8 of 48 495, 8 of 64
// 2930, where the logits are read in 56, 42 and 56.
#include "nls_beam.h"
#include "nls_primitives.h"

namespace nls {
namespace {

constexpr int kNT = kBeamThreads, kWaves = kNT / kWave;
constexpr int kList = 512;              // logits of a slice that reach the bound, as held
constexpr int kMerge = 1024;            // candidates of a group likewise

typedef float f4v __attribute__((ext_vector_type(4), aligned(4)));  // (rows may start off 16 bytes)

__device__ __forceinline__ bool takes_part(const BeamArgs& a, int row) {
  return a.scores[row] > -__builtin_inff() && !(a.ended && a.ended[row]);
}

template <int kPer>
__global__ __launch_bounds__(kNT, 4) void beam_slice_kernel(BeamArgs a) {
  constexpr int kSlice = kPer * kNT;
  __shared__ float sh_max[kWaves];
  __shared__ double sh_sum[kWaves];
  __shared__ uint32_t sh_bound[kWaves];
  __shared__ int count;
  __shared__ BeamEntry list[kList];
  __shared__ BeamEntry best[kWaves];
  const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  if (!takes_part(a, row)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float none = -__builtin_inff();
  const float* x = a.logits + (int64_t)row * a.vocab + (int64_t)slice * kSlice;
  const int n = (int)(a.vocab - (int64_t)slice * kSlice < kSlice ? a.vocab - (int64_t)slice * kSlice : kSlice);
  float l[kPer];  // element (k, e) of a thread: logit (k 256 + thread) 4 + e of the slice
#pragma unroll
  for (int k = 0; k < kPer / 4; ++k) {
    const int at = (k * kNT + (int)threadIdx.x) * 4;
    if (n == kSlice || at + 4 <= n) {
      const f4v v = __builtin_nontemporal_load(reinterpret_cast<const f4v*>(x + at));
#pragma unroll
      for (int e = 0; e < 4; ++e) l[4 * k + e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) l[4 * k + e] = at + e < n ? x[at + e] : none;
    }
  }
  float top = none;
#pragma unroll
  for (int j = 0; j < kPer; ++j) top = fmaxf(top, l[j]);  // (NaN is passed over)
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
  // (the largest term is exactly 1; a product rounded once in the exponent of the
  // others is 2^-24 of a number that weighs exp(-it))
  auto term = [&](float v) {
    if (mx == __builtin_inff()) return v == mx ? 1.f : 0.f;  // those of +infinity, each as much
    return __builtin_amdgcn_exp2f((v - mx) * 1.44269504f);
  };
  float sum = 0.f;
  if (mx > none) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += term(l[j]);
    if (__ballot(!(sum < __builtin_inff()))) {  // a NaN among them
      sum = 0.f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) sum += l[j] > none ? term(l[j]) : 0.f;
    }
  }
  double all = sum;
#pragma unroll
  for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d);
  if (lane == 0) sh_sum[wave] = all;
  const float least = bound ? key2f(bound) : none;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (l[j] >= least && l[j] > none) {
      const int at = atomicAdd(&count, 1);
      if (at < kList) list[at] = {l[j], (int32_t)(slice * kSlice + ((j >> 2) * kNT + threadIdx.x) * 4 + (j & 3))};
    }
  __syncthreads();
  const int64_t part = blockIdx.x;
  BeamEntry* out = a.entries + part * a.beams;
  if (threadIdx.x == 0) a.parts[part] = {sh_sum[0] + sh_sum[1] + sh_sum[2] + sh_sum[3], mx};
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
  // Too many reach the bound (equal ones, or nearly as many beams as a wave has
  // lanes, whose least maximum is a low one: two slices of normal logits in a hundred
  // at 56 beams, all at 64): one after another, each the first behind the one before it.
  BeamEntry last{__builtin_inff(), -1};
  for (int r = 0; r < a.beams; ++r) {
    BeamEntry e{none, 0x7fffffff};
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int v = slice * kSlice + ((j >> 2) * kNT + threadIdx.x) * 4 + (j & 3);
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
  __shared__ float s_score[kMaxBeams];
  __shared__ double s_of[kMaxBeams], s_sum[kMaxBeams];  // ln sum exp(l): of + sum
  __shared__ int s_kind[kMaxBeams];  // 0 no candidates, 1 the row's, 2 itself, 3 the row's of +infinity
  __shared__ uint32_t s_bound[kWaves];
  __shared__ Candidate s_wave[kWaves];
  __shared__ Candidate list[kMerge];
  __shared__ int32_t s_eog[kNT];
  __shared__ int count;
  const int g = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double none = -__builtin_inf();
  const int lists = a.beams * a.slices;
  const BeamEntry* entries = a.entries + (int64_t)g * lists * a.beams;
  // (what does not wait for the sums is requested before them)
  constexpr int kHeld = 8;
  BeamEntry held[kHeld];  // of list threadIdx.x
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    held[k] = {-__builtin_inff(), -1};
    if ((int)threadIdx.x < lists && k < a.beams) held[k] = entries[(int64_t)threadIdx.x * a.beams + k];
  }
  if ((int)threadIdx.x < a.n_eog) s_eog[threadIdx.x] = a.eog[threadIdx.x];
  // a row's parts: 16 lanes
  for (int b = threadIdx.x / 16; b < a.beams; b += kNT / 16) {
    const int row = g * a.beams + b, part = threadIdx.x & 15;
    const float score = a.scores[row];
    const bool live = score > -__builtin_inff(), ended = a.ended && a.ended[row];
    const BeamPart* p = a.parts + (int64_t)row * a.slices;
    const BeamPart held_part = p[part < a.slices ? part : 0];
    // the maximum first, so that a part's exponential is one (what is against
    // +infinity stands alone)
    const bool asks = live && !ended;
    float top = asks && part < a.slices ? held_part.max : -__builtin_inff();
    if (asks)
      for (int s = part + 16; s < a.slices; s += 16) top = fmaxf(top, p[s].max);
#pragma unroll
    for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const double of = top;
    auto share = [&](const BeamPart& q) { return q.max == top ? q.sum : q.sum * exp((double)q.max - of); };
    double sum = asks && part < a.slices ? share(held_part) : 0.0;
    if (asks)
      for (int s = part + 16; s < a.slices; s += 16) sum += share(p[s]);
#pragma unroll
    for (int d = 8; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (part == 0) {
      s_score[b] = score;
      s_of[b] = of;
      s_sum[b] = log(sum);
      s_kind[b] = !live ? 0 : ended ? 2 : of == __builtin_inf() ? 3 : of > none ? 1 : 0;
    }
  }
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  // entry i of a list, or none
  auto worth = [&](const BeamEntry& e, int b) {
    const int kind = s_kind[b];
    if (e.v < 0 || (kind == 3 && e.l != __builtin_inff())) return Candidate{none, 0};
    const double x = kind == 3 ? 0.0 : (double)e.l - s_of[b];
    return Candidate{(x - s_sum[b]) + (double)s_score[b], (int64_t)b << 32 | (uint32_t)(e.v + 1)};
  };
  auto candidate = [&](int which, int i) {
    const int b = which / a.slices, s = which - b * a.slices, kind = s_kind[b];
    if (kind & 1) return worth(entries[(int64_t)which * a.beams + i], b);
    if (kind == 2 && s == 0 && i == 0) return Candidate{(double)s_score[b], (int64_t)b << 32};
    return Candidate{none, 0};
  };
  // The bound, as the slices': the beams-th largest of a wave's lanes' best, each
  // of another list or more.  (Its number is rounded down to fp32.)
  auto key_of = [&](const Candidate& c) { return c.c > none ? f2key(__double2float_rd(c.c)) : 0u; };
  uint32_t mine = 0;
  for (int i = threadIdx.x; i < lists; i += kNT) {
    const int b = i / a.slices;
    const uint32_t k = key_of(i < kNT && (s_kind[b] & 1) ? worth(held[0], b) : candidate(i, 0));
    mine = k > mine ? k : mine;
  }
  const uint32_t wave_bound = wave_kth_largest(mine, a.beams);
  if (lane == 0) s_bound[wave] = wave_bound;
  __syncthreads();
  uint32_t bound = s_bound[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) bound = max(bound, s_bound[w]);
  // (a list is in order)
  auto take = [&](const Candidate& c) {
    if (!(c.c > none) || key_of(c) < bound) return false;
    const int at = atomicAdd(&count, 1);
    if (at < kMerge) list[at] = c;
    return true;
  };
  for (int i = threadIdx.x; i < lists; i += kNT) {
    const int b = i / a.slices;
    bool more = true;
    if (i < kNT && (s_kind[b] & 1)) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) more = more && k < a.beams && take(worth(held[k], b));
      for (int k = kHeld; more && k < a.beams; ++k) more = take(candidate(i, k));
    } else {
      for (int k = 0; more && k < a.beams; ++k) more = take(candidate(i, k));
    }
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
      for (int i = 0; i < a.n_eog; ++i) over |= v >= 0 && v == (i < kNT ? s_eog[i] : a.eog[i]);
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
  // More than the list holds (most groups of 48 beams and more): one after another.
  Candidate last{__builtin_inf(), -1};
  for (int r = 0; r < a.beams; ++r) {
    Candidate c{none, 0};
    for (int i = threadIdx.x; i < lists; i += kNT) {
      Candidate first{none, 0};  // of this list, which is in the order of its logits: equal worths may not be
      for (int k = 0; k < a.beams; ++k) {
        const Candidate o = candidate(i, k);
        if (!(o.c > none) || o.c < first.c) break;
        if (before(last, o) && (first.c == none || before(o, first))) first = o;
      }
      if (first.c > none && (c.c == none || before(first, c))) c = first;
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
  if (a.per == kBeamPer)
    beam_slice_kernel<kBeamPer><<<a.groups * a.beams * a.slices, kNT, 0, s>>>(a);
  else
    beam_slice_kernel<kBeamPerFew><<<a.groups * a.beams * a.slices, kNT, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  beam_merge_kernel<<<a.groups, kNT, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace nls
