// nls_beam.h -- arguments of the kernels of beam search's selection
// (nls_beam.hip).
#pragma once
#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

namespace nls {

constexpr int kMaxBeams = 64;
constexpr int kBeamThreads = 256;
constexpr int kBeamPer = 32, kBeamPerFew = 8;  // logits of a thread

// The largest logit of a slice, the sum of exp(l - max), and behind the parts (in
// the workspace) its `beams` largest logits in order.
struct BeamPart {
  double sum;
  float max;
};
struct BeamEntry {
  float l;
  int32_t v;  // -1: none
};

struct BeamArgs {
  const float* logits;
  int groups, beams;
  int64_t vocab;
  const float* scores;
  const int32_t* ended;
  const int32_t* eog;
  int n_eog;
  int32_t *parents, *tokens;
  float* out_scores;
  int32_t* out_ended;
  int per, slices;  // logits of a thread, slices of a row
  BeamPart* parts;
  BeamEntry* entries;
};

// 32 logits to a thread, 32 KB on their way to each workgroup; 8 where that leaves
// less than a workgroup for a CU (4 x 32000: 7.0 us with 32, 5.6 with 8).
inline int beam_per(int64_t rows, int64_t vocab) {
  const int64_t slice = (int64_t)kBeamPer * kBeamThreads;
  return rows * ((vocab + slice - 1) / slice) < 256 ? kBeamPerFew : kBeamPer;
}
inline int64_t beam_slices(int64_t rows, int64_t vocab) {
  const int64_t slice = (int64_t)beam_per(rows, vocab) * kBeamThreads;
  return (vocab + slice - 1) / slice;
}
hipError_t launch_beam(const BeamArgs& a, hipStream_t s);

}  // namespace nls
