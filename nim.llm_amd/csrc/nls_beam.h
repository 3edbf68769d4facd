// nls_beam.h -- arguments of the kernels of beam search's selection
// (nls_beam.hip).
#pragma once
#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

namespace nls {

constexpr int kMaxBeams = 64;
constexpr int kBeamThreads = 256;
constexpr int kBeamSlice = 32 * kBeamThreads;  // logits of a workgroup

// The largest logit of a slice, the sum of exp(l - max), and behind them (in
// the workspace) its `beams` largest logits in order.
struct BeamPart {
  float max, sum;
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
  int slices;  // of a row
  BeamPart* parts;
  BeamEntry* entries;
};

inline int beam_slices(int64_t vocab) { return (int)((vocab + kBeamSlice - 1) / kBeamSlice); }
hipError_t launch_beam(const BeamArgs& a, hipStream_t s);

}  // namespace nls
