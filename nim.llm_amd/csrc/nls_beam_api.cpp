// nls_beam_api.cpp -- host side of the C ABI in include/nimllm_beam.h: the
// arguments' checks and the launches.  Every check comes before any device
// work, and no call keeps anything.
#include <hip/hip_runtime.h>

#include "../../include/nimllm_beam.h"
#include "../../include/nimllm_sampler.h"
#include "nls_beam.h"
#include "nls_internal.h"

using namespace nls;

namespace {

int bad(const char* what) { return api_error(NLS_ERR_INVALID_ARGUMENT, what); }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

const char* check_sizes(int32_t groups, int32_t beams, int64_t vocab) {
  if (groups < 0 || beams < 1 || beams > kMaxBeams) return "beams: groups is negative, or beams not in 1 .. 64";
  if ((int64_t)groups * beams >= 1 << 24) return "beams: 2^24 rows or more";
  if (vocab < 0 || vocab >= int64_t{1} << 29) return "beams: vocab is negative or 2^29 or more";
  // (a launch has fewer than 2^32 threads)
  if ((int64_t)groups * beams * beam_slices((int64_t)groups * beams, vocab) >= 1 << 24) return "beams: rows times vocab is too large";
  return nullptr;
}
size_t align256(size_t n) { return (n + 255) & ~size_t{255}; }
size_t part_bytes(int64_t parts) { return align256(parts * sizeof(BeamPart)); }

}  // namespace

extern "C" {

size_t nls_beam_workspace(int32_t groups, int32_t beams, int64_t vocab) {
  if (check_sizes(groups, beams, vocab)) return 0;
  const int64_t rows = (int64_t)groups * beams, parts = rows * beam_slices(rows, vocab);
  return part_bytes(parts) + align256(parts * beams * sizeof(BeamEntry));
}

int32_t nls_beam_select(const float* d_logits, int32_t groups, int32_t beams, int64_t vocab, const float* d_scores,
                        const int32_t* d_ended, const int32_t* d_eog, int32_t n_eog, int32_t* d_parents,
                        int32_t* d_tokens, float* d_out_scores, int32_t* d_out_ended, void* d_work, size_t work_bytes,
                        void* stream) {
  if (const char* why = check_sizes(groups, beams, vocab)) return bad(why);
  if (n_eog < 0) return bad("beams: n_eog is negative");
  if (groups == 0) return NLS_OK;
  if (vocab == 0) return api_error(NLS_ERR_EMPTY_VOCAB, "beams: an empty vocabulary");
  if (!d_logits || !d_scores || !d_parents || !d_tokens || !d_out_scores || (n_eog > 0 && !d_eog))
    return bad("beams: NULL logits, scores, eog or outputs");
  if (!aligned(d_logits, 4) || !aligned(d_scores, 4) || !aligned(d_ended, 4) || !aligned(d_eog, 4) ||
      !aligned(d_parents, 4) || !aligned(d_tokens, 4) || !aligned(d_out_scores, 4) || !aligned(d_out_ended, 4))
    return bad("beams: misaligned pointers");
  if (!d_work || !aligned(d_work, 256) || work_bytes < nls_beam_workspace(groups, beams, vocab))
    return bad("beams: workspace NULL, misaligned or too small");
  BeamArgs a{};
  a.logits = d_logits;
  a.groups = groups;
  a.beams = beams;
  a.vocab = vocab;
  a.scores = d_scores;
  a.ended = d_ended;
  a.eog = d_eog;
  a.n_eog = n_eog;
  a.parents = d_parents;
  a.tokens = d_tokens;
  a.out_scores = d_out_scores;
  a.out_ended = d_out_ended;
  a.per = beam_per((int64_t)groups * beams, vocab);
  a.slices = (int)beam_slices((int64_t)groups * beams, vocab);
  a.parts = static_cast<BeamPart*>(d_work);
  a.entries = reinterpret_cast<BeamEntry*>(static_cast<char*>(d_work) + part_bytes((int64_t)groups * beams * a.slices));
  const hipError_t e = launch_beam(a, reinterpret_cast<hipStream_t>(stream));
  return e == hipSuccess ? NLS_OK : api_hip_error(e, "nls_beam_select");
}

}  // extern "C"
