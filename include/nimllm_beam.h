/*
 * nimllm_beam.h -- C ABI of the MI355X (gfx950) selection of beam search.
 *
 * A group of `beams` contexts follows the most probable continuations of one
 * prompt together.  One step of all groups is
 *
 *   nls_lm_head        logits of all beams                (nimllm_lmhead.h)
 *   nls_beam_select    the best continuations of each group
 *   nls_cache_reorder  every context becomes what its parent was
 *   nls_cache_reserve  room for the new tokens            (nimllm_attention.h)
 *
 * where nls_sample would choose for each context by itself.  Everything stays
 * on the device, ordered on `stream`; nothing here synchronises, allocates or
 * keeps anything between calls, so a step can be captured and replayed.
 *
 * Status codes are nimllm_sampler.h's NLS_* values.
 */
#ifndef NIMLLM_BEAM_H
#define NIMLLM_BEAM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Beam b of group g is row r = g * beams + b.  Its candidates are
 *   (r, v), 0 <= v < vocab, worth scores[r] + ln softmax(logits[r])[v],
 * or, where d_ended is given and ended[r] is not 0, itself alone: (r, -1),
 * worth scores[r].  The `beams` best candidates of a group, in descending
 * order (of equal ones the lowest (r, v) first), become its next beams: for
 * place j of group g, at g * beams + j,
 *   d_parents     the row r it goes on from
 *   d_tokens      its token v, -1 for a beam that had ended
 *   d_out_scores  what it is worth
 *   d_out_ended   1 where the parent had ended, or v is one of d_eog[0 .. n_eog)
 * (NULL: not wanted).  Where a group has fewer candidates than beams, the last
 * places have their own row as parent, token -1, score -infinity and ended 0.
 *
 * A logit of -infinity or NaN is no candidate and has no share in the sum; a
 * row of which nothing is left has none, nor has one whose score is -infinity
 * or NaN (a first step, say, has score 0 for one beam and -infinity for the
 * others).  Logits of +infinity share the probability of their row.
 *
 * A row takes part with its `beams` largest logits (of equal ones the lowest v);
 * where it is read in parts, of 2048 or 8192, with as many of each.  (It shows only
 * where so many unlike logits are worth the same in float64, beside scores 10^15
 * times their difference.)
 * Candidates are compared in float64: the exponentials of a row and the sums
 * of up to 32 of them are fp32, everything after that is float64; scores are
 * rounded once to fp32.  d_out_scores may be d_scores, and d_out_ended d_ended.
 *
 * d_logits: fp32 [groups * beams, vocab].  beams: 1 .. 64; fewer than 2^24 rows,
 * vocab below 2^29.  d_work: nls_beam_workspace() bytes, 256-byte aligned; it
 * needs no preparation and belongs to one call at a time.
 */
size_t nls_beam_workspace(int32_t groups, int32_t beams, int64_t vocab);
int32_t nls_beam_select(const float* d_logits, int32_t groups, int32_t beams, int64_t vocab, const float* d_scores,
                        const int32_t* d_ended, const int32_t* d_eog, int32_t n_eog, int32_t* d_parents,
                        int32_t* d_tokens, float* d_out_scores, int32_t* d_out_ended, void* d_work, size_t work_bytes,
                        void* stream);

#ifdef __cplusplus
}
#endif

#endif
