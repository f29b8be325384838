// Device state of samples that a decoder draws with drafts, round by round.
#pragma once

#include "common.hpp"

namespace syn {

// n samples with k drafts a round.  A round decodes, for each sample, the token
// drawn last and its drafts, at positions len .. len + k of its sequence.
struct SampleState {
  int n, k, eos, max_new;
  int32_t *round;     // one: rounds done, column of the draws
  int32_t *len;       // [n] positions in the cache, the last token's not among them
  int32_t *out;       // [n] tokens drawn
  int32_t *drafting;  // [n] 0, or -1 for a sample that has ended
  int32_t *drafts;    // [n] k, or -1
  int32_t *room;      // [n] positions of a round: len + k + 1, or 0
  int32_t *pos, *seq;  // [n][k + 1] place and sample of a round's tokens (pos -1: ended)
  int32_t *draft_pos, *draft_len;  // [k][n] place and length of a draft step's tokens
  uint32_t *last;     // [n] the token drawn last
  uint32_t *ids;      // [n][k + 1] a round's tokens
  uint32_t *drafted;  // [n][k]
  uint32_t *history;  // [n][max_new]
  const float *draws; // n, then [max_new][n][2 k + 1]
  float *u_draft, *u;  // [k][n], [n][k + 1]: this round's
};

// ids and drafted take draft `step` of every sample
syn_status_t launch_sample_drafted(const SampleState &st, int step, const uint32_t *token, hipStream_t s);
// the tokens of a verification [n][width], count of them each, into the history;
// then everything is that of the next round
syn_status_t launch_sample_advance(const SampleState &st, const uint32_t *token, int width,
                                   const int32_t *count, hipStream_t s);

}  // namespace syn
