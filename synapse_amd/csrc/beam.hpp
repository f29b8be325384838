// Device state of a beam search that a decoder runs step by step.
#pragma once

#include "common.hpp"

namespace syn {

// Per beam, all advanced by one a step: the rotation position of the token
// being decoded, its place in the beam's suffix, and the suffix length with it.
struct BeamCounters {
  int32_t *pos, *index, *len, *step;  // step: one, the history's next column
};

// history[b][step] = token[b], then the counters advance
syn_status_t launch_beam_advance(const BeamCounters &c, int n_beams, const uint32_t *token,
                                 uint32_t *history, size_t ld_history, hipStream_t s);

}  // namespace syn
