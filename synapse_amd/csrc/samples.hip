// What samples keep between a round's forward passes: a few integers each.
#include "samples.hpp"

namespace syn {

namespace {

constexpr int kNT = 64;

__global__ void __launch_bounds__(kNT) k_sample_drafted(SampleState st, int step, const uint32_t *token) {
  const int s = threadIdx.x;
  if (s >= st.n) return;
  st.ids[s * (st.k + 1) + step + 1] = token[s];
  st.drafted[s * st.k + step] = token[s];
}

// One workgroup, a thread a sample.
__global__ void __launch_bounds__(kNT)
    k_sample_advance(SampleState st, const uint32_t *token, int width, const int32_t *count) {
  const int s = threadIdx.x, k = st.k, round = *st.round;
  __syncthreads();
  if (s == 0) *st.round = round + 1;
  if (s >= st.n) return;
  int out = st.out[s], len = st.len[s];
  uint32_t last = 0;
  bool ended = st.drafting[s] < 0;
  if (!ended) {
    const int n = count[s];
    len += out ? n : 0;  // (the first token is the prompt's: no position is added)
    for (int i = 0; i < n && !ended; i++) {
      last = token[s * width + i];
      st.history[(size_t)s * st.max_new + out++] = last;
      ended = out >= st.max_new || (st.eos >= 0 && last == (uint32_t)st.eos);
    }
  }
  st.out[s] = out;
  st.len[s] = len;
  st.drafting[s] = ended ? -1 : 0;
  st.drafts[s] = ended ? -1 : k;
  st.room[s] = ended ? 0 : len + k + 1;
  st.last[s] = st.ids[s * (k + 1)] = last;
  for (int j = 0; j <= k; j++) {
    st.pos[s * (k + 1) + j] = ended ? -1 : len + j;
    st.seq[s * (k + 1) + j] = s;
  }
  const float *d = st.draws + st.n + ((size_t)round * st.n + s) * (2 * k + 1);
  for (int i = 0; i < k; i++) {
    st.draft_pos[i * st.n + s] = ended ? -1 : len + i;
    st.draft_len[i * st.n + s] = ended ? 0 : len + i + 1;
    st.u_draft[i * st.n + s] = d[i];
  }
  for (int j = 0; j <= k; j++) st.u[s * (k + 1) + j] = d[k + j];
}

}  // namespace

syn_status_t launch_sample_drafted(const SampleState &st, int step, const uint32_t *token, hipStream_t s) {
  hipLaunchKernelGGL(k_sample_drafted, dim3(1), dim3(kNT), 0, s, st, step, token);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

syn_status_t launch_sample_advance(const SampleState &st, const uint32_t *token, int width,
                                   const int32_t *count, hipStream_t s) {
  hipLaunchKernelGGL(k_sample_advance, dim3(1), dim3(kNT), 0, s, st, token, width, count);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // namespace syn
