// Verification of drafted tokens against the target's probabilities, from given
// random numbers, and the token that follows the accepted ones.
//
// With p_i = softmax(target_i / T) and q_i = softmax(draft_i / T), draft x_i is
// accepted when u_i q_i(x_i) < p_i(x_i) and all before it are.  The next token is
// drawn from max(p_r - q_r, 0) where draft r is the first that is not, from p_n
// where all n are: the lowest t whose sum of weights up to t is above u times
// the sum of all.  Accepted and drawn tokens together are distributed as tokens
// drawn from the target one by one.
//
// Precision: a draw's borders between tokens lie as close as a vocabulary's
// probabilities are small, so exponentials and sums are f64 throughout: in f32
// one in a hundred draws over 150000 tokens would fall to a neighbour.
#include <algorithm>

#include "kv_pages.hpp"
#include "wave_ops.hpp"

namespace syn {

namespace {

constexpr int kNT = 256;
constexpr float kNone = -__builtin_huge_valf();
constexpr double kLog2e = 1.44269504088896340736;
constexpr double kLn2 = 0.69314718055994530942;
constexpr uint32_t kMaxDraft = 64;

// of a chunk of a row, or of a row: its largest logit, the first token that has
// it, and the sum of exp((logit - top) / T)
struct Stat {
  double sum;
  float top;
  int at;
};

struct VerifyArgs {
  const float *target, *draft, *heat, *u;
  const uint32_t *token;
  const int32_t *n_draft;
  uint32_t *out;
  int32_t *count;
  float *logp;
  Stat *stat;     // [n_seqs][target rows, then draft rows][chunks]
  double *weight; // [n_seqs][chunks]
  size_t ld_target, target_stride, ld_draft, draft_stride;
  int n_seqs, K, rows, vocab, chunks, per;
  uint32_t pad;
};

// drafts of a sequence; -1: it is left out
__device__ __forceinline__ int drafts_of(const VerifyArgs &a, int s) {
  const int n = a.n_draft ? a.n_draft[s] : a.K;
  return n < 0 ? -1 : min(n, a.K);
}
// log2(e) / T, or 0 for a greedy sequence
__device__ __forceinline__ double scale_of(const VerifyArgs &a, int s) {
  const float t = a.heat ? a.heat[s] : 1.0f;
  return t > 0.0f && t < __builtin_huge_valf() ? kLog2e / (double)t : 0.0;
}
__device__ __forceinline__ const float *row_of(const VerifyArgs &a, int s, int r) {
  return r <= a.K ? a.target + (size_t)s * a.target_stride + (size_t)r * a.ld_target
                  : a.draft + (size_t)s * a.draft_stride + (size_t)(r - a.K - 1) * a.ld_draft;
}

// 2^z for z <= 0, within 2^-40 of itself: z to the nearest whole number and a
// remainder f of at most 1/2, 2^f by the first terms of its series in f ln 2
// (the next, (ln 2 / 2)^12 / 12!, is below 2^-47)
__device__ __forceinline__ double exp2_of(double z) {
  z = fmax(z, -1200.0);
  const double k = rint(z), f = (z - k) * kLn2;
  double y = 1.0 / 39916800;
  y = __builtin_fma(y, f, 1.0 / 3628800);
  y = __builtin_fma(y, f, 1.0 / 362880);
  y = __builtin_fma(y, f, 1.0 / 40320);
  y = __builtin_fma(y, f, 1.0 / 5040);
  y = __builtin_fma(y, f, 1.0 / 720);
  y = __builtin_fma(y, f, 1.0 / 120);
  y = __builtin_fma(y, f, 1.0 / 24);
  y = __builtin_fma(y, f, 1.0 / 6);
  y = __builtin_fma(y, f, 0.5);
  y = __builtin_fma(y, f, 1.0);
  y = __builtin_fma(y, f, 1.0);
  return __builtin_ldexp(y, (int)k);
}
// exp((x - top) / T); a top of +inf shares among the infinities, one of -inf
// leaves nothing
__device__ __forceinline__ double term(float x, float top, double c) {
  if (fabsf(top) == __builtin_huge_valf()) return x == top && top > 0.0f ? 1.0 : 0.0;
  return exp2_of(((double)x - (double)top) * c);
}
__device__ __forceinline__ float logit(float x) { return fmaxf(x, kNone); }  // NaN: -inf

// (top, at) with the largest top, the lowest at
__device__ __forceinline__ void first_top(float *top, int *at) {
  for (int o = 32; o > 0; o >>= 1) {
    const float t = __shfl_xor(*top, o);
    const int i = __shfl_xor(*at, o);
    if (t > *top || (t == *top && i < *at)) *top = t, *at = i;
  }
}

// grid (chunk, sequence and row): the statistics of a chunk of a row.
__global__ void __launch_bounds__(kNT) k_verify_rows(VerifyArgs a) {
  __shared__ float wtop[4];
  __shared__ int wat[4];
  __shared__ double wsum[4];
  const int s = blockIdx.y / a.rows, r = blockIdx.y - s * a.rows, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, n = drafts_of(a, s);
  const double c = scale_of(a, s);
  const bool is_draft = r > a.K;
  if (is_draft ? r - a.K - 1 >= n || c == 0.0 : r > n) return;
  const int first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
  const float *x = row_of(a, s, r);
  float top = kNone;
  int at = 0x7fffffff;
  for (int t = first + tid; t < end; t += kNT) {
    const float v = logit(x[t]);
    if (v > top) top = v, at = t;
  }
  first_top(&top, &at);
  if (lane == 0) wtop[wave] = top, wat[wave] = at;
  __syncthreads();
  top = wtop[0], at = wat[0];
  for (int w = 1; w < 4; w++)
    if (wtop[w] > top || (wtop[w] == top && wat[w] < at)) top = wtop[w], at = wat[w];
  double sum = 0.0;
  if (c != 0.0)
    for (int t = first + tid; t < end; t += kNT) sum += term(logit(x[t]), top, c);
  sum = wave_sum(sum);
  if (lane == 0) wsum[wave] = sum;
  __syncthreads();
  if (tid == 0)
    a.stat[(size_t)blockIdx.y * a.chunks + blockIdx.x] =
        Stat{(wsum[0] + wsum[1]) + (wsum[2] + wsum[3]), top, at};
}

// A wave joins the chunks of a row.
__device__ __forceinline__ Stat join(const VerifyArgs &a, int s, int r, double c) {
  const Stat *st = a.stat + ((size_t)s * a.rows + r) * a.chunks;
  const int lane = threadIdx.x & 63;
  float top = kNone;
  int at = 0x7fffffff;
  for (int i = lane; i < a.chunks; i += 64) {
    const Stat q = st[i];
    if (q.top > top) top = q.top, at = q.at;
  }
  first_top(&top, &at);
  double sum = 0.0;
  for (int i = lane; i < a.chunks; i += 64) {
    const Stat q = st[i];
    sum += q.sum * term(q.top, top, c);
  }
  return Stat{wave_sum(sum), top, at};
}

// What is decided of a sequence: drafts accepted, and the rows' statistics.
struct Choice {
  int n, r;
  bool greedy;
  double c;
  Stat row[kMaxDraft + 1], of[kMaxDraft];  // target rows, draft rows
  bool fine[kMaxDraft];
};

// The workgroup decides on the drafts of a sequence.
__device__ __forceinline__ void decide(const VerifyArgs &a, int s, int n, Choice *d) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double c = scale_of(a, s);
  for (int i = wave; i <= n; i += kNT / 64) {
    const Stat p = join(a, s, i, c);
    if (lane == 0) d->row[i] = p;
    if (i == n) break;
    const uint32_t t = a.token[(size_t)s * a.K + i];
    bool fine = false;
    Stat q{1.0, 0.0f, 0};
    if (c == 0.0) {
      fine = p.top > kNone && t == (uint32_t)p.at;
    } else {
      if (a.draft) q = join(a, s, a.K + 1 + i, c);
      if (t < (uint32_t)a.vocab && p.sum > 0.0) {
        const double pt = term(logit(row_of(a, s, i)[t]), p.top, c) / p.sum;
        double qt = 1.0;
        if (a.draft) qt = q.sum > 0.0 ? term(logit(row_of(a, s, a.K + 1 + i)[t]), q.top, c) / q.sum : 0.0;
        fine = (double)a.u[(size_t)s * (a.K + 1) + i] * qt < pt;
      }
    }
    if (lane == 0) d->of[i] = q, d->fine[i] = fine;
  }
  __syncthreads();
  int r = 0;
  while (r < n && d->fine[r]) r++;
  if (threadIdx.x == 0) d->n = n, d->r = r, d->c = c, d->greedy = c == 0.0;
  __syncthreads();
}

// the weight of token t after r accepted drafts; plain: of p_r alone
struct Weights {
  const float *x, *y;
  Stat p, q;
  double c;
  uint32_t except;  // a draft that was certain
  __device__ __forceinline__ double of(int t, bool plain) const {
    const double w = term(logit(x[t]), p.top, c) / p.sum;
    if (plain) return w;
    if (!y) return (uint32_t)t == except ? 0.0 : w;
    return fmax(w - (q.sum > 0.0 ? term(logit(y[t]), q.top, c) / q.sum : 0.0), 0.0);
  }
};
__device__ __forceinline__ Weights weights_of(const VerifyArgs &a, int s, const Choice &d, bool *plain) {
  const int r = d.r;
  *plain = r == d.n;
  Weights w{row_of(a, s, r), nullptr, d.row[r], Stat{}, d.c, 0};
  if (!*plain) {
    w.except = a.token[(size_t)s * a.K + r];
    w.q = d.of[r];
    if (a.draft) w.y = row_of(a, s, a.K + 1 + r);
  }
  return w;
}

// grid (chunk, sequence): the sums of the weights
__global__ void __launch_bounds__(kNT) k_verify_weights(VerifyArgs a) {
  __shared__ Choice d;
  __shared__ double wsum[4];
  const int s = blockIdx.y, n = drafts_of(a, s), tid = threadIdx.x;
  if (n < 0 || scale_of(a, s) == 0.0) return;
  decide(a, s, n, &d);
  bool plain;
  const Weights w = weights_of(a, s, d, &plain);
  const int first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
  double sum = 0.0;
  if (w.p.sum > 0.0)
    for (int t = first + tid; t < end; t += kNT) sum += w.of(t, plain);
  sum = wave_sum(sum);
  if ((tid & 63) == 0) wsum[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) a.weight[(size_t)s * a.chunks + blockIdx.x] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
}

// The first token of [first, end) whose weights up to it, and `before`, are above
// `border`; where rounding leaves none, the last one that has a weight.
__device__ __forceinline__ int pick(const Weights &w, bool plain, int first, int end, double before,
                                    double border) {
  __shared__ double wsum[4];
  __shared__ int found, last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int each = (end - first + kNT - 1) / kNT;  // a thread's tokens, next to each other
  const int t0 = first + tid * each, t1 = min(end, t0 + each);
  __syncthreads();
  if (tid == 0) found = 0x7fffffff, last = -1;
  double sum = 0.0;
  int mine = -1;
  for (int t = t0; t < t1; t++) {
    const double x = w.of(t, plain);
    sum += x;
    if (x > 0.0) mine = t;
  }
  double base = wave_before(sum);
  if (lane == 63) wsum[wave] = base + sum;
  __syncthreads();
  for (int i = 0; i < wave; i++) base += wsum[i];
  base += before;
  if (mine >= 0) atomicMax(&last, mine);
  if (base + sum > border) {
    double x = base;
    for (int t = t0; t < t1; t++) {
      const double v = w.of(t, plain);
      x += v;
      if (x > border && v > 0.0) {
        atomicMin(&found, t);
        break;
      }
    }
  }
  __syncthreads();
  return found < 0x7fffffff ? found : last;
}

// one workgroup a sequence: the token, and what is told of all
__global__ void __launch_bounds__(kNT) k_verify_pick(VerifyArgs a) {
  __shared__ Choice d;
  const int s = blockIdx.x, n = drafts_of(a, s), tid = threadIdx.x;
  uint32_t *out = a.out + (size_t)s * (a.K + 1);
  float *logp = a.logp ? a.logp + (size_t)s * (a.K + 1) : nullptr;
  if (n < 0) {
    for (int i = tid; i <= a.K; i += kNT) {
      out[i] = a.pad;
      if (logp) logp[i] = 0.0f;
    }
    if (tid == 0) a.count[s] = 0;
    return;
  }
  decide(a, s, n, &d);
  const int r = d.r;
  const Stat p = d.row[r];
  int t = -1;
  if (d.greedy) {
    t = p.top > kNone ? p.at : -1;
  } else if (p.sum > 0.0) {
    bool plain;
    const Weights w = weights_of(a, s, d, &plain);
    const double *sums = a.weight + (size_t)s * a.chunks;
    double total = 0.0;
    for (int i = 0; i < a.chunks; i++) total += sums[i];
    const double u = (double)a.u[(size_t)s * (a.K + 1) + a.K];
    if (total > 0.0) {
      const double border = u * total;
      double before = 0.0, x = 0.0;
      int at = -1;
      for (int i = 0; i < a.chunks && !(at >= 0 && x > border); i++)
        if (sums[i] > 0.0) at = i, before = x, x += sums[i];
      t = pick(w, plain, at * a.per, min(a.vocab, (at + 1) * a.per), before, border);
    } else {  // p_r is nowhere above q_r: from p_r
      t = pick(w, true, 0, a.vocab, 0.0, u);
    }
  }
  for (int i = tid; i <= a.K; i += kNT) {
    const bool drafted = i < r;
    const uint32_t x = drafted ? a.token[(size_t)s * a.K + i] : (i == r && t >= 0 ? (uint32_t)t : a.pad);
    out[i] = x;
    if (logp) {
      double l = 0.0;
      if (i == r && t < 0)
        l = -__builtin_huge_val();
      else if (i <= r && !d.greedy)
        l = log(term(logit(row_of(a, s, i)[x]), d.row[i].top, d.c) / d.row[i].sum);
      logp[i] = (float)l;
    }
  }
  if (tid == 0) a.count[s] = r + 1;
}

// ---------------------------------------------------------------- host
struct Space {
  int per, chunks, rows;
  size_t stat, weight, total;
};
Space space_of(const syn_hip_draft_verify_params &p) {
  Space s;
  s.rows = 2 * (int)p.max_draft + 1;
  s.per = 8192;
  s.chunks = (int)cdiv(p.vocab, s.per);
  s.stat = 0;
  s.weight = (size_t)p.n_seqs * s.rows * s.chunks * sizeof(Stat);
  s.total = s.weight + round_up((size_t)p.n_seqs * s.chunks * 8, 16);
  return s;
}

syn_status_t check(const syn_hip_draft_verify_params *p) {
  if (!p) return SYN_ERR_NULL_PTR;
  if (p->max_draft > kMaxDraft || !p->vocab || p->vocab > 0x7ff00000u ||
      (uint64_t)p->n_seqs * (2 * p->max_draft + 1) > 65535u) {
    set_error("draft_verify: at most 64 drafts, 2^31 - 2^20 tokens, 65535 rows of target and draft");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->ld_target < p->vocab || (p->max_draft && p->ld_draft && p->ld_draft < p->vocab)) {
    set_error("draft_verify: rows of logits shorter than the vocabulary");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  return SYN_OK;
}

}  // namespace

}  // namespace syn

using namespace syn;

extern "C" {

syn_status_t syn_hip_draft_verify_workspace(const syn_hip_draft_verify_params *p, size_t *bytes) {
  if (!bytes) return SYN_ERR_NULL_PTR;
  SYN_TRY(check(p));
  *bytes = space_of(*p).total;
  return SYN_OK;
}

syn_status_t syn_hip_draft_verify(const syn_hip_draft_verify_params *p, const float *d_target,
                                  const float *d_draft, const uint32_t *d_drafted,
                                  const int32_t *d_n_draft, const float *d_temperature,
                                  const float *d_u, uint32_t *d_token, int32_t *d_count, float *d_logp,
                                  void *d_workspace, size_t workspace_bytes, void *stream) {
  SYN_TRY(check(p));
  if (p->n_seqs == 0) return SYN_OK;
  if (!d_target || !d_u || !d_token || !d_count || (p->max_draft && !d_drafted) || !d_workspace)
    return SYN_ERR_NULL_PTR;
  if (p->max_draft && d_draft && p->ld_draft < p->vocab) {
    set_error("draft_verify: rows of logits shorter than the vocabulary");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  if (d_token == d_drafted) {
    set_error("draft_verify: d_token is apart from d_drafted");
    return SYN_ERR_INVALID_ARG;
  }
  const Space sp = space_of(*p);
  if (!aligned16(d_workspace) || workspace_bytes < sp.total) {
    set_error("draft_verify: workspace unaligned or too small");
    return SYN_ERR_INVALID_ARG;
  }
  SYN_TRY(ensure_init());
  uint8_t *ws = static_cast<uint8_t *>(d_workspace);
  VerifyArgs a{};
  a.target = d_target;
  a.draft = p->max_draft ? d_draft : nullptr;
  a.heat = d_temperature;
  a.u = d_u;
  a.token = d_drafted;
  a.n_draft = d_n_draft;
  a.out = d_token;
  a.count = d_count;
  a.logp = d_logp;
  a.stat = reinterpret_cast<Stat *>(ws + sp.stat);
  a.weight = reinterpret_cast<double *>(ws + sp.weight);
  a.ld_target = p->ld_target;
  a.target_stride = p->target_stride;
  a.ld_draft = p->ld_draft;
  a.draft_stride = p->draft_stride;
  a.n_seqs = (int)p->n_seqs;
  a.K = (int)p->max_draft;
  a.rows = a.draft ? sp.rows : a.K + 1;
  a.vocab = (int)p->vocab;
  a.chunks = sp.chunks;
  a.per = sp.per;
  a.pad = p->pad;
  hipStream_t s = pick_stream(stream);
  hipLaunchKernelGGL(k_verify_rows, dim3(a.chunks, p->n_seqs * a.rows), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_verify_weights, dim3(a.chunks, p->n_seqs), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_verify_pick, dim3(p->n_seqs), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // extern "C"
