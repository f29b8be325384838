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
constexpr int kBlock = 8 * kNT;  // tokens that a workgroup has in registers at a time
constexpr float kNone = -__builtin_huge_valf();
constexpr double kLog2e = 1.44269504088896340736;
constexpr uint32_t kMaxDraft = 64;

// Of a chunk of a row, or of a row: the sum of exp((logit - ref) / T), ref being
// one of its larger logits, and of a greedy sequence's the first largest one.  A
// ref of +inf: how many logits are; of -inf: there is none above.
struct Stat {
  double sum;
  float ref;
  int at;
};

struct VerifyArgs {
  const float *target, *draft, *heat, *u;
  const uint32_t *token;
  const int32_t *n_draft;
  uint32_t *out;
  int32_t *count;
  float *logp;
  Stat *stat;      // [n_seqs][target rows, then draft rows][chunks]
  double *weight;  // [n_seqs][chunks]
  int32_t *done;   // [n_seqs] chunks whose weights are summed
  size_t ld_target, target_stride, ld_draft, draft_stride;
  int n_seqs, K, rows, vocab, chunks, per;
  uint32_t pad;
};

// drafts of a sequence; -1: it is left out
__device__ __forceinline__ int drafts_of(const VerifyArgs &a, int s) {
  const int n = a.n_draft ? a.n_draft[s] : a.K;
  return n < 0 ? -1 : min(n, a.K);
}
// 32 log2(e) / T, or 0 for a greedy sequence
__device__ __forceinline__ double scale_of(const VerifyArgs &a, int s) {
  const float t = a.heat ? a.heat[s] : 1.0f;
  return t > 0.0f && t < __builtin_huge_valf() ? 32.0 * kLog2e / (double)t : 0.0;
}
__device__ __forceinline__ const float *row_of(const VerifyArgs &a, int s, int r) {
  return r <= a.K ? a.target + (size_t)s * a.target_stride + (size_t)r * a.ld_target
                  : a.draft + (size_t)s * a.draft_stride + (size_t)(r - a.K - 1) * a.ld_draft;
}

// exp((x - ref) / T) in f64, within 2^-43 of itself: with y = (x - ref) 32 log2(e) / T
// = k + f, |f| <= 1/2, it is 2^(k / 32), 32 values of which are in a table (in LDS,
// where 64 banks hold it whole: no two lanes conflict), times 2^(f / 32).  Of that
// the series in f ln 2 / 32 up to the fourth power, the fifth replaced by what it
// leaves of lower powers (Chebyshev's economization: a sixteenth of its error).
struct Exps {
  double ref, c32, least;  // what is 2^-1000 of the whole counts as nothing
  __device__ __forceinline__ Exps(float ref_, double c32_) : ref(ref_), c32(c32_), least(-32000.0 / c32_) {}
  // how far above ref a logit may be: 2^400 (finite, so that +inf is above it)
  __device__ __forceinline__ float limit() const { return fminf((float)(ref + 12800.0 / c32), 3.402823466e38f); }
  // of d = x - ref, 2^-1000 where that is less (or x NaN)
  __device__ __forceinline__ double at(double d, const uint64_t *tab) const {
    const double kShift = 0x1.8p+52;
    d = fmax(d, least);
    double kd = __builtin_fma(d, c32, kShift);
    const uint32_t k = (uint32_t)__double_as_longlong(kd);
    kd -= kShift;
    const double f = __builtin_fma(d, c32, -kd);
    double y = 0x1.3b2ab6fba4e77p-27;
    y = __builtin_fma(y, f, 0x1.c6b167e549176p-20);
    y = __builtin_fma(y, f, 0x1.ebfbdff82c58ep-13);
    y = __builtin_fma(y, f, 0x1.62e42fef6d01bp-6);
    y = __builtin_fma(y, f, 1.0);
    const uint64_t t = tab[k & 31u] + ((uint64_t)k << 47);
    return y * __longlong_as_double((long long)t);
  }
  __device__ __forceinline__ double at_least(float x, const uint64_t *tab) const {
    return at((double)x - ref, tab);
  }
  __device__ __forceinline__ double of(float x, const uint64_t *tab) const {
    if (ref == __builtin_huge_val()) return x == __builtin_huge_valf() ? 1.0 : 0.0;
    const double d = (double)x - ref, y = at(d, tab);
    return d >= least ? y : 0.0;
  }
};
__device__ __forceinline__ void copy_table(uint64_t *tab) {
  if (threadIdx.x < 32) tab[threadIdx.x] = syn_exp2_tab[threadIdx.x];
}

// A workgroup's block of a row: element 4 h + j of thread t is token 1024 h + 4 t
// + j; -inf behind the end.
__device__ __forceinline__ void load_block(const float *x, int left, float *v) {
  // (a 16-byte load needs 4-byte alignment only)
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
  const int t = threadIdx.x * 4;
  if (left >= kBlock) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const f32x4u y = *reinterpret_cast<const f32x4u *>(x + h * (kBlock / 2) + t);
#pragma unroll
      for (int j = 0; j < 4; j++) v[4 * h + j] = y[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = x[min(i / 4 * (kBlock / 2) + t + i % 4, left - 1)];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i / 4 * (kBlock / 2) + t + i % 4 < left ? v[i] : kNone;
  }
}
// fn(first token of the block, values) for the blocks of [0, n), the next one's
// loads ahead
template <class F> __device__ __forceinline__ void over_blocks(const float *x, int n, F fn) {
  float next[8], v[8];
  load_block(x, n, next);
  for (int b = 0; b < n; b += kBlock) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = next[i];
    if (b + kBlock < n) load_block(x + b + kBlock, n - b - kBlock, next);
    fn(b, v);
  }
}

// (top, at) with the largest top, the lowest at
__device__ __forceinline__ void first_top(float *top, int *at) {
  for (int o = 32; o > 0; o >>= 1) {
    const float t = __shfl_xor(*top, o);
    const int i = __shfl_xor(*at, o);
    if (t > *top || (t == *top && i < *at)) *top = t, *at = i;
  }
}

// grid (chunk, sequence and row): the statistics of a chunk of a row, in one pass:
// each wave's sum is relative to the largest logit of its first block that has
// one, until one is 2^400 above that.
__global__ void __launch_bounds__(kNT) k_verify_rows(VerifyArgs a) {
  __shared__ uint64_t tab[32];
  __shared__ Stat part[4];
  const int s = blockIdx.y / a.rows, r = blockIdx.y - s * a.rows, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, n = drafts_of(a, s);
  const double c32 = scale_of(a, s);
  if (r == 0 && blockIdx.x == 0 && tid == 0) a.done[s] = 0;
  if (r > a.K ? r - a.K - 1 >= n || c32 == 0.0 : r > n) return;
  const int first = blockIdx.x * a.per, left = min(a.per, a.vocab - first);
  const float *x = row_of(a, s, r) + first;
  copy_table(tab);
  __syncthreads();
  Stat mine{0.0, kNone, 0x7fffffff};
  if (c32 == 0.0) {
    over_blocks(x, left, [&](int b, const float *v) {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (v[i] > mine.ref) mine.ref = v[i], mine.at = first + b + i / 4 * (kBlock / 2) + tid * 4 + i % 4;
    });
    first_top(&mine.ref, &mine.at);
  } else {
    Exps e(0.0f, c32);
    float limit = kNone;
    double sum = 0.0;
    bool above = false;  // +inf
    over_blocks(x, left, [&](int, const float *v) {
      float top = kNone;
#pragma unroll
      for (int i = 0; i < 8; i++) top = fmaxf(top, v[i]);
      if (__any(top > limit) && !above) {
        top = wave_max(top);
        above = top == __builtin_huge_valf();
        if (above) return;
        const Exps to(top, c32);
        sum = mine.ref == kNone ? 0.0 : sum * to.at_least(mine.ref, tab);
        e = to;
        mine.ref = top;
        limit = e.limit();
      }
      if (mine.ref == kNone || above) return;
#pragma unroll
      for (int i = 0; i < 8; i++) sum += e.at_least(v[i], tab);
    });
    if (__any(above)) {
      sum = 0.0;
      mine.ref = __builtin_huge_valf();
      over_blocks(x, left, [&](int, const float *v) {
#pragma unroll
        for (int i = 0; i < 8; i++) sum += v[i] == mine.ref ? 1.0 : 0.0;
      });
    }
    mine.sum = wave_sum(sum);
  }
  if (lane == 0) part[wave] = mine;
  __syncthreads();
  if (tid) return;
  Stat all = part[0];
  for (int w = 1; w < 4; w++)
    if (part[w].ref > all.ref || (part[w].ref == all.ref && part[w].at < all.at)) all = part[w];
  if (c32 != 0.0) {
    const Exps e(all.ref, c32);
    all.sum = 0.0;
    for (int w = 0; w < 4; w++)
      if (part[w].ref > kNone) all.sum += part[w].sum * e.of(part[w].ref, tab);
  }
  a.stat[(size_t)blockIdx.y * a.chunks + blockIdx.x] = all;
}

// A wave joins the chunks of a row.
__device__ __forceinline__ Stat join(const VerifyArgs &a, int s, int r, double c32, const uint64_t *tab) {
  const Stat *st = a.stat + ((size_t)s * a.rows + r) * a.chunks;
  const int lane = threadIdx.x & 63;
  const Stat q0 = st[min(lane, a.chunks - 1)];
  Stat all{0.0, kNone, 0x7fffffff};
  for (int i = lane; i < a.chunks; i += 64) {
    const Stat q = i == lane ? q0 : st[i];
    if (q.ref > all.ref) all.ref = q.ref, all.at = q.at;
  }
  if (c32 == 0.0) {
    first_top(&all.ref, &all.at);
    return all;
  }
  all.ref = wave_max(all.ref);
  const Exps e(all.ref, c32);
  for (int i = lane; i < a.chunks; i += 64) {
    const Stat q = i == lane ? q0 : st[i];
    if (q.ref > kNone) all.sum += q.sum * e.of(q.ref, tab);
  }
  all.sum = wave_sum(all.sum);
  return all;
}

// What is decided of a sequence: drafts accepted, and the rows' statistics.
struct Choice {
  Stat row[kMaxDraft + 1], of[kMaxDraft];  // target rows, draft rows
  double p[kMaxDraft];                     // of the drafts
  int fine[kMaxDraft];
};

// The workgroup decides on the n drafts of a sequence: how many are accepted.
__device__ __forceinline__ int decide(const VerifyArgs &a, int s, int n, double c32, const uint64_t *tab,
                                      Choice *d) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = wave; i <= n; i += kNT / 64) {
    const bool last = i == n, drafted = !last && a.draft && c32 != 0.0;
    const uint32_t t = last ? 0xffffffffu : a.token[(size_t)s * a.K + i];
    const bool known = t < (uint32_t)a.vocab;
    // (asked for ahead of the sums)
    const float lp = known ? row_of(a, s, i)[t] : kNone;
    const float lq = known && drafted ? row_of(a, s, a.K + 1 + i)[t] : kNone;
    const float u = last ? 0.0f : a.u[(size_t)s * (a.K + 1) + i];
    const Stat p = join(a, s, i, c32, tab);
    Stat q{0.0, kNone, 0};
    if (drafted) q = join(a, s, a.K + 1 + i, c32, tab);
    double pt = 0.0, qt = known && !a.draft ? 1.0 : 0.0;
    bool fine;
    if (c32 == 0.0) {
      fine = p.ref > kNone && t == (uint32_t)p.at;
      pt = 1.0;
    } else {
      if (p.sum > 0.0) pt = Exps(p.ref, c32).of(lp, tab) / p.sum;
      if (q.sum > 0.0) qt = Exps(q.ref, c32).of(lq, tab) / q.sum;
      fine = known && (double)u * qt < pt;
    }
    if (lane == 0) {
      d->row[i] = p;
      if (!last) d->of[i] = q, d->p[i] = pt, d->fine[i] = fine;
    }
  }
  __syncthreads();
  int r = 0;
  while (r < n && d->fine[r]) r++;
  return r;
}

// The weights after r accepted drafts; PLAIN: of p_r alone.
struct Weights {
  const float *x, *y;
  Exps p, q;
  double ip, iq;
  uint32_t except;  // a draft that was certain, and rejected
  __device__ __forceinline__ double of(int t, float lx, float ly, bool plain, const uint64_t *tab) const {
    const double w = p.of(lx, tab) * ip;
    if (plain) return w;
    if (!y) return (uint32_t)t == except ? 0.0 : w;
    return fmax(w - q.of(ly, tab) * iq, 0.0);
  }
  __device__ __forceinline__ double at(int t, bool plain, const uint64_t *tab) const {
    return of(t, x[t], plain || !y ? 0.0f : y[t], plain, tab);
  }
};

// The first token of [first, end) whose weights up to it, and `before`, are above
// `border`; where rounding leaves none, the last one that has a weight.
__device__ __forceinline__ int pick(const Weights &w, bool plain, int first, int end, double before,
                                    double border, const uint64_t *tab) {
  __shared__ double wsum[4];
  __shared__ int wfound[4], wlast[4], chosen;
  __shared__ double base_of;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int each = (end - first + kNT - 1) / kNT;  // a thread's tokens, next to each other
  const int t0 = first + min(tid * each, end - first), t1 = min(end, t0 + each);
  double sum = 0.0;
  int last = -1;
  for (int t = t0; t < t1; t++) {
    const double x = w.at(t, plain, tab);
    sum += x;
    if (x > 0.0) last = t;
  }
  double base = wave_before(sum);
  if (lane == 63) wsum[wave] = base + sum;
  __syncthreads();
  for (int i = 0; i < wave; i++) base += wsum[i];
  base += before;
  const uint64_t over = __ballot(sum > 0.0 && base + sum > border), some = __ballot(last >= 0);
  if (lane == 0) {
    wfound[wave] = over ? wave * 64 + __ffsll((unsigned long long)over) - 1 : kNT;
    wlast[wave] = some ? wave * 64 + 63 - __clzll((long long)some) : -1;
  }
  __syncthreads();
  int who = min(min(wfound[0], wfound[1]), min(wfound[2], wfound[3]));
  if (who == kNT) who = max(max(wlast[0], wlast[1]), max(wlast[2], wlast[3]));
  if (tid == who) base_of = base, chosen = last;
  __syncthreads();
  if (who < 0) return -1;
  // that thread's tokens again, by the first wave's lanes
  if (wave == 0) {
    double x = base_of;
    const int f = first + who * each, g = min(end, f + each);
    for (int b = f; b < g; b += 64) {
      const double v = b + lane < g ? w.at(b + lane, plain, tab) : 0.0;
      const double up = x + wave_before(v) + v;
      const uint64_t hit = __ballot(v > 0.0 && up > border);
      if (hit) {
        if (lane == 0) chosen = b + __ffsll((unsigned long long)hit) - 1;
        break;
      }
      x = __shfl(up, 63);
    }
  }
  __syncthreads();
  return chosen;
}

// grid (chunk, sequence): every workgroup of a sequence decides on its drafts and
// sums its chunk of the weights; the last one to have done so draws.
__global__ void __launch_bounds__(kNT) k_verify_draw(VerifyArgs a) {
  __shared__ uint64_t tab[32];
  __shared__ Choice d;
  __shared__ double wsum[4];
  __shared__ int mine;
  const int s = blockIdx.y, n = drafts_of(a, s), tid = threadIdx.x;
  uint32_t *out = a.out + (size_t)s * (a.K + 1);
  float *logp = a.logp ? a.logp + (size_t)s * (a.K + 1) : nullptr;
  const double c32 = scale_of(a, s);
  if (blockIdx.x && (n < 0 || c32 == 0.0)) return;
  if (n < 0) {
    for (int i = tid; i <= a.K; i += kNT) {
      out[i] = a.pad;
      if (logp) logp[i] = 0.0f;
    }
    if (tid == 0) a.count[s] = 0;
    return;
  }
  copy_table(tab);
  __syncthreads();
  const int r = decide(a, s, n, c32, tab, &d);
  const Stat p = d.row[r];
  int t = -1;
  double pt = 1.0;
  if (c32 == 0.0) {
    t = p.ref > kNone ? p.at : -1;
  } else {
    const Stat q = r == n ? Stat{0.0, kNone, 0} : d.of[r];
    const bool plain = r == n || (a.draft && !(q.sum > 0.0));  // (a draft row of -inf: q is 0)
    const Weights w{row_of(a, s, r),
                    plain || !a.draft ? nullptr : row_of(a, s, a.K + 1 + r),
                    Exps(p.ref, c32),
                    Exps(q.ref, c32),
                    p.sum > 0.0 ? 1.0 / p.sum : 0.0,
                    q.sum > 0.0 ? 1.0 / q.sum : 0.0,
                    r == n ? 0 : a.token[(size_t)s * a.K + r]};
    const int first = blockIdx.x * a.per, left = min(a.per, a.vocab - first);
    double sum = 0.0;
    if (p.sum > 0.0) {
      float y[8], ynext[8];
      const float *yr = w.y ? w.y + first : nullptr;
      if (yr) load_block(yr, left, ynext);
      over_blocks(w.x + first, left, [&](int b, const float *v) {
        if (yr) {
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = ynext[i];
          if (b + kBlock < left) load_block(yr + b + kBlock, left - b - kBlock, ynext);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
          sum += w.of(first + b + i / 4 * (kBlock / 2) + tid * 4 + i % 4, v[i], yr ? y[i] : 0.0f, plain, tab);
      });
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) wsum[tid >> 6] = sum;
    __syncthreads();
    double *sums = a.weight + (size_t)s * a.chunks;
    if (tid == 0) {
      __hip_atomic_store(sums + blockIdx.x, (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      mine = __hip_atomic_fetch_add(a.done + s, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1;
    }
    __syncthreads();
    if (!mine) return;
    // the chunk that the draw falls into, by the first wave
    __shared__ double before_of, border_of;
    __shared__ int chunk_of;
    if (tid < 64) {
      double total = 0.0;
      for (int i0 = 0; i0 < a.chunks; i0 += 64) {
        const double x = i0 + tid < a.chunks ? __hip_atomic_load(sums + i0 + tid, __ATOMIC_RELAXED,
                                                                 __HIP_MEMORY_SCOPE_AGENT)
                                             : 0.0;
        total += __shfl(wave_before(x) + x, 63);
      }
      const double u = (double)a.u[(size_t)s * (a.K + 1) + a.K], border = u * total;
      double base = 0.0, before = 0.0;
      int at = -1;
      for (int i0 = 0; i0 < a.chunks; i0 += 64) {
        const double x = i0 + tid < a.chunks ? __hip_atomic_load(sums + i0 + tid, __ATOMIC_RELAXED,
                                                                 __HIP_MEMORY_SCOPE_AGENT)
                                             : 0.0;
        const double lo = base + wave_before(x);
        const uint64_t some = __ballot(x > 0.0), over = __ballot(x > 0.0 && lo + x > border);
        // the first above the border, or the last that has a weight
        const uint64_t from = over ? over : some;
        if (from) {
          const int l = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
          at = i0 + l;
          before = __shfl(lo, l);
        }
        if (over) break;
        base = __shfl(lo + x, 63);
      }
      if (tid == 0) before_of = before, border_of = at < 0 ? u : border, chunk_of = at;
    }
    __syncthreads();
    const int at = chunk_of;
    if (at >= 0)
      t = pick(w, plain, at * a.per, at * a.per + min(a.per, a.vocab - at * a.per), before_of, border_of, tab);
    else if (p.sum > 0.0)  // p_r is nowhere above q_r: from p_r
      t = pick(w, true, 0, a.vocab, 0.0, border_of, tab);
    if (t >= 0) pt = w.p.of(w.x[t], tab) * w.ip;
  }
  for (int i = tid; i <= a.K; i += kNT) {
    out[i] = i < r ? a.token[(size_t)s * a.K + i] : (i == r && t >= 0 ? (uint32_t)t : a.pad);
    if (!logp) continue;
    double l = 0.0;
    if (i < r) l = log(d.p[i]);
    if (i == r) l = t < 0 ? -__builtin_huge_val() : log(pt);
    logp[i] = (float)l;
  }
  if (tid == 0) a.count[s] = r + 1;
}

// ---------------------------------------------------------------- host
struct Space {
  int per, chunks, rows;
  size_t stat, weight, done, total;
};
Space space_of(const syn_hip_draft_verify_params &p) {
  Space s;
  s.rows = 2 * (int)p.max_draft + 1;
  // chunks of 2048 to 16384 tokens, as long as there are workgroups for the chip
  s.per = kBlock;
  while (s.per < 8 * kBlock && p.n_seqs * (size_t)s.rows * cdiv(p.vocab, 2 * s.per) >= 2048) s.per *= 2;
  s.chunks = (int)cdiv(p.vocab, s.per);
  s.stat = 0;
  s.weight = (size_t)p.n_seqs * s.rows * s.chunks * sizeof(Stat);
  s.done = s.weight + (size_t)p.n_seqs * s.chunks * 8;
  s.total = round_up(s.done + (size_t)p.n_seqs * 4, 16);
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
  a.done = reinterpret_cast<int32_t *>(ws + sp.done);
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
  hipLaunchKernelGGL(k_verify_draw, dim3(a.chunks, p->n_seqs), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // extern "C"
