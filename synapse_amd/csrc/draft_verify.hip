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
// probabilities are small, so exponentials and sums are f64 throughout: with
// sums off by 2^-24 one in a hundred draws over 150000 tokens would fall to a
// neighbour.
//
// Three launches: every row read once (the statistics), the decisions, and the
// weights of one target and one draft row of a sequence summed by blocks, whose
// last workgroup draws.  64 sequences of up to 8 drafts, 151936 tokens, 506 MB of
// rows: 101 us (5.0 TB/s, a large copy reaches 4.7), 5.6 and 30; one of 4 drafts and
// 32000 tokens 3.4, 3.2 and 8.1, each a chain of dependent loads.
#include <algorithm>

#include "kv_pages.hpp"
#include "wave_ops.hpp"

namespace syn {

namespace {

constexpr int kNT = 256;
constexpr int kBlock = 8 * kNT;  // tokens that a workgroup has in registers at a time
constexpr int kDraws = 4;  // blocks of a workgroup that sums weights, at most
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

// The draw that is left of a sequence when its drafts are decided on: weights
// max(p / sum - q / sum, 0) from the logits of a target row, and of a draft row.
struct Draw {
  double ip, iq;    // 1 / sum
  float pref, qref;
  int r;            // drafts accepted; -1: nothing to draw
  uint32_t except;  // a draft that was certain, and rejected
  int32_t plain;    // p alone
};

struct VerifyArgs {
  const float *target, *draft, *heat, *u;
  const uint32_t *token;
  const int32_t *n_draft;
  uint32_t *out;
  int32_t *count;
  float *logp;
  Stat *stat;      // [n_seqs][target rows, then draft rows][chunks]
  Draw *draw;      // [n_seqs]
  uint64_t *weight;  // [n_seqs][blocks] sums (f64)
  int32_t *done;     // [n_seqs] workgroups that have theirs
  size_t ld_target, target_stride, ld_draft, draft_stride;
  int K, rows, vocab, chunks, per, blocks, draws;  // per: tokens of a chunk, whole blocks
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
  // of d = x - ref, 2^-1000 where that is less (or x NaN), plus sum
  __device__ __forceinline__ double at(double d, const uint64_t *tab, double sum = 0.0) const {
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
    return __builtin_fma(y, __longlong_as_double((long long)t), sum);
  }
  __device__ __forceinline__ double at_least(float x, const uint64_t *tab, double sum = 0.0) const {
    return at((double)x - ref, tab, sum);
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
// one, until one is 2^400 above that.  Bound by its bytes, with vector instructions
// in some 80 % of the SIMDs' cycles beside them (a tenth more of those, 101 us as
// before).
__global__ void __launch_bounds__(kNT) k_verify_rows(VerifyArgs a) {
  __shared__ uint64_t tab[32];
  __shared__ Stat part[4];
  const int s = blockIdx.y / a.rows, r = blockIdx.y - s * a.rows, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, n = drafts_of(a, s);
  const double c32 = scale_of(a, s);
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
      for (int i = 0; i < 8; i++) sum = e.at_least(v[i], tab, sum);
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

// over the 16 lanes of a row
template <class F, class Op> __device__ __forceinline__ F over_16(F x, Op op) {
  x = op(x, partner<8>(x));
  x = op(x, partner<4>(x));
  x = op(x, partner<2>(x));
  return op(x, partner<1>(x));
}

constexpr int kDecideNT = 512;

// One workgroup a sequence: 16 lanes join the chunks of a row, all rows at once,
// and a lane a draft says whether it is accepted.  (Done again by every workgroup
// that sums weights instead, 64 sequences of 8 drafts took 179 us and not 141.)
__global__ void __launch_bounds__(kDecideNT) k_verify_decide(VerifyArgs a) {
  __shared__ uint64_t tab[32];
  __shared__ Stat row[2 * kMaxDraft + 1];    // target rows, then draft rows
  __shared__ double prob[2 * kMaxDraft + 1]; // of the row's draft
  __shared__ int accepted;
  const int s = blockIdx.x, n = drafts_of(a, s), tid = threadIdx.x, l = tid & 15;
  const double c32 = scale_of(a, s);
  const bool greedy = c32 == 0.0;
  uint32_t *out = a.out + (size_t)s * (a.K + 1);
  float *logp = a.logp ? a.logp + (size_t)s * (a.K + 1) : nullptr;
  if (n < 0) {
    if (tid <= a.K) {
      out[tid] = a.pad;
      if (logp) logp[tid] = 0.0f;
    }
    if (tid == 0) a.count[s] = 0, a.draw[s].r = -1;
    return;
  }
  copy_table(tab);
  __syncthreads();
  const int rows = n + 1 + (a.draft && !greedy ? n : 0);
  for (int k = tid >> 4; k < rows; k += kDecideNT / 16) {
    const bool of_draft = k > n;
    const int i = of_draft ? k - n - 1 : k, r = of_draft ? a.K + 1 + i : i;
    const Stat *st = a.stat + ((size_t)s * a.rows + r) * a.chunks;
    const Stat q0 = st[min(l, a.chunks - 1)];
    float x = kNone;
    if (i < n && !greedy) {
      const uint32_t t = a.token[(size_t)s * a.K + i];
      if (t < (uint32_t)a.vocab) x = row_of(a, s, r)[t];
    }
    Stat all{0.0, kNone, 0x7fffffff};
    for (int c = l; c < a.chunks; c += 16) {
      const Stat q = c == l ? q0 : st[c];
      if (q.ref > all.ref) all.ref = q.ref, all.at = q.at;
    }
    if (greedy) {
      for (int o = 8; o > 0; o >>= 1) {
        const float t = __shfl_xor(all.ref, o);
        const int at = __shfl_xor(all.at, o);
        if (t > all.ref || (t == all.ref && at < all.at)) all.ref = t, all.at = at;
      }
    } else {
      all.ref = over_16(all.ref, [](float p, float q) { return fmaxf(p, q); });
      const Exps e(all.ref, c32);
      for (int c = l; c < a.chunks; c += 16) {
        const Stat q = c == l ? q0 : st[c];
        if (q.ref > kNone) all.sum += q.sum * e.of(q.ref, tab);
      }
      all.sum = over_16(all.sum, [](double p, double q) { return p + q; });
      if (l == 0) prob[k] = all.sum > 0.0 ? e.of(x, tab) / all.sum : 0.0;
    }
    if (l == 0) row[k] = all;
  }
  __syncthreads();
  if (tid < 64) {  // (at most 64 drafts)
    bool fine = true;
    if (tid < n) {
      const uint32_t t = a.token[(size_t)s * a.K + tid];
      const double u = (double)a.u[(size_t)s * (a.K + 1) + tid];
      if (greedy)
        fine = row[tid].ref > kNone && t == (uint32_t)row[tid].at;
      else
        fine = t < (uint32_t)a.vocab && u * (a.draft ? prob[n + 1 + tid] : 1.0) < prob[tid];
    }
    const uint64_t wrong = __ballot(!fine);
    if (tid == 0) accepted = wrong ? __ffsll((unsigned long long)wrong) - 1 : n;
  }
  __syncthreads();
  const int r = accepted;
  const Stat p = row[r];
  const bool none = greedy ? p.ref == kNone : !(p.sum > 0.0);
  if (tid <= a.K) {  // (a token that is drawn comes later)
    out[tid] = tid < r ? a.token[(size_t)s * a.K + tid] : (tid == r && greedy && !none ? (uint32_t)p.at : a.pad);
    if (logp)
      logp[tid] = tid == r && none ? kNone : (tid < r && !greedy ? (float)log(prob[tid]) : 0.0f);
  }
  if (tid == 0) {
    a.count[s] = r + 1;
    Draw d{};
    d.r = greedy || none ? -1 : r;
    d.pref = p.ref;
    d.ip = 1.0 / p.sum;
    d.plain = r == n;
    if (r < n) {
      d.except = a.token[(size_t)s * a.K + r];
      if (a.draft && !greedy) {
        const Stat q = row[n + 1 + r];
        d.qref = q.ref;
        d.iq = 1.0 / q.sum;
        d.plain = !(q.sum > 0.0);  // (a draft row of -inf: q is 0)
      }
    }
    a.draw[s] = d;
    a.done[s] = 0;
  }
}

struct Weights {
  const float *x, *y;  // y: null where the weights are p's alone
  Exps p, q;
  double ip, iq;
  uint32_t except;  // a draft that was certain, and rejected; the vocabulary: none
  bool infinite;    // a row's largest logit is +inf
  // of token t with logits lx and ly
  template <bool INF> __device__ __forceinline__ double of(int t, float lx, float ly, const uint64_t *tab) const {
    double w = (INF ? p.of(lx, tab) : p.at_least(lx, tab)) * ip;
    if (y)
      w -= (INF ? q.of(ly, tab) : q.at_least(ly, tab)) * iq;
    else
      w = (uint32_t)t == except ? 0.0 : w;
    return w > 1e-290 ? w : 0.0;  // (2^-1000 is nothing)
  }
};

// wsum[block][wave]: the sums of the weights of the blocks of [first, first + n)
template <bool INF>
__device__ __forceinline__ void block_sums(const Weights &w, int first, int n, const uint64_t *tab,
                                           double (*wsum)[4]) {
  const float *yr = w.y ? w.y + first : nullptr;
  float y[8] = {}, ynext[8] = {};
  if (yr) load_block(yr, n, ynext);
  over_blocks(w.x + first, n, [&](int b, const float *v) {
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = ynext[i];
    if (yr && b + kBlock < n) load_block(yr + b + kBlock, n - b - kBlock, ynext);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++)
      sum += w.of<INF>(first + b + i / 4 * (kBlock / 2) + (int)threadIdx.x * 4 + i % 4, v[i], y[i], tab);
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) wsum[b / kBlock][threadIdx.x >> 6] = sum;
  });
}
__device__ __forceinline__ void sum_blocks(const Weights &w, int first, int n, const uint64_t *tab,
                                           double (*wsum)[4]) {
  if (w.infinite)
    block_sums<true>(w, first, n, tab, wsum);
  else
    block_sums<false>(w, first, n, tab, wsum);
}

// The first token of a block whose weights up to it, and `before`, are above
// `border`; where rounding leaves none, the last one that has a weight.
__device__ __forceinline__ int pick(const Weights &w, int first, int left, double before, double border,
                                    const uint64_t *tab) {
  __shared__ double wsum[4];
  __shared__ int wfound[4], wlast[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float v[8], y[8] = {};  // of 8 tokens next to each other
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = w.x[first + min(8 * tid + i, left - 1)];
  if (w.y)
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = w.y[first + min(8 * tid + i, left - 1)];
  double up[8], sum = 0.0;
  uint32_t some = 0;  // that have a weight
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int t = first + 8 * tid + i;
    const double in = w.infinite ? w.of<true>(t, v[i], y[i], tab) : w.of<false>(t, v[i], y[i], tab);
    const double x = 8 * tid + i < left ? in : 0.0;
    sum += x;
    up[i] = sum;
    some |= x > 0.0 ? 1u << i : 0u;
  }
  const double upto = wave_upto(sum);
  double base = wave_shifted(upto);
  if (lane == 63) wsum[wave] = upto;
  __syncthreads();
  for (int i = 0; i < wave; i++) base += wsum[i];
  base += before;
  int found = 0x7fffffff;
#pragma unroll
  for (int i = 7; i >= 0; i--)
    if ((some >> i & 1) && base + up[i] > border) found = 8 * tid + i;
  int last = some ? 8 * tid + 31 - __clz(some) : -1;
  found = over_wave(found, [](int p, int q) { return min(p, q); });
  last = over_wave(last, [](int p, int q) { return max(p, q); });
  if (lane == 0) wfound[wave] = found, wlast[wave] = last;
  __syncthreads();
  found = min(min(wfound[0], wfound[1]), min(wfound[2], wfound[3]));
  last = max(max(wlast[0], wlast[1]), max(wlast[2], wlast[3]));
  return first + (found < left ? found : last);
}

// grid (some blocks, sequence): the sums of the weights by blocks; the last
// workgroup of a sequence to have its sums draws.  As many blocks a workgroup as
// leave 1024 of them (64 sequences of 151936 tokens: one block each 50 us, four 30).
__global__ void __launch_bounds__(kNT) k_verify_draw(VerifyArgs a) {
  __shared__ uint64_t tab[32];
  __shared__ double wsum[kDraws][4];
  __shared__ int mine, block_of;
  __shared__ double before_of, border_of;
  const int s = blockIdx.y, tid = threadIdx.x;
  const Draw d = a.draw[s];
  if (d.r < 0) return;
  const double c32 = scale_of(a, s), u = (double)a.u[(size_t)s * (a.K + 1) + a.K];
  copy_table(tab);
  __syncthreads();
  Weights w{row_of(a, s, d.r),
            d.plain || !a.draft ? nullptr : row_of(a, s, a.K + 1 + d.r),
            Exps(d.pref, c32),
            Exps(d.qref, c32),
            d.ip,
            d.iq,
            d.plain ? (uint32_t)a.vocab : d.except,
            fmaxf(d.pref, d.qref) == __builtin_huge_valf()};
  const int first = blockIdx.x * a.draws * kBlock;
  sum_blocks(w, first, min(a.draws * kBlock, a.vocab - first), tab, wsum);
  __syncthreads();
  uint64_t *sums = a.weight + (size_t)s * a.blocks;
  if (tid < 64) {
    // As in split_k.hpp: an exchange that has returned is at the point where every
    // XCD's atomics are, so relaxed ones suffice (an acquire and a release each
    // write back and drop an L2: 142 us where this kernel then took 53).
    const int b = blockIdx.x * a.draws + tid;
    if (tid < a.draws && b < a.blocks) {
      const double x = (wsum[tid][0] + wsum[tid][1]) + (wsum[tid][2] + wsum[tid][3]);
      const uint64_t seen = __hip_atomic_exchange(sums + b, (uint64_t)__double_as_longlong(x), __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("" ::"v"(seen));
    }
    if (tid == 0)
      mine = __hip_atomic_fetch_add(a.done + s, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!mine) return;
  if (tid < 64) {  // the block that the draw falls into
    auto load = [&](int i) {
      return i < a.blocks ? __longlong_as_double((long long)__hip_atomic_load(
                                sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
                          : 0.0;
    };
    const double held[2] = {load(tid), load(64 + tid)};
    double total = held[0] + held[1];
    for (int i0 = 128; i0 < a.blocks; i0 += 64) total += load(i0 + tid);
    const double border = u * wave_sum(total);
    double base = 0.0, before = 0.0;
    int at = -1;
    for (int i0 = 0; i0 < a.blocks; i0 += 64) {
      const double x = i0 == 0 ? held[0] : (i0 == 64 ? held[1] : load(i0 + tid));
      const double upto = wave_upto(x), lo = base + wave_shifted(upto);
      const uint64_t some = __ballot(x > 0.0), over = __ballot(x > 0.0 && lo + x > border);
      if (over | some) {  // the first above the border, or the last that has a weight
        const int k = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)some);
        at = i0 + k;
        before = __shfl(lo, k);
      }
      if (over) break;
      base += __shfl(upto, 63);
    }
    if (tid == 0) before_of = before, border_of = border, block_of = at;
  }
  __syncthreads();
  int at = block_of;
  double before = before_of, border = border_of;
  if (at < 0) {  // p_r is nowhere above q_r: from p_r, whose weights sum to 1
    w.y = nullptr;
    w.except = (uint32_t)a.vocab;
    border = u;
    before = 0.0;
    double in = 0.0;
    for (int b = 0; b < a.blocks; b++) {
      __syncthreads();
      sum_blocks(w, b * kBlock, min(kBlock, a.vocab - b * kBlock), tab, wsum);
      __syncthreads();
      const double x = (wsum[0][0] + wsum[0][1]) + (wsum[0][2] + wsum[0][3]);
      if (!(x > 0.0)) continue;
      before += in;
      in = x;
      at = b;
      if (before + x > border) break;
    }
  }
  const int t = pick(w, at * kBlock, min(kBlock, a.vocab - at * kBlock), before, border, tab);
  if (tid == 0) {
    const size_t o = (size_t)s * (a.K + 1) + d.r;
    a.out[o] = (uint32_t)t;
    if (a.logp) a.logp[o] = (float)log(w.p.of(w.x[t], tab) * w.ip);
  }
}

// ---------------------------------------------------------------- host
struct Space {
  int per, chunks, rows, draws;
  size_t stat, draw, weight, done, total;
};
Space space_of(const syn_hip_draft_verify_params &p) {
  Space s;
  s.rows = 2 * (int)p.max_draft + 1;
  // Chunks of 2048 tokens, of up to 16384 as long as 2048 workgroups are left: a row's
  // chunks are joined one by one.  (64 sequences of up to 8 drafts, 151936 tokens, 124
  // us, 203 in chunks of 2048 alone; 32000 tokens 47 and 65.  The chip holds 1280, five
  // a CU by their 90 registers: down to as many, 8 sequences of 4 drafts and 151936
  // tokens 32.0 where this takes 33.3, the rest the same.)
  s.per = kBlock;
  while (s.per < 8 * kBlock && p.n_seqs * (size_t)s.rows * cdiv(p.vocab, 2 * s.per) >= 2048) s.per *= 2;
  s.chunks = (int)cdiv(p.vocab, s.per);
  s.draws = 1;
  while (s.draws < kDraws && p.n_seqs * cdiv(p.vocab, 2 * s.draws * kBlock) >= 1024) s.draws *= 2;
  s.stat = 0;
  s.draw = (size_t)p.n_seqs * s.rows * s.chunks * sizeof(Stat);
  s.weight = s.draw + p.n_seqs * sizeof(Draw);
  s.done = s.weight + (size_t)p.n_seqs * cdiv(p.vocab, kBlock) * 8;
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
  a.weight = reinterpret_cast<uint64_t *>(ws + sp.weight);
  a.done = reinterpret_cast<int32_t *>(ws + sp.done);
  a.draw = reinterpret_cast<Draw *>(ws + sp.draw);
  a.ld_target = p->ld_target;
  a.target_stride = p->target_stride;
  a.ld_draft = p->ld_draft;
  a.draft_stride = p->draft_stride;
  a.K = (int)p->max_draft;
  a.rows = a.draft ? sp.rows : a.K + 1;
  a.vocab = (int)p->vocab;
  a.chunks = sp.chunks;
  a.per = sp.per;
  a.blocks = (int)cdiv(p->vocab, kBlock);
  a.draws = sp.draws;
  a.pad = p->pad;
  hipStream_t s = pick_stream(stream);
  hipLaunchKernelGGL(k_verify_rows, dim3(a.chunks, p->n_seqs * a.rows), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_verify_decide, dim3(p->n_seqs), dim3(kDecideNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_verify_draw, dim3((unsigned)cdiv(a.blocks, a.draws), p->n_seqs), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // extern "C"
