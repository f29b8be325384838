// Beam search's choice over beams and vocabulary, and the states that follow
// it.
#include "beam.hpp"
#include "kv_pages.hpp"
#include "wave_ops.hpp"

namespace syn {

namespace {

// ---------------------------------------------------------------- choice
// Value of (beam b, token t): score_b + logit_t - log sum exp(logits of b).
// Rows are cut into chunks over the whole chip: a workgroup reads its chunk
// once into registers, forms max and sum of exp, and keeps the n_select best
// logits (the order within a beam is that of its logits); one workgroup a
// group then joins the sums in f64 and chooses among the chunks' candidates by
// their values in f64.  A chunk's sum is f32: in units of 2^-24 of it, its
// terms' arguments, up to ln 8192 below the top where they weigh, are off by 23
// at most, the exponential by 2, the additions (31 in a thread, 8 over lanes and
// waves) by 39, so that a row's logarithm is off by less than 2^-18.  (f64
// exponentials, a polynomial of degree 8, take 39.4 us where these take 29.2, 128
// rows of 151936.)  The selection itself never sorts: if G >= n groups of values
// are formed, n values at least are not below the least of the groups' maxima,
// and few are; those go to LDS, where each counts the ones before it.
//
// 128 rows of 151936 logits, 16 to choose: 29.4 us, the chunks 20 (3.9 TB/s),
// the join of 152 lists of 16 a group 9; 32 rows of 128256: 13.5 us; 4 rows of
// 32000: 9.2, two launches.  The chunks are bound neither by the read (16 us at a
// copy's rate) nor by their instructions (vector instructions in 45 % of the
// SIMDs' cycles): a workgroup has loaded all of its chunk before it computes and
// has nothing in flight then, and 2432 workgroups at six a CU are 1.6 rounds.  A
// single launch would need counters that are zero at the start, which a caller's
// workspace is not.
//
// Equal values go to the lower beam; within a beam the order is that of the
// logits everywhere (f64 may hold two of them as the same value), equal ones
// by token.  A value of -inf is a candidate only when a group has fewer than
// n_select others, so the chunks leave those out and the second kernel fills
// up with them in order.
struct Cand {
  float x;
  int i;  // token
};
struct ChunkStat {
  float top, sum;  // largest logit, sum of exp(logit - top)
};

struct SelectArgs {
  const float *logits, *scores;
  const int32_t *finished;
  int32_t *parent, *finished_out;
  uint32_t *token;
  float *score;
  Cand *cand;       // [rows][chunks][n_select], best first, then places of -inf
  ChunkStat *stat;  // [rows][chunks]
  size_t ld;
  int vocab, chunks, n_beams, n_select, eos, pad;
};

constexpr float kNone = -__builtin_huge_valf();

__device__ __forceinline__ bool is_dead(const SelectArgs &a, size_t row) {
  return !isfinite(a.scores[row]);
}
__device__ __forceinline__ bool is_done(const SelectArgs &a, size_t row) {
  return a.finished && a.finished[row] != 0;
}

// The lanes in G groups (a power of two): the steps above G give every lane its
// group's maximum, those below the least of them.
template <class F> __device__ __forceinline__ F group_max(F x, int G) {
  if (G <= 32) x = greater(x, partner<32>(x));
  if (G <= 16) x = greater(x, partner<16>(x));
  if (G <= 8) x = greater(x, partner<8>(x));
  if (G <= 4) x = greater(x, partner<4>(x));
  if (G <= 2) x = greater(x, partner<2>(x));
  if (G <= 1) x = greater(x, partner<1>(x));
  return x;
}
template <class F> __device__ __forceinline__ F least_group(F x, int G) {
  if (G > 1) x = lesser(x, partner<1>(x));
  if (G > 2) x = lesser(x, partner<2>(x));
  if (G > 4) x = lesser(x, partner<4>(x));
  if (G > 8) x = lesser(x, partner<8>(x));
  if (G > 16) x = lesser(x, partner<16>(x));
  if (G > 32) x = lesser(x, partner<32>(x));
  return x;
}

// keys that order as (value descending, index ascending) when the larger is
// first; no key is 0 (-0.0 + 0.0 is 0.0: zeros are equal, and so are their keys)
__device__ __forceinline__ uint32_t ordered(float x) {  // larger for larger x
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  return (uint64_t)ordered(x) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ Cand cand_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return Cand{__uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u), (int)~(uint32_t)key};
}

constexpr int kChunkNT = 256;
constexpr int kWaveCap = 256;  // of a wave's candidates

// PER values a thread, which stay in registers; six waves a SIMD (29.5 us at 128
// rows of 151936, five 29.9, seven 30.8).
template <int PER>
__global__ void __launch_bounds__(kChunkNT, 6) k_beam_chunks(SelectArgs a) {
  __shared__ __align__(16) uint64_t list[4][kWaveCap];
  __shared__ float wtop[4], wsum[4], wgroup[4][64];
  __shared__ int count[4], ri[4];
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t at = (size_t)row * a.chunks + chunk;
  Cand *out = a.cand + at * a.n_select;
  if (is_dead(a, row) || is_done(a, row)) {
    if (tid == 0) a.stat[at] = ChunkStat{kNone, 0.0f};
    for (int i = tid; i < a.n_select; i += kChunkNT) out[i] = Cand{kNone, 0};
    return;
  }
  // element e of thread t: t * 4 + e % 4 of every 1024
  const int first = chunk * (kChunkNT * PER), left = min(a.vocab - first, kChunkNT * PER);
  const float *x0 = a.logits + (size_t)row * a.ld + first;
  float x[PER];
  if (left >= 4) {
    // (a 16-byte load needs 4-byte alignment only: 128 rows of 151935, 80 of them
    // live, 8 to choose, 20.5 us; 25.6 with 4-byte loads)
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      const int at4 = min(i * kChunkNT + tid * 4, left - 4);
      const f32x4u v = __builtin_nontemporal_load(reinterpret_cast<const f32x4u *>(x0 + at4));
#pragma unroll
      for (int j = 0; j < 4; j++) x[i + j] = v[j];
    }
    if (left < kChunkNT * PER)
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        // the four that the row ends in were loaded `back` early: turn them
        const int e = i * kChunkNT + tid * 4, back = e - min(e, left - 4);
        const float y[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
        float z[4];
#pragma unroll
        for (int j = 0; j < 4; j++) z[j] = back & 1 ? y[(j + 1) & 3] : y[j];
#pragma unroll
        for (int j = 0; j < 4; j++) x[i + j] = e + j >= left ? kNone : (back & 2 ? z[(j + 2) & 3] : z[j]);
      }
  } else {  // (no load behind a branch: all are in flight together)
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] = x0[min((i / 4 * kChunkNT + tid) * 4 + i % 4, left - 1)];
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] = (i / 4 * kChunkNT + tid) * 4 + i % 4 < left ? x[i] : kNone;
  }
  float top = kNone, half = kNone;  // of all values; of the second half
#pragma unroll
  for (int i = 0; i < PER; i++) {
    x[i] = fmaxf(x[i], kNone);  // NaN: -inf
    if (i < PER / 2)
      top = fmaxf(top, x[i]);
    else
      half = fmaxf(half, x[i]);
  }
  // Groups of threads, the same of every wave; above 64, two of each lane's
  // values, both of which are not below the lesser.
  const int n = a.n_select;
  const int pow2 = n <= 1 ? 1 : 1 << (32 - __builtin_clz(n - 1)), G = min(pow2, 64);
  wgroup[wave][lane] = group_max(pow2 > 64 ? fminf(top, half) : fmaxf(top, half), G);
  top = wave_max(fmaxf(top, half));
  if (lane == 0) wtop[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(wtop[0], wtop[1]), fmaxf(wtop[2], wtop[3]));
  const float tau = fmaxf(least_group(fmaxf(fmaxf(wgroup[0][lane], wgroup[1][lane]),
                                            fmaxf(wgroup[2][lane], wgroup[3][lane])), G),
                          -3.402823466e38f);  // finite: -inf is no candidate
  float sum = 0.0f;
  if (top == __builtin_huge_valf()) {
#pragma unroll
    for (int i = 0; i < PER; i++) sum += x[i] == top ? 1.0f : 0.0f;
  } else if (top > kNone) {
#pragma unroll
    for (int i = 0; i < PER; i++) sum += __builtin_amdgcn_exp2f((x[i] - top) * 1.44269504088896340736f);
  }
  sum = wave_sum(sum);
  if (lane == 0) wsum[wave] = sum;
  int held = 0;  // the same in every lane
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const bool in = x[i] >= tau;
    const uint64_t who = __ballot(in);
    if (!who) continue;
    const int k = held + __popcll(who & ((1ull << lane) - 1));
    if (in && k < kWaveCap) list[wave][k] = key_of(x[i], first + (i / 4 * kChunkNT + tid) * 4 + i % 4);
    held += __popcll(who);
  }
  if (lane == 0) count[wave] = held;
  if (lane < 8 && held + lane < kWaveCap) list[wave][held + lane] = 0;  // read in eights
  __syncthreads();
  const int K = count[0] + count[1] + count[2] + count[3];
  const int most = max(max(count[0], count[1]), max(count[2], count[3]));
  if (most <= kWaveCap) {
    for (int k = lane; k < held; k += 64) {
      const uint64_t key = list[wave][k];
      int before = 0;
      for (int w = 0; w < 4; w++)
        for (int j = 0; j < count[w]; j += 8) {
          uint64_t o[8];
#pragma unroll
          for (int u = 0; u < 8; u++) o[u] = list[w][j + u];
#pragma unroll
          for (int u = 0; u < 8; u++) before += o[u] > key;
        }
      if (before < n) out[before] = cand_of(key);
    }
    for (int i = K + tid; i < n; i += kChunkNT) out[i] = Cand{kNone, 0};
  } else {
    // many values alike: one after the other, each the first behind the last
    float pv = __builtin_huge_valf();
    int pi = -1;
    for (int r = 0; r < n; r++) {
      float bv = kNone;
      int bi = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int e = first + (i / 4 * kChunkNT + tid) * 4 + i % 4;
        const bool behind = x[i] < pv || (x[i] == pv && e > pi);
        if (behind && x[i] > kNone && (x[i] > bv || (x[i] == bv && e < bi))) bv = x[i], bi = e;
      }
      for (int o = 32; o > 0; o >>= 1) {
        const float v = __shfl_xor(bv, o);
        const int i = __shfl_xor(bi, o);
        if (v > bv || (v == bv && i < bi)) bv = v, bi = i;
      }
      __syncthreads();
      if (lane == 0) wtop[wave] = bv, ri[wave] = bi;
      __syncthreads();
      bv = wtop[0], bi = ri[0];
      for (int w = 1; w < 4; w++)
        if (wtop[w] > bv || (wtop[w] == bv && ri[w] < bi)) bv = wtop[w], bi = ri[w];
      if (tid == 0) out[r] = Cand{bv, bi};
      pv = bv;
      pi = bi;
    }
  }
  if (tid == 0) a.stat[at] = ChunkStat{top, (wsum[0] + wsum[1]) + (wsum[2] + wsum[3])};
}

constexpr int kMergeNT = 1024;
constexpr int kMergeCap = 1024;

// One workgroup a group: the sums of a beam's chunks joined in f64, then the
// best of all lists.  4.3 us for one group of 4 beams, 9 for 16 groups of 152
// lists at once: latency (f64 logarithms, four barriers, the ranks in LDS).
__global__ void __launch_bounds__(kMergeNT) k_beam_merge(SelectArgs a) {
  struct Pick {
    double v;
    int b, t, j;  // j: the place among the beam's candidates, which goes up with t where x is the same
    float x;
  };
  __shared__ Pick list[kMergeCap];
  __shared__ uint64_t keys[kMergeCap + 4], index[kMergeCap + 4];
  __shared__ double logsum[kMaxBeams], wtau[16];
  __shared__ float top[kMaxBeams], score[kMaxBeams];
  __shared__ int state[kMaxBeams];  // 0 live, 1 finished, 2 without a continuation
  __shared__ int done[kMaxBeams];
  __shared__ int count, chosen, rj[16];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int W = a.n_beams, n = a.n_select, C = a.chunks;
  const size_t row0 = (size_t)g * W;
  if (tid == 0) count = 0, chosen = 0;
  const int L = W * C, T = L * n;  // lists, and places in them
  const Cand *cand = a.cand + row0 * C * n;
  // the thread's first candidates are asked for ahead of the sums
  constexpr int kHeld = 4;
  Cand mine[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; k++) mine[k] = cand[min(tid + k * kMergeNT, T - 1)];
  // Lists are in order: if the D-th of a list is not below tau, D of it are
  // not.  Of the lists of a wave in G groups, D G >= n, the least group maximum.
  const int G = min(n <= 1 ? 1 : 1 << (32 - __builtin_clz(n - 1)), 1 << (31 - __builtin_clz(min(L, 64))));
  const int D = (n + G - 1) / G;
  const Cand front = cand[min(tid, L - 1) * n + D - 1];
  for (int b = wave; b < W; b += kMergeNT / 64) {
    const ChunkStat *st = a.stat + (row0 + b) * C;
    const ChunkStat q0 = st[min(lane, C - 1)];
    float m = q0.top;
    for (int c = lane + 64; c < C; c += 64) m = fmaxf(m, st[c].top);
    m = wave_max(m);
    double s = 0.0;
    for (int c = lane; c < C; c += 64) {
      const ChunkStat q = c == lane ? q0 : st[c];
      if (q.top > kNone) s += q.top == m ? (double)q.sum : (double)q.sum * exp((double)q.top - (double)m);
    }
    s = wave_sum(s);
    if (lane == 0) {
      top[b] = m;
      logsum[b] = s > 0.0 ? log(s) : 0.0;
      score[b] = a.scores[row0 + b];
      done[b] = is_done(a, row0 + b);
      state[b] = is_dead(a, row0 + b) ? 2 : done[b];
    }
  }
  __syncthreads();
  const double none = -__builtin_huge_val();
  auto value = [&](int b, float x) {  // of a live beam
    const double d = x == top[b] ? 0.0 : (double)x - (double)top[b];
    return x == kNone ? none : (double)score[b] + (d - logsum[b]);
  };
  // candidate j: the lists' places (those of beams that do not live are empty)
  auto pick = [&](int j, const Cand &c) {
    const int b = (int)((uint32_t)j / (uint32_t)n / (uint32_t)C);
    return Pick{value(b, c.x), b, c.i, j - b * C * n, c.x};
  };
  auto closed = [&](int b) { return Pick{(double)score[b], b, a.pad, 0, 0.0f}; };  // a finished beam's
  // two logits of a beam may be so close that their values are the same
  auto ahead = [](const Pick &p, const Pick &q) {
    if (p.v != q.v) return p.v > q.v;
    if (p.b != q.b) return p.b < q.b;
    return p.x > q.x || (p.x == q.x && p.t < q.t);
  };
  double key = none;
  for (int q = tid; q < L; q += kMergeNT) {
    const int j = q * n + D - 1;
    key = fmax(key, pick(j, q == tid ? front : cand[j]).v);
  }
  const double tau_w = least_group(group_max(key, G), G);
  if (lane == 0) wtau[wave] = tau_w;
  __syncthreads();
  double tau = none;
  for (int w = 0; w < kMergeNT / 64; w++) tau = fmax(tau, wtau[w]);
  auto offer = [&](const Pick &p) {
    if (p.v >= tau && p.v > none) {
      const int k = atomicAdd(&count, 1);
      if (k < kMergeCap) list[k] = p;
    }
  };
#pragma unroll
  for (int k = 0; k < kHeld; k++)
    if (tid + k * kMergeNT < T) offer(pick(tid + k * kMergeNT, mine[k]));
  for (int j = tid + kHeld * kMergeNT; j < T; j += kMergeNT) offer(pick(j, cand[j]));
  if (tid < W && state[tid] == 1) offer(closed(tid));
  __syncthreads();
  const int K = count;
  auto emit = [&](int r, const Pick &p) {
    const size_t o = (size_t)g * n + r;
    a.parent[o] = p.b;
    a.token[o] = (uint32_t)p.t;
    a.score[o] = (float)p.v;
    if (a.finished_out) a.finished_out[o] = done[p.b] || p.t == a.eos;
  };
  if (K <= kMergeCap) {
    for (int k = tid; k < K + 4; k += kMergeNT) {
      const Pick p = list[max(min(k, K - 1), 0)];
      const uint64_t u = (uint64_t)__double_as_longlong(p.v + 0.0);  // (as in key_of)
      keys[k] = k < K ? (u >> 63 ? ~u : u | 1ull << 63) : 0;
      // (places of a beam are below 2^26: at most 2^18 chunks of 128)
      index[k] = ~((uint64_t)p.b << 58 | (uint64_t)~ordered(p.x) << 26 | (uint32_t)p.j);
    }
    __syncthreads();
    for (int k = tid; k < K; k += kMergeNT) {
      const uint64_t key = keys[k], mine_at = index[k];
      int before = 0;
      for (int j = 0; j < K; j += 4) {
        uint64_t o[4], i[4];
#pragma unroll
        for (int u = 0; u < 4; u++) o[u] = keys[j + u], i[u] = index[j + u];
#pragma unroll
        for (int u = 0; u < 4; u++) before += (o[u] > key) | ((o[u] == key) & (i[u] > mine_at));
      }
      if (before < n) emit(before, list[k]);
    }
    if (tid == 0) chosen = min(K, n);
  } else {
    Pick last{__builtin_huge_val(), -1, -1, 0, 0.0f};
    for (int r = 0; r < n; r++) {
      Pick p{none, 0x7fffffff, 0, 0, 0.0f};
      for (int j = tid; j < T + W; j += kMergeNT) {
        Pick q{none, 0, 0, 0, 0.0f};
        if (j < T)
          q = pick(j, cand[j]);
        else if (state[j - T] == 1)
          q = closed(j - T);
        if (q.v > none && ahead(last, q) && ahead(q, p)) p = q;
      }
      // the first of the wave, of the workgroup
      for (int o = 32; o > 0; o >>= 1) {
        const Pick q{__shfl_xor(p.v, o), __shfl_xor(p.b, o), __shfl_xor(p.t, o), 0, __shfl_xor(p.x, o)};
        if (ahead(q, p)) p = q;
      }
      __syncthreads();
      if (lane == 0) list[wave] = p;
      __syncthreads();
      for (int w = 0; w < kMergeNT / 64; w++)
        if (ahead(list[w], p)) p = list[w];
      if (tid == 0) emit(r, p);
      last = p;
    }
    if (tid == 0) chosen = n;
  }
  __syncthreads();
  if (chosen >= n) return;
  // Fewer than n_select: the rest are the first continuations of value -inf.
  int have = chosen;
  for (int b = 0; b < W && have < n; b++)
    for (int t0 = 0; t0 < a.vocab && have < n; t0 += kMergeNT) {
      const int t = t0 + tid;
      bool in = false;
      if (t < a.vocab)
        in = state[b] == 2 || (state[b] == 1 ? t != a.pad
                                             : value(b, fmaxf(a.logits[(row0 + b) * a.ld + t], kNone)) == none);
      const uint64_t who = __ballot(in);
      __syncthreads();
      if (lane == 0) rj[wave] = __popcll(who);
      __syncthreads();
      int at = have, all = 0;
      for (int w = 0; w < kMergeNT / 64; w++) {
        at += w < wave ? rj[w] : 0;
        all += rj[w];
      }
      at += __popcll(who & ((1ull << lane) - 1));
      if (in && at < n) emit(at, Pick{none, b, t, 0, 0.0f});
      have += all;
    }
}

syn_status_t check_select(const syn_hip_beam_select_params *p) {
  if (!p) return SYN_ERR_NULL_PTR;
  if (!p->n_beams || p->n_beams > kMaxBeams || !p->n_select || p->n_select > kMaxSelect) {
    set_error("beam_select: 1 to 64 beams and 1 to 128 continuations");
    return SYN_ERR_INVALID_ARG;
  }
  if (!p->vocab || p->vocab > 0x7ff00000u || (uint64_t)p->n_select > p->n_beams * (uint64_t)p->vocab ||
      (uint64_t)p->n_groups * p->n_beams > 65535u ||
      // (the join steps over the lists' places by 1024 in 32 bits)
      (uint64_t)p->n_beams * p->n_select * cdiv(p->vocab, 2048) > 0x7fff0000u) {
    set_error("beam_select: fewer continuations than n_select, or too many rows or candidates");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->ld_logits < p->vocab) {
    set_error("beam_select: rows of logits shorter than the vocabulary");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  return SYN_OK;
}

struct SelectSpace {
  int per, chunks;
  size_t stat, cand, total;
};
SelectSpace select_space(const syn_hip_beam_select_params &p) {
  const size_t rows = (size_t)p.n_groups * p.n_beams;
  SelectSpace s;
  // Chunks of 8192 logits; of 2048 where fewer than 128 would be at work (4 rows
  // of 32000, 16 chunks: 10.6 us against 9.5; 4 of 128256, 64: 10.6 and 10.1; 8 of
  // 128256, 128: 12.7 and 13.6; 32: 14.7 and 17.4).  At 128 rows of 151936 4096 a
  // chunk take 38 us where 8192 take 29.5, 16384 35: the lists that are joined,
  // and registers.
  s.per = rows * cdiv(p.vocab, kChunkNT * 32) >= 128 ? 32 : 8;
  s.chunks = (int)cdiv(p.vocab, (size_t)kChunkNT * s.per);
  s.stat = 0;
  s.cand = round_up(rows * s.chunks * sizeof(ChunkStat), 16);
  s.total = s.cand + round_up(rows * s.chunks * p.n_select * sizeof(Cand), 16);
  return s;
}

// ---------------------------------------------------------------- reordering
// One workgroup moves 64 units (of U bytes) of every row of a group: a unit's
// rows are all read before any is written, so the move is in place.  Bound by
// its bytes: 8 rows of 128 KiB in 48 buffers 11.2 us, 4.5 TB/s (a large copy
// reaches 4.8).
template <class U>
__global__ void __launch_bounds__(64)
    k_reorder_rows(const int32_t *parent, int W, uint8_t *rows, size_t units, size_t row_stride,
                   size_t buffer_stride) {
  extern __shared__ __align__(16) uint8_t raw[];
  U *stage = reinterpret_cast<U *>(raw);  // [W][64]
  const int l = threadIdx.x;
  const size_t u = (size_t)blockIdx.x * 64 + l, row0 = (size_t)blockIdx.y * W;
  const int32_t *par = parent + row0;
  uint8_t *base = rows + (size_t)blockIdx.z * buffer_stride + row0 * row_stride + u * sizeof(U);
  if (u >= units) return;
  for (int b = 0; b < W; b++) {
    const int p = par[b];
    if (p != b && (uint32_t)p < (uint32_t)W)
      stage[b * 64 + l] = *reinterpret_cast<const U *>(base + (size_t)p * row_stride);
  }
  for (int b = 0; b < W; b++) {
    const int p = par[b];
    if (p != b && (uint32_t)p < (uint32_t)W)
      *reinterpret_cast<U *>(base + (size_t)b * row_stride) = stage[b * 64 + l];
  }
}

struct PagesArgs {
  const int32_t *parent, *len;
  int32_t *table, *spare;
  size_t ld_table;
  int W;
  uint32_t n_pages;
  int n_layers, nkv, hd, ps, ps_shift, esz;
  uint8_t *k, *v;
};

// The positions a group holds: full pages, and those of the page after them.
__device__ __forceinline__ void held(const PagesArgs &a, int g, size_t *full, int *rest) {
  const long long room = (long long)a.ld_table << a.ps_shift;
  const long long n = min((long long)max(0, a.len[g]), room);
  *full = (size_t)(n >> a.ps_shift);
  *rest = (int)(n & (a.ps - 1));
}

// grid (layer * kv head, row): the parent's part of a page into the spare page.
// Bound by its bytes, 5.5 to 6 TB/s: 32 rows of 43 positions, 28 layers of 8 kv
// heads of 128, f16: 25 us, and 4 for the tables (parents are read by several
// rows, once from HBM).
__global__ void __launch_bounds__(256) k_copy_pages(PagesArgs a) {
  const int row = blockIdx.y, g = row / a.W, b = row - g * a.W;
  const int p = a.parent[row];
  size_t full;
  int rest;
  held(a, g, &full, &rest);
  if (p == b || (uint32_t)p >= (uint32_t)a.W || rest == 0) return;
  const int src = a.table[(size_t)(g * a.W + p) * a.ld_table + full], dst = a.spare[row];
  if ((uint32_t)src >= a.n_pages || (uint32_t)dst >= a.n_pages) return;
  const int n8 = (rest + 7) >> 3;  // groups of 8 positions
  const int layer = blockIdx.x / a.nkv, h = blockIdx.x - layer * a.nkv;
  const size_t head = (size_t)a.hd * a.ps * a.esz;
  const size_t off = (size_t)layer * a.n_pages;
  const size_t so = ((off + src) * a.nkv + h) * head, to = ((off + dst) * a.nkv + h) * head;
  const int v16 = n8 * a.hd * a.esz / 2;  // 16-byte units: 8 elements of each dim, whole groups
  for (int i = threadIdx.x; i < v16; i += 256)
    *reinterpret_cast<uint4 *>(a.v + to + (size_t)i * 16) =
        *reinterpret_cast<const uint4 *>(a.v + so + (size_t)i * 16);
  const int run = n8 * 4 * a.esz;  // 16-byte units of n8 * 8 positions at 8 dims
  const size_t pitch = (size_t)a.ps * 8 * a.esz;
  for (int i = threadIdx.x; i < run * (a.hd >> 3); i += 256) {
    const int c = i / run;
    const size_t o = c * pitch + (size_t)(i - c * run) * 16;
    *reinterpret_cast<uint4 *>(a.k + to + o) = *reinterpret_cast<const uint4 *>(a.k + so + o);
  }
}

// grid (columns / 64, group), after the copies: the waves take the rows in
// turn, all entries of a column are read before one is written
__global__ void __launch_bounds__(256) k_reorder_tables(PagesArgs a) {
  __shared__ int32_t stage[kMaxBeams][64];
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, g = blockIdx.y, W = a.W;
  const size_t col = (size_t)blockIdx.x * 64 + l;
  size_t full;
  int rest;
  held(a, g, &full, &rest);
  if ((size_t)blockIdx.x * 64 > full) return;
  const int32_t *par = a.parent + (size_t)g * W;
  int32_t *t = a.table + (size_t)g * W * a.ld_table + col, *spare = a.spare + (size_t)g * W;
  const bool gather = col < full;
#pragma unroll 4
  for (int b = wave; b < W; b += 4) {
    const int p = par[b];
    if (gather) stage[b][l] = t[((uint32_t)p < (uint32_t)W ? p : b) * a.ld_table];
  }
  __syncthreads();
#pragma unroll 4
  for (int b = wave; b < W; b += 4) {
    const int p = par[b];
    if (gather) {
      t[b * a.ld_table] = stage[b][l];
    } else if (col == full && col < a.ld_table && rest && p != b && (uint32_t)p < (uint32_t)W) {
      const int32_t mine = t[b * a.ld_table];
      t[b * a.ld_table] = spare[b];
      spare[b] = mine;
    }
  }
}

__global__ void __launch_bounds__(64)
    k_beam_advance(BeamCounters c, int n_beams, const uint32_t *token, uint32_t *history, size_t ld) {
  const int b = threadIdx.x, step = *c.step;
  __syncthreads();
  if (b < n_beams) {
    history[b * ld + step] = token[b];
    c.pos[b]++;
    c.index[b]++;
    c.len[b]++;
  }
  if (b == 0) *c.step = step + 1;
}

syn_status_t check_beams(size_t n_groups, size_t n_beams, const char *who) {
  if (!n_beams || n_beams > kMaxBeams || n_groups > 65535u / n_beams) {
    set_error(std::string(who) + ": 1 to 64 beams, at most 65535 rows");
    return SYN_ERR_INVALID_ARG;
  }
  return SYN_OK;
}

}  // namespace

syn_status_t launch_beam_advance(const BeamCounters &c, int n_beams, const uint32_t *token,
                                 uint32_t *history, size_t ld_history, hipStream_t s) {
  hipLaunchKernelGGL(k_beam_advance, dim3(1), dim3(64), 0, s, c, n_beams, token, history, ld_history);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // namespace syn

using namespace syn;

extern "C" {

syn_status_t syn_hip_beam_select_workspace(const syn_hip_beam_select_params *p, size_t *bytes) {
  if (!bytes) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_select(p));
  *bytes = select_space(*p).total;
  return SYN_OK;
}

syn_status_t syn_hip_beam_select(const syn_hip_beam_select_params *p, const float *d_logits,
                                 const float *d_scores, const int32_t *d_finished,
                                 int32_t *d_parent, uint32_t *d_token, float *d_score,
                                 int32_t *d_finished_out, void *d_workspace,
                                 size_t workspace_bytes, void *stream) {
  SYN_TRY(check_select(p));
  if (p->n_groups == 0) return SYN_OK;
  if (!d_logits || !d_scores || !d_parent || !d_token || !d_score || !d_workspace)
    return SYN_ERR_NULL_PTR;
  if (d_finished && (p->pad < 0 || (size_t)p->pad >= p->vocab)) {
    set_error("beam_select: pad outside the vocabulary");
    return SYN_ERR_INVALID_ARG;
  }
  const SelectSpace sp = select_space(*p);
  if (!aligned16(d_workspace) || workspace_bytes < sp.total) {
    set_error("beam_select: workspace unaligned or too small");
    return SYN_ERR_INVALID_ARG;
  }
  SYN_TRY(ensure_init());
  uint8_t *ws = static_cast<uint8_t *>(d_workspace);
  const SelectArgs a{d_logits, d_scores, d_finished, d_parent, d_finished_out, d_token, d_score,
                     reinterpret_cast<Cand *>(ws + sp.cand), reinterpret_cast<ChunkStat *>(ws),
                     p->ld_logits, (int)p->vocab, sp.chunks, (int)p->n_beams, (int)p->n_select,
                     p->eos, p->pad};
  hipStream_t s = pick_stream(stream);
  const dim3 grid((unsigned)sp.chunks, p->n_groups * p->n_beams);
  if (sp.per == 32)
    hipLaunchKernelGGL(k_beam_chunks<32>, grid, dim3(kChunkNT), 0, s, a);
  else
    hipLaunchKernelGGL(k_beam_chunks<8>, grid, dim3(kChunkNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_beam_merge, dim3(p->n_groups), dim3(kMergeNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

syn_status_t syn_hip_beam_reorder_rows(size_t n_groups, size_t n_beams, const int32_t *d_parent,
                                       void *d_rows, size_t row_bytes, size_t row_stride,
                                       size_t n_buffers, size_t buffer_stride, void *stream) {
  SYN_TRY(check_beams(n_groups, n_beams, "beam_reorder_rows"));
  const size_t rows = n_groups * n_beams;
  if (row_stride < row_bytes || (n_buffers > 1 && rows && buffer_stride < (rows - 1) * row_stride + row_bytes)) {
    set_error("beam_reorder_rows: rows or buffers overlap");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  if (n_buffers > 65535u) {
    set_error("beam_reorder_rows: at most 65535 buffers");
    return SYN_ERR_INVALID_ARG;
  }
  if (!n_groups || !row_bytes || !n_buffers) return SYN_OK;
  if (!d_parent || !d_rows) return SYN_ERR_NULL_PTR;
  const size_t all = reinterpret_cast<uintptr_t>(d_rows) | row_bytes | row_stride |
                     (n_buffers > 1 ? buffer_stride : 0);
  const size_t unit = all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1), units = row_bytes / unit;
  if (cdiv(units, 64) > kMaxThreads / 64) {
    set_error("beam_reorder_rows: rows too long for their alignment");
    return SYN_ERR_INVALID_ARG;
  }
  SYN_TRY(ensure_init());
  const dim3 grid((unsigned)cdiv(units, 64), (unsigned)n_groups, (unsigned)n_buffers);
  const size_t shm = n_beams * 64 * unit;
  hipStream_t s = pick_stream(stream);
  uint8_t *r = static_cast<uint8_t *>(d_rows);
  if (unit == 16)
    hipLaunchKernelGGL(k_reorder_rows<uint4>, grid, dim3(64), shm, s, d_parent, (int)n_beams, r,
                       units, row_stride, buffer_stride);
  else if (unit == 4)
    hipLaunchKernelGGL(k_reorder_rows<uint32_t>, grid, dim3(64), shm, s, d_parent, (int)n_beams, r,
                       units, row_stride, buffer_stride);
  else
    hipLaunchKernelGGL(k_reorder_rows<uint8_t>, grid, dim3(64), shm, s, d_parent, (int)n_beams, r,
                       units, row_stride, buffer_stride);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

syn_status_t syn_hip_beam_reorder_pages(const syn_hip_kv_pages *pages, size_t n_groups,
                                        size_t n_beams, const int32_t *d_parent,
                                        const int32_t *d_len, int32_t *d_table, size_t ld_table,
                                        int32_t *d_spare, void *stream) {
  SYN_TRY(check_pages(pages, "beam_reorder_pages"));
  SYN_TRY(check_beams(n_groups, n_beams, "beam_reorder_pages"));
  if ((uint64_t)pages->n_layers * pages->n_kv_heads > kMaxThreads / 256 ||
      cdiv(ld_table, 64) > kMaxThreads / 256) {
    set_error("beam_reorder_pages: too many layers, heads or table columns");
    return SYN_ERR_INVALID_ARG;
  }
  if (!n_groups || !ld_table) return SYN_OK;
  if (!d_parent || !d_len || !d_table || !d_spare) return SYN_ERR_NULL_PTR;
  SYN_TRY(ensure_init());
  const PagesArgs a{d_parent, d_len, d_table, d_spare, ld_table, (int)n_beams, pages->n_pages,
                    (int)pages->n_layers, (int)pages->n_kv_heads, (int)pages->head_dim,
                    (int)pages->page_size, 31 - __builtin_clz(pages->page_size),
                    (int)kv_elem_bytes(pages->dtype), static_cast<uint8_t *>(pages->k),
                    static_cast<uint8_t *>(pages->v)};
  hipStream_t s = pick_stream(stream);
  hipLaunchKernelGGL(k_copy_pages,
                     dim3(pages->n_layers * pages->n_kv_heads, (unsigned)(n_groups * n_beams)),
                     dim3(256), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_reorder_tables, dim3((unsigned)cdiv(ld_table, 64), (unsigned)n_groups),
                     dim3(256), 0, s, a);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // extern "C"
