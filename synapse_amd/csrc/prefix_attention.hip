// Attention of one query token per sequence over a paged cache, for groups of
// sequences that share a prefix.
//
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q k_j, in one pass
// with the running maximum m.  The query rows that read one kv head (of all
// members of a group over the prefix, of one sequence over its suffix) are the
// columns of two matrix products, S^T = K Q^T and O^T = V^T P^T, 16 rows to a
// tile: every key and value read serves all of them.  A wave takes 32
// positions at a time.  The pool's layout (kv_pages.hpp) is that of the
// products' operands, so K and V go from memory to registers to the matrix
// cores with no LDS between; and with positions 8g .. 8g+7 in rows 4g .. 4g+3
// of two 16-row tiles of S^T, the lanes that hold the weights of a query row
// are those that the second product wants them in, so P needs none either.
//
// Precision: queries and weights are f32 and stay so: for a 16-bit pool each
// is split into parts of the pool's type (two f16 carry 22 bits, three bf16
// carry 24) whose products with the stored K and V are exact in the f32
// accumulators; an f32 pool takes the f32 matrix instructions.
#include <algorithm>
#include <cmath>

#include "kv_pages.hpp"

namespace syn {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kWaves = 4;
constexpr int kTile = 32;  // positions a wave takes at a time

struct AttnArgs {
  const float *q;
  const int32_t *ptable, *plen, *table, *slen;
  float *out;
  size_t ldq, ldo, ld_ptable, ld_table;
  int nh, rep, group_size, n_seqs, max_prefix, max_suffix;
  float scale;  // times log2(e): exponentials are powers of two
  // the split: positions of a part (a multiple of kTile * kWaves), parts of
  // the longest prefix and suffix; parts of query row (sequence, head) are
  // po[(sequence * nh + head) * (npp + nsp) + part][hd], pml[..][2] (max, sum)
  int pchunk, schunk, npp, nsp;
  float *po, *pml;
};

// ---------------------------------------------------------------- products
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct f32x8 {
  f32x4 lo, hi;
};

template <class T> struct Frag;
template <> struct Frag<_Float16> {
  using V = f16x8;
  static constexpr int kParts = 2;
  // A weight is at least 2^kBias where its score is the reference maximum, so
  // that the second part of the small ones is still a normal f16.
  static constexpr float kBias = 6.0f;
  static __device__ __forceinline__ V load(const _Float16 *p) {
    return *reinterpret_cast<const V *>(p);
  }
  static __device__ __forceinline__ void split(const float *x, V *p) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      p[0][j] = (_Float16)x[j];
      p[1][j] = (_Float16)__builtin_fmaf((float)p[0][j], -1.0f, x[j]);
    }
  }
  static __device__ __forceinline__ f32x4 mma(const V &a, const V *b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b[0], c, 0, 0, 0);
  }
  static __device__ __forceinline__ void clear(V &v, int j) { v[j] = (_Float16)0.0f; }
};
template <> struct Frag<__bf16> {
  using V = bf16x8;
  static constexpr int kParts = 3;
  static constexpr float kBias = 0.0f;
  static __device__ __forceinline__ V load(const __bf16 *p) {
    return *reinterpret_cast<const V *>(p);
  }
  static __device__ __forceinline__ void split(const float *x, V *p) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      p[0][j] = (__bf16)x[j];
      const float r = x[j] - (float)p[0][j];
      p[1][j] = (__bf16)r;
      p[2][j] = (__bf16)(r - (float)p[1][j]);
    }
  }
  static __device__ __forceinline__ f32x4 mma(const V &a, const V *b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[0], c, 0, 0, 0);
  }
  static __device__ __forceinline__ void clear(V &v, int j) { v[j] = (__bf16)0.0f; }
};
template <> struct Frag<float> {
  using V = f32x8;
  static constexpr int kParts = 1;
  static constexpr float kBias = 0.0f;
  static __device__ __forceinline__ V load(const float *p) {
    return V{*reinterpret_cast<const f32x4 *>(p), *reinterpret_cast<const f32x4 *>(p + 4)};
  }
  static __device__ __forceinline__ void split(const float *x, V *p) {
#pragma unroll
    for (int j = 0; j < 4; j++) p[0].lo[j] = x[j], p[0].hi[j] = x[j + 4];
  }
  // element j of every lane is one step of four of the contraction
  static __device__ __forceinline__ f32x4 mma(const V &a, const V *b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[j], b->lo[j], c, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[j], b->hi[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ void clear(V &v, int j) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (i == j) v.lo[i] = 0.0f;
      if (i + 4 == j) v.hi[i] = 0.0f;
    }
  }
};

// over the four groups of 16 lanes
__device__ __forceinline__ float groups_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float groups_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// What a workgroup works on: query rows row0 .. row0 + rows of kv head `head`
// (row = member * rep + its query head), and up to two runs of positions.
struct Run {
  const int32_t *table;
  int from, to, len;  // positions from .. min(to, len)
};

// RT: tiles of 16 query rows; NC: 32 dims each (hd <= 32 NC)
template <class T, int NC, int RT> struct Attend {
  using F = Frag<T>;
  using V = typename F::V;
  static constexpr int DT = 2 * NC;
  V q[RT][NC][F::kParts];
  f32x4 o[RT][DT];
  float m[RT], l[RT], unscale[RT];

  // the rows' queries times scale, each row of an f16 pool times the power of
  // two that puts its largest element into [2^11, 2^12): both parts of every
  // element that matters are normal
  __device__ __forceinline__ void load_queries(const AttnArgs &a, int hd, int seq0, int head, int row0,
                                               int rows) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const int r = row0 + t * 16 + n;
      const bool on = t * 16 + n < rows;
      const int member = on ? r / a.rep : 0;
      const float *src = a.q + (size_t)(seq0 + member) * a.ldq +
                         (size_t)(head * a.rep + (on ? r - member * a.rep : 0)) * hd;
      float x[NC][8], top = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const int d = (c * 4 + g) * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[c][j] = on && d < hd ? src[d + j] * a.scale : 0.0f;
          top = fmaxf(top, fabsf(x[c][j]));
        }
      }
      int e = 0;
      if constexpr (F::kParts == 2) {
        top = groups_max(top);
        if (top > 0.0f && top < __builtin_huge_valf()) e = 11 - ilogbf(top);
        // a power of two within f32's own range either way
        e = min(max(e, -120), 120);
      }
      const float up = __builtin_ldexpf(1.0f, e);
      unscale[t] = __builtin_ldexpf(1.0f, -e);
#pragma unroll
      for (int c = 0; c < NC; c++) {
        if constexpr (F::kParts == 2)
#pragma unroll
          for (int j = 0; j < 8; j++) x[c][j] *= up;
        F::split(x[c], q[t][c]);
      }
      m[t] = kNegInf;
      l[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; d++) o[t][d] = f32x4{0, 0, 0, 0};
    }
  }

  // the wave's tiles of a run: kTile positions every kTile * kWaves
  __device__ __forceinline__ void run(const KvPool<T> &pool, int head, int rows, const Run &r) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int to = min(r.to, r.len), hd = pool.hd, d8 = hd >> 3;
    const int last = (to - 1) & ~7;  // the last group of 8 positions
    for (int k0 = r.from + wave * kTile; k0 < to; k0 += kTile * kWaves) {
      // lane (g, n): K of the 8 positions of group n / 4, V of those of group g
      const int kk = min(k0 + 8 * (n >> 2), last), kv = min(k0 + 8 * g, last);
      int pk = r.table[kk >> pool.ps_shift], pv = r.table[kv >> pool.ps_shift];
      const bool has_k = pool.has(pk), has_v = pool.has(pv);
      // whole: every position of the tile is there
      const bool whole = __all(k0 + kTile <= to && has_k && has_v);
      pk = has_k ? pk : 0;
      pv = has_v ? pv : 0;
      const T *kp = pool.k + pool.base(pk, head) + (size_t)((kk & (pool.ps - 1)) + (n & 3)) * 8;
      const T *vp = pool.v + pool.base(pv, head) + (size_t)((kv & (pool.ps - 1)) >> 3) * hd * 8;
      V kf[2][NC], vf[DT];
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const size_t at = (size_t)min(c * 4 + g, d8 - 1) * pool.ps * 8;
        kf[0][c] = F::load(kp + at);
        kf[1][c] = F::load(kp + at + 32);
      }
#pragma unroll
      for (int d = 0; d < DT; d++) vf[d] = F::load(vp + (size_t)min(d * 16 + n, hd - 1) * 8);
      uint32_t there = 0xff;  // of the positions 8g .. 8g+7 whose weights this lane holds
      if (!whole) {
        const int left = has_v ? to - (k0 + 8 * g) : 0;
        there = left >= 8 ? 0xff : (left <= 0 ? 0 : (1u << left) - 1);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (!(there >> j & 1)) F::clear(vf[d], j);
      }
#pragma unroll
      for (int t = 0; t < RT; t++) {
        if (RT > 1 && t * 16 >= rows) break;
        f32x4 s0{0, 0, 0, 0}, s1{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NC; c++) {
          s0 = F::mma(kf[0][c], q[t][c], s0);
          s1 = F::mma(kf[1][c], q[t][c], s1);
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = s0[j] * unscale[t], x[j + 4] = s1[j] * unscale[t];
        if (!whole)
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = there >> j & 1 ? x[j] : kNegInf;
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; j++) top = fmaxf(top, x[j]);
        top = fmaxf(groups_max(top), m[t]);
        const float ref = top == kNegInf ? 0.0f : top;
        const float back = __builtin_amdgcn_exp2f(m[t] - ref);
        m[t] = top;
        l[t] *= back;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[j] = __builtin_amdgcn_exp2f(x[j] - ref + F::kBias);
          l[t] += x[j];
        }
        V p[F::kParts];
        F::split(x, p);
#pragma unroll
        for (int d = 0; d < DT; d++) {
          o[t][d] *= back;
          o[t][d] = F::mma(vf[d], p, o[t][d]);
        }
      }
    }
  }

  // the four waves' results joined, in the order of the waves; a row's goes to
  // the output, or to its part of the workspace
  __device__ __forceinline__ void finish(const AttnArgs &a, int hd, int seq0, int head, int row0, int rows,
                                         int part, float *buf, float *ml) {
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4, wave = tid >> 6;
    constexpr int LD = 32 * NC + 4;  // rows on different banks
#pragma unroll
    for (int t = 0; t < RT; t++) {
      if (t * 16 >= rows) break;
      const float sum = groups_sum(l[t]);
      __syncthreads();
      if (g == 0) ml[(wave * 16 + n) * 2] = m[t], ml[(wave * 16 + n) * 2 + 1] = sum;
      __syncthreads();
      float top = ml[n * 2];
#pragma unroll
      for (int w = 1; w < kWaves; w++) top = fmaxf(top, ml[(w * 16 + n) * 2]);
      const float f = m[t] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m[t] - top);
#pragma unroll
      for (int d = 0; d < DT; d++)
        *reinterpret_cast<f32x4 *>(buf + (wave * 16 + n) * LD + d * 16 + g * 4) = o[t][d] * f;
      __syncthreads();
      for (int i = tid; i < 16 * hd; i += 64 * kWaves) {
        const int r = i / hd, d = i - r * hd;
        if (t * 16 + r >= rows) break;
        float mx = ml[r * 2], ls = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; w++) mx = fmaxf(mx, ml[(w * 16 + r) * 2]);
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
          const float mw = ml[(w * 16 + r) * 2];
          x += buf[(w * 16 + r) * LD + d];
          // (the sum of a wave with no position is 0, or NaN if its scores were)
          ls += ml[(w * 16 + r) * 2 + 1] * (mw == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mw - mx));
        }
        const int row = row0 + t * 16 + r, member = row / a.rep;
        const size_t qh = (size_t)head * a.rep + (row - member * a.rep), seq = seq0 + member;
        if (part < 0) {
          a.out[seq * a.ldo + qh * hd + d] = ls == 0.0f ? 0.0f : x / ls;
        } else {
          const size_t at = (seq * a.nh + qh) * (a.npp + a.nsp) + part;
          a.po[at * hd + d] = x;
          if (d == 0) a.pml[at * 2] = mx, a.pml[at * 2 + 1] = ls;
        }
      }
    }
  }
};

__device__ __forceinline__ int clamped(const int32_t *len, int i, int most) {
  return most ? max(0, min(len[i], most)) : 0;
}

// kJoined: one workgroup has both runs of a sequence whole; else the parts of
// the prefixes, or of the suffixes
enum { kJoined, kPrefix, kSuffix };

template <class T, int NC, int RT, int WHAT>
__global__ void __launch_bounds__(64 * kWaves) k_attend(AttnArgs a, KvPool<T> pool) {
  __shared__ __align__(16) float buf[kWaves * 16 * (32 * NC + 4)];
  __shared__ float ml[kWaves * 16 * 2];
  const int members = WHAT == kPrefix ? a.group_size : 1;  // sequences whose rows go together
  const int all = members * a.rep, blocks = (all + RT * 16 - 1) / (RT * 16);
  const int parts = WHAT == kPrefix ? a.npp : (WHAT == kSuffix ? a.nsp : 1);
  // workgroup i runs on XCD i % 8: the blocks of rows that read the same
  // positions come 8 apart and share that XCD's L2
  const int i = blockIdx.x, j = i >> 3;
  const int unit = (j / blocks) * 8 + (i & 7), block = j % blocks;
  const int head = unit % pool.nkv, u = unit / pool.nkv;
  const int part = u % parts, owner = u / parts;  // group or sequence
  if (owner * members >= a.n_seqs) return;
  const int seq0 = owner * members, row0 = block * RT * 16, rows = min(RT * 16, all - row0);
  const int group = WHAT == kPrefix ? owner : owner / a.group_size;
  const int plen = WHAT == kSuffix ? 0 : clamped(a.plen, group, a.max_prefix);
  const int slen = WHAT == kPrefix ? 0 : clamped(a.slen, seq0, a.max_suffix);
  const int32_t *pt = a.ptable + (size_t)group * a.ld_ptable;
  const int32_t *st = a.table + (size_t)seq0 * a.ld_table;
  Attend<T, NC, RT> w;
  if (WHAT != kJoined) {
    const int len = WHAT == kPrefix ? plen : slen, chunk = WHAT == kPrefix ? a.pchunk : a.schunk;
    const int from = part * chunk;
    if (from >= len) {  // nothing here: no rows to write, a sum of 0
      for (int r = threadIdx.x; r < rows; r += 64 * kWaves) {
        const int row = row0 + r, member = row / a.rep;
        const size_t at = ((size_t)(seq0 + member) * a.nh + (size_t)head * a.rep +
                           (row - member * a.rep)) * (a.npp + a.nsp) +
                          (WHAT == kPrefix ? part : a.npp + part);
        a.pml[at * 2] = kNegInf;
        a.pml[at * 2 + 1] = 0.0f;
      }
      return;
    }
    w.load_queries(a, pool.hd, seq0, head, row0, rows);
    w.run(pool, head, rows, Run{WHAT == kPrefix ? pt : st, from, min(from + chunk, len), len});
    w.finish(a, pool.hd, seq0, head, row0, rows, WHAT == kPrefix ? part : a.npp + part, buf, ml);
  } else {
    w.load_queries(a, pool.hd, seq0, head, row0, rows);
    for (int k = 0; k < 2; k++) {
      const int len = k ? slen : plen;
      w.run(pool, head, rows, Run{k ? st : pt, 0, len, len});
    }
    w.finish(a, pool.hd, seq0, head, row0, rows, -1, buf, ml);
  }
}

// one wave a query row: the parts in order
__global__ void __launch_bounds__(256) k_join_parts(AttnArgs a, int hd) {
  const int lane = threadIdx.x & 63;
  const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (size_t)a.n_seqs * a.nh) return;
  const int n = a.npp + a.nsp;
  const float *ml = a.pml + row * n * 2, *po = a.po + row * n * hd;
  float top = kNegInf;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, ml[2 * i]);
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  float x[4] = {0, 0, 0, 0}, l = 0.0f;
  for (int i = 0; i < n; i++) {
    const float lp = ml[2 * i + 1];
    if (lp == 0.0f) continue;
    const float f = __builtin_amdgcn_exp2f(ml[2 * i] - top);
    l += lp * f;
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (lane + 64 * k < hd) x[k] = __builtin_fmaf(po[(size_t)i * hd + lane + 64 * k], f, x[k]);
  }
  const size_t seq = row / a.nh, head = row - seq * a.nh;
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (lane + 64 * k < hd)
      a.out[seq * a.ldo + head * hd + lane + 64 * k] = l == 0.0f ? 0.0f : x[k] / l;
}

// ---------------------------------------------------------------- host
syn_status_t check_attention(const syn_hip_kv_pages *pages,
                             const syn_hip_prefix_attention_params *p) {
  if (!p) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_pages(pages, "prefix_attention"));
  const size_t hd = pages->head_dim, rows = (size_t)p->n_groups * p->group_size;
  if (p->layer >= pages->n_layers || !p->n_heads || p->n_heads % pages->n_kv_heads ||
      p->n_heads > 65535u) {
    set_error("prefix_attention: layer outside the pool, or n_heads no multiple of n_kv_heads");
    return SYN_ERR_INVALID_ARG;
  }
  if (rows > 65535u || p->max_prefix > 0x7fffff00u || p->max_suffix > 0x7fffff00u) {
    set_error("prefix_attention: more than 65535 sequences or 2^31 positions");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->ldq < p->n_heads * hd || p->ldo < p->n_heads * hd ||
      p->ld_prefix_table < cdiv(p->max_prefix, pages->page_size) ||
      p->ld_table < cdiv(p->max_suffix, pages->page_size)) {
    set_error("prefix_attention: rows or page tables shorter than the heads or the lengths");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  return SYN_OK;
}

// tiles of 16 query rows that a workgroup holds: the registers allow 4 (two
// parts of 64 dims) to 1
int row_tiles(int nc, int parts, int rows) {
  const int most = nc * parts <= 8 ? 4 : (nc <= 4 ? 2 : 1);
  const int need = (rows + 15) / 16;
  return need >= 3 && most == 4 ? 4 : (need >= 2 && most >= 2 ? 2 : 1);
}

struct Plan {
  bool joined;
  int nc, prt, srt;      // dims, row tiles of prefix and suffix workgroups
  int pchunk, schunk, npp, nsp;
  size_t rows, po_bytes, pml_bytes;
};

Plan make_plan(const syn_hip_kv_pages &pg, const syn_hip_prefix_attention_params &p) {
  Plan w{};
  const int hd = (int)pg.head_dim, nkv = (int)pg.n_kv_heads, rep = (int)p.n_heads / nkv;
  const int parts = pg.dtype == SYN_HIP_KV_F32 ? 2 : (pg.dtype == SYN_HIP_KV_F16 ? 2 : 3);
  w.nc = hd <= 64 ? 2 : (hd <= 128 ? 4 : 8);
  w.rows = (size_t)p.n_groups * p.group_size * p.n_heads;
  w.prt = row_tiles(w.nc, parts, (int)p.group_size * rep);
  w.srt = row_tiles(w.nc, parts, rep);
  const size_t step = kTile * kWaves, seqs = (size_t)p.n_groups * p.group_size;
  w.joined = (size_t)p.max_prefix + p.max_suffix <= 4 * step;
  if (w.joined) return w;
  // parts enough for two workgroups a CU
  auto cut = [&](size_t items, size_t len, int *chunk, int *n) {
    const size_t tiles = cdiv(len, step), want = std::max<size_t>(1, cdiv(512, items));
    const size_t per = std::max<size_t>(1, cdiv(tiles, want));
    *chunk = (int)(per * step);
    *n = (int)cdiv(tiles, per);
  };
  const size_t pblocks = cdiv((size_t)p.group_size * rep, 16 * w.prt);
  cut(std::max<size_t>(1, p.n_groups * nkv * pblocks), p.max_prefix, &w.pchunk, &w.npp);
  cut(std::max<size_t>(1, seqs * nkv * cdiv(rep, 16 * w.srt)), p.max_suffix, &w.schunk, &w.nsp);
  const size_t n = w.rows * (size_t)(w.npp + w.nsp);
  w.po_bytes = round_up(n * hd * 4, 16);
  w.pml_bytes = round_up(n * 8, 16);
  return w;
}

template <class T, int NC, int RT, int WHAT>
syn_status_t launch_one(const AttnArgs &a, const KvPool<T> &pool, hipStream_t s) {
  const size_t members = WHAT == kPrefix ? a.group_size : 1;
  const size_t blocks = cdiv(members * a.rep, RT * 16);
  const size_t parts = WHAT == kPrefix ? a.npp : (WHAT == kSuffix ? a.nsp : 1);
  const size_t units = round_up(a.n_seqs / members * parts * pool.nkv, 8);
  if (units * blocks > 0x7fffffffu) {
    set_error("prefix_attention: more workgroups than a launch takes");
    return SYN_ERR_INVALID_ARG;
  }
  hipLaunchKernelGGL((k_attend<T, NC, RT, WHAT>), dim3((unsigned)(units * blocks)),
                     dim3(64 * kWaves), 0, s, a, pool);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

template <class T, int NC, int WHAT>
syn_status_t launch_rt(int rt, const AttnArgs &a, const KvPool<T> &pool, hipStream_t s) {
  if constexpr (NC * (Frag<T>::kParts == 3 ? 3 : 2) <= 8)
    if (rt == 4) return launch_one<T, NC, 4, WHAT>(a, pool, s);
  if constexpr (NC <= 4)
    if (rt >= 2) return launch_one<T, NC, 2, WHAT>(a, pool, s);
  return launch_one<T, NC, 1, WHAT>(a, pool, s);
}

template <class T, int NC>
syn_status_t launch_nc(const Plan &w, const AttnArgs &a, const KvPool<T> &pool, hipStream_t s) {
  if (w.joined) return launch_rt<T, NC, kJoined>(w.srt, a, pool, s);
  if (w.npp) SYN_TRY((launch_rt<T, NC, kPrefix>(w.prt, a, pool, s)));
  if (w.nsp) SYN_TRY((launch_rt<T, NC, kSuffix>(w.srt, a, pool, s)));
  hipLaunchKernelGGL(k_join_parts, dim3((unsigned)cdiv(w.rows, 4)), dim3(256), 0, s, a, pool.hd);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // namespace

}  // namespace syn

using namespace syn;

extern "C" syn_status_t syn_hip_prefix_attention_workspace(
    const syn_hip_kv_pages *pages, const syn_hip_prefix_attention_params *p, size_t *bytes) {
  if (!bytes) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_attention(pages, p));
  const Plan w = make_plan(*pages, *p);
  *bytes = w.po_bytes + w.pml_bytes;
  return SYN_OK;
}

extern "C" syn_status_t syn_hip_prefix_attention(
    const syn_hip_kv_pages *pages, const syn_hip_prefix_attention_params *p, const float *d_q,
    const int32_t *d_prefix_table, const int32_t *d_prefix_len, const int32_t *d_table,
    const int32_t *d_len, float *d_out, void *d_workspace, size_t workspace_bytes, void *stream) {
  SYN_TRY(check_attention(pages, p));
  const size_t rows = (size_t)p->n_groups * p->group_size;
  if (rows == 0) return SYN_OK;
  if (!d_q || !d_out || (p->max_prefix && (!d_prefix_table || !d_prefix_len)) ||
      (p->max_suffix && (!d_table || !d_len)))
    return SYN_ERR_NULL_PTR;
  const Plan w = make_plan(*pages, *p);
  const size_t need = w.po_bytes + w.pml_bytes;
  if (need && !d_workspace) return SYN_ERR_NULL_PTR;
  if (need && (!aligned16(d_workspace) || workspace_bytes < need)) {
    set_error("prefix_attention: workspace unaligned or too small");
    return SYN_ERR_INVALID_ARG;
  }
  SYN_TRY(ensure_init());
  AttnArgs a{};
  a.q = d_q;
  a.ptable = d_prefix_table;
  a.plen = d_prefix_len;
  a.table = d_table;
  a.slen = d_len;
  a.out = d_out;
  a.ldq = p->ldq;
  a.ldo = p->ldo;
  a.ld_ptable = p->ld_prefix_table;
  a.ld_table = p->ld_table;
  a.nh = (int)p->n_heads;
  a.rep = (int)(p->n_heads / pages->n_kv_heads);
  a.group_size = (int)p->group_size;
  a.n_seqs = (int)rows;
  a.max_prefix = (int)p->max_prefix;
  a.max_suffix = (int)p->max_suffix;
  a.scale = (p->scale != 0.0f ? p->scale : 1.0f / sqrtf((float)pages->head_dim)) * kLog2e;
  a.pchunk = w.pchunk;
  a.schunk = w.schunk;
  a.npp = w.npp;
  a.nsp = w.nsp;
  a.po = static_cast<float *>(d_workspace);
  a.pml = reinterpret_cast<float *>(static_cast<uint8_t *>(d_workspace) + w.po_bytes);
  hipStream_t s = pick_stream(stream);
  return kv_dispatch(pages->dtype, [&](auto t) -> syn_status_t {
    using T = decltype(t);
    const KvPool<T> pool = kv_pool<T>(*pages, p->layer);
    if (w.nc == 2) return launch_nc<T, 2>(w, a, pool, s);
    if (w.nc == 4) return launch_nc<T, 4>(w, a, pool, s);
    return launch_nc<T, 8>(w, a, pool, s);
  });
}
