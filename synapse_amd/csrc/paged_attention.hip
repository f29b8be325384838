// Causal attention of the new tokens of each sequence over its pages: one token
// (decoding), a few (drafts to be verified), many (a prompt's chunk).
//
// Row j of a sequence's n new tokens, which are the last n of its len positions,
// is softmax(scale q k_i) over i from len - n + j back, as far as the window
// reaches.  The rows of a kv head, all tokens' query heads that read it, are the
// columns of the two products of attend_rows.hpp, 16, 32 or 64 to a workgroup: a
// key or value that several tokens see is read for all of them at once.  A row's
// own limits only mask its scores, in the tiles that some row of the wave does not
// see whole; positions that no row of the workgroup sees are not read.  The second
// product multiplies values by weights of 0 there, so in those tiles values that are
// not finite are taken out of it, and the rows that do see them made NaN (no more
// than 1.5 % of a call; most measure no difference).
//
// What bounds it (a large copy reaches 4.7 TB/s here, large products 1100 TFLOP/s
// in f16): up to 32 rows of a kv head, bytes: 64 sequences of one token at up to
// 12000 positions, 32 heads of 64, bf16, 211 us, 5.6 TB/s; 24 of up to 8 tokens at
// 8200, 32 heads of 128, f16, 131 to 143 us, 4.7 to 4.3 TB/s.  Chunks, their steps
// of a tile: two of 1536 tokens at 12001, 24 heads of 128, f16, 661 to 760 us, 483
// to 555 TFLOP/s of the formula and twice that in matrix instructions with the
// operands' second parts, which take 51 % of the SIMDs' cycles, the vector ones 60 %
// (with two workgroups a CU 815 to 893 us, 41 and 48 %): a wave's scores, weights and
// values of a tile come one after the other.  Four sequences of five tokens at 213,
// f32: 10.1 us, one launch and dependent loads.
#include <algorithm>
#include <cmath>

#include "attend_rows.hpp"

namespace syn {

namespace {

struct PagedArgs : RowArgs {
  const int32_t *start, *len, *table;
  size_t ld_table;
  int n_seqs, n_tokens, max_new, max_len, window;
  int chunk;   // positions of a part (a multiple of kTile)
  int blocks;  // workgroups for the rows of the longest sequence
  bool solo;   // a wave for a sequence's rows
};

__device__ __forceinline__ int scalar(const int32_t *p, int i) {
  const auto *t = (const __attribute__((address_space(4))) int32_t *)(uintptr_t)p;  // a scalar load
  return t[i];
}
// a sequence's new tokens: the first one's row, and how many
__device__ __forceinline__ int first_of(const PagedArgs &a, int s) {
  return a.start ? min(max(scalar(a.start, s), 0), a.n_tokens) : s * a.max_new;
}
__device__ __forceinline__ int count_of(const PagedArgs &a, int s, int first) {
  const int end = a.start ? min(max(scalar(a.start, s + 1), first), a.n_tokens) : first + a.max_new;
  return min(end - first, a.max_new);
}

// 64 rows of 128 dims in 16 bits: a ring of three tiles and 168 registers leave
// room for three workgroups a CU (30 chunks of 100 tokens at 1000, 32 heads of 128,
// f16, 92 us, 107 with two; two of 1200 at 9000, bf16, 752 and 789).  Four in f16
// would have to spill.  (Of all instances one does: f32, heads of 136 to 248, 16 rows
// to a workgroup, 98 registers, 216 bytes a lane.)
template <class T, int NC, int RW> constexpr bool kThree = RW == 4 && NC == 4 && sizeof(T) == 2;

// 16 rows of 64 dims in f16: 128 registers, four workgroups a CU (130 without the bound)
template <class T, int NC, int RW> constexpr bool kFour = RW == 1 && NC == 2 && Frag<T>::kParts == 2;

// RW: tiles of 16 rows of a workgroup
template <class T, int NC, bool FULL, int RW>
__global__ void __launch_bounds__(64 * kWaves, (kThree<T, NC, RW>          ? 3
                                                : kFour<T, NC, RW> && FULL ? 4
                                                                           : kResident<T, NC, FULL>))
    k_attend_new(PagedArgs a, KvPool<T> pool) {
  using W = Rows<T, NC, FULL, true, kThree<T, NC, RW> ? 3 : 0>;
  __shared__ __align__(16) uint8_t lds[W::kLdsBytes];
  __shared__ float ml[kWaves * 16 * 2];
  // workgroup i runs on XCD i % 8: the blocks of rows that read the same
  // positions come 8 apart and share that XCD's L2; the last rows, which see
  // most, go first
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = blockIdx.x, j = i >> 3, block = a.blocks - 1 - j % a.blocks;
  int unit = (j / a.blocks) * 8 + (i & 7);
  if (a.solo) unit = unit * kWaves + wave;
  const int head = unit % pool.nkv, u = unit / pool.nkv;
  const int part = u % a.parts, s = u / a.parts;
  if (s >= a.n_seqs) return;
  const int first = first_of(a, s), count = count_of(a, s, first), all = count * a.rep;
  const int row0 = block * RW * 16, rows = min(RW * 16, all - row0);
  if (rows <= 0) return;
  const int len = min(max(scalar(a.len, s), 0), a.max_len);
  // token j sees the positions below lim_of(j), from lo_of(j) on
  auto lim_of = [&](int token) { return len - count + token + 1; };
  auto lo_of = [&](int token) { return a.window && lim_of(token) > a.window ? lim_of(token) - a.window : 0; };
  const int last = row0 + rows - 1;
  const int to = max(0, lim_of(last / a.rep)), from = min(lo_of(row0 / a.rep) & ~(kTile - 1), to);
  Run r{a.table + (size_t)s * a.ld_table, from, to, 0};
  int at = -1;
  if (a.parts > 1) {
    at = part;
    const int64_t begin = from + (int64_t)part * a.chunk;
    if (begin >= to) {  // nothing here: no rows to write, a sum of 0
      for (int k = a.solo ? (int)threadIdx.x & 63 : (int)threadIdx.x; k < rows; k += 64 * kWaves) {
        const int row = row0 + k, token = row / a.rep;
        const size_t p = ((size_t)(first + token) * a.nh + (size_t)head * a.rep + (row - token * a.rep)) * a.parts + at;
        a.pml[p * 2] = kNegInf;
        a.pml[p * 2 + 1] = 0.0f;
      }
      return;
    }
    r.from = (int)begin;
    r.to = r.from + min(a.chunk, to - r.from);
  }
  const size_t head_bytes = (size_t)pool.hd * pool.ps * sizeof(T);
  const HeadBase hb{reinterpret_cast<const uint8_t *>(pool.k) + head * head_bytes,
                    reinterpret_cast<const uint8_t *>(pool.v) + head * head_bytes,
                    (uint32_t)(pool.nkv * head_bytes)};
  const bool wide = pool.ps >= kTile;
  uint32_t ok = 0;
  if constexpr (RW > 1)
    ok = wide ? W::template start_shared<true, 4 / RW>(pool, hb, r, lds)
              : W::template start_shared<false, 4 / RW>(pool, hb, r, lds);
  W w;
  const int mine = row0 + (wave & (RW - 1)) * 16;
  w.load_queries(a, pool.hd, first, head, mine, last);
  {
    const int token = min(mine + (int)(threadIdx.x & 15), last) / a.rep;
    w.see(lo_of(token), lim_of(token), lo_of(min(mine + 15, last) / a.rep), lim_of(min(mine, last) / a.rep));
  }
  if constexpr (RW == 1) {
    if (wide)
      w.template run_alone<true>(pool, hb, r, a.solo ? 1 : kWaves);
    else
      w.template run_alone<false>(pool, hb, r, a.solo ? 1 : kWaves);
    if (a.solo) {
      w.finish_alone(a, pool.hd, first, head, row0, rows, at);
      return;
    }
  } else if (wide) {
    w.template run_shared<true, 4 / RW>(pool, hb, r, lds, ok);
  } else {
    w.template run_shared<false, 4 / RW>(pool, hb, r, lds, ok);
  }
  w.finish(a, pool.hd, first, head, row0, rows, RW, at, reinterpret_cast<float *>(lds), ml);
}

// a query row of a sequence to a workgroup (those past its last token leave)
template <int LANES> __global__ void __launch_bounds__(256) k_join_new(PagedArgs a, int hd) {
  const size_t row = blockIdx.x / a.nh;
  const int head = blockIdx.x - row * a.nh, s = row / a.max_new, token = row - (size_t)s * a.max_new;
  const int first = first_of(a, s);
  if (token >= count_of(a, s, first)) return;
  join_parts<LANES>(a, hd, (size_t)(first + token) * a.nh + head);
}

constexpr int kFewParts = 16;

// ... or, of few parts, to LANES lanes with four dims each, all parts in flight
// together (6144 rows of three parts of 128 dims 13.6 us with a workgroup each).
template <int LANES> __global__ void __launch_bounds__(256) k_join_few(PagedArgs a, int hd, uint32_t rows) {
  const uint32_t at = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (at >= rows) return;
  const uint32_t row = at / a.nh, head = at - row * a.nh;
  const int s = row / a.max_new, token = row - (uint32_t)s * a.max_new, c4 = 4 * (threadIdx.x % LANES);
  const int start = a.start ? a.start[s] : 0, end = a.start ? a.start[s + 1] : 0;
  const int first = a.start ? min(max(start, 0), a.n_tokens) : s * a.max_new;
  const int count = a.start ? min(min(max(end, first), a.n_tokens) - first, a.max_new) : a.max_new;
  if (token >= count || c4 >= hd) return;
  const size_t q = (size_t)(first + token) * a.nh + head;
  const float *ml = a.pml + q * a.parts * 2, *po = a.po + q * a.parts * hd + c4;
  const int n = a.parts;
  float m[kFewParts], l[kFewParts], top = kNegInf, sum = 0.0f;
  f32x4 y[kFewParts], x{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kFewParts; i++)
    if (i < n) {
      m[i] = ml[2 * i];
      l[i] = ml[2 * i + 1];
      y[i] = *reinterpret_cast<const f32x4 *>(po + (size_t)i * hd);
    }
#pragma unroll
  for (int i = 0; i < kFewParts; i++)
    if (i < n) top = fmaxf(top, m[i]);
#pragma unroll
  for (int i = 0; i < kFewParts; i++)
    if (i < n && l[i] != 0.0f) {  // (a part with no position has left its row unwritten)
      const float f = __builtin_amdgcn_exp2f(m[i] - top);
      sum = __builtin_fmaf(l[i], f, sum);
#pragma unroll
      for (int c = 0; c < 4; c++) x[c] = __builtin_fmaf(y[i][c], f, x[c]);
    }
  float *out = a.out + (size_t)(first + token) * a.ldo + (size_t)head * hd + c4;
#pragma unroll
  for (int c = 0; c < 4; c++) out[c] = sum == 0.0f ? 0.0f : x[c] / sum;
}

// ---------------------------------------------------------------- host
constexpr double kMostSpace = 192 << 20;  // of a workspace, where runs need not be split
constexpr size_t kMostWgs = kMaxThreads / (64 * kWaves);  // of a launch, of either kernel

struct Plan {
  bool solo;
  int nc, rw, blocks, chunk, parts;
  size_t seqs;  // of a launch; 0: not even one
  size_t po_bytes, pml_bytes;
  size_t wgs(size_t n, size_t nkv) const {
    return round_up(solo ? cdiv(n * nkv * parts, kWaves) : n * nkv * parts, 8) * blocks;
  }
};

Plan make_plan(const syn_hip_kv_pages &pg, const syn_hip_paged_attention_params &p) {
  Plan w{};
  const int hd = (int)pg.head_dim, nkv = (int)pg.n_kv_heads;
  const size_t rep = p.n_heads / nkv, rows = p.max_new * rep;
  w.nc = hd <= 64 ? 2 : (hd <= 128 ? 4 : 8);
  const bool small = w.nc * (pg.dtype == SYN_HIP_KV_F32 ? 2 : 1) <= 4;  // (a ring of four tiles)
  w.rw = rows <= 16 ? 1 : (rows <= 32 ? (small ? 2 : 1) : 4);
  w.blocks = (int)cdiv(rows, 16 * w.rw);
  // the positions of a workgroup's rows
  const size_t tokens = std::min<size_t>(p.max_new, 16 * w.rw / rep + 2);
  const size_t span = p.window ? std::min<size_t>(p.max_len, (size_t)p.window + tokens + kTile) : p.max_len;
  const size_t tiles = cdiv(span, kTile), units = (size_t)p.n_seqs * nkv;
  // workgroups that the chip holds at once (with 16 rows each one a CU fewer where
  // heads do not fill their tiles, f32 or f16, and of 64 dims in bf16)
  const bool f32 = pg.dtype == SYN_HIP_KV_F32;
  const size_t want = w.nc == 8 ? 256 : (w.nc == 2 && !f32 ? 1024 : (w.rw == 4 && !f32 ? 768 : 512));
  const size_t whole = pg.dtype == SYN_HIP_KV_F32 ? 2 : (units <= 512 ? 8 : 4);
  constexpr size_t kFix = 6;
  auto alone = [&](size_t units, size_t tiles) {
    return w.rw == 1 && cdiv(cdiv(units, kWaves) * w.blocks, want) * (kFix + tiles) <
                            cdiv(units * w.blocks, want) * (kFix + cdiv(tiles, kWaves));
  };
  w.parts = 1;
  w.chunk = (int)(tiles * kTile);
  auto cut = [&](size_t parts) {
    const size_t grain = w.rw == 1 ? kWaves : 2, per = round_up(cdiv(tiles, parts), grain);
    w.chunk = (int)(per * kTile);
    w.parts = (int)cdiv(tiles, per);
  };
  const size_t all = units * w.blocks;
  if (tiles > whole * kWaves && w.rw == 1 && all < want) {
    // few rows are bound by their bytes: as many workgroups as the chip holds
    cut(cdiv(want, all));
  } else if (tiles > whole * kWaves && w.rw > 1) {
    // Many rows are bound by their steps of a tile: of the ways to cut a run, the
    // one with the fewest, counted in rounds of workgroups (half a round of them,
    // one a CU, takes 0.8 of one), a fixed time each, and the join, which reads and
    // writes every part (4.5 TB/s; a step takes 0.9 us, of an f32 pool 3.5).  One
    // chunk of 1536 tokens at 12001, 24 heads of 128, f16: whole 526 us, in four parts
    // 449; two such sequences 844, in two 790; 200 tokens at 20000, 32 heads, 564, 222
    // in three, 151 as chosen; 512 tokens at 8000, f32, 602, in five 435; 16 tokens of
    // four sequences at 8200, bf16, 176, in five 51, 40 as chosen.
    const double step = pg.dtype == SYN_HIP_KV_F32 ? 3.5e-6 : 0.9e-6;
    double least = 0;
    size_t best = 1;
    for (size_t parts = 1; parts <= 8 || parts * all <= 4 * want; parts += 1 + parts / 16) {
      cut(parts);
      const size_t wgs = all * w.parts, rest = wgs % want;
      const double rounds = (double)(wgs / want) + (rest == 0 ? 0.0 : (rest <= want / 2 ? 0.8 : 1.0));
      const double join = (double)p.n_tokens * p.n_heads * w.parts * 8 * (hd + 2) / 4.5e12 / step + 5;
      const double steps = rounds * (kFix + w.chunk / kTile) + (w.parts > 1 ? join : 0.0);
      const bool fits = (double)p.n_tokens * p.n_heads * w.parts * 4 * (hd + 2) <= kMostSpace;
      if (parts == 1 || (fits && steps < least)) least = steps, best = parts;
    }
    cut(best);
  }
  w.solo = alone(units * w.parts, w.chunk / kTile);
  // Most calls are one launch.  Every sequence counts as max_new tokens here, so a
  // batch with few tokens may need more workgroups, or more rows joined, than a
  // launch takes: then some sequences at a time.
  w.seqs = kMostWgs / w.blocks / 8 * 8 * (w.solo ? kWaves : 1) / ((size_t)nkv * w.parts);
  if (w.parts > 1) w.seqs = std::min(w.seqs, kMostWgs / ((size_t)p.max_new * p.n_heads));
  w.seqs = std::min<size_t>(w.seqs, p.n_seqs);
  if (w.parts > 1) {
    const size_t n = (size_t)p.n_tokens * p.n_heads * w.parts;
    w.po_bytes = round_up(n * hd * 4, 16);
    w.pml_bytes = round_up(n * 8, 16);
  }
  return w;
}

syn_status_t check(const syn_hip_kv_pages *pages, const syn_hip_paged_attention_params *p) {
  if (!p) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_pages(pages, "paged_attention"));
  const size_t hd = pages->head_dim;
  if (p->layer >= pages->n_layers || !p->n_heads || p->n_heads % pages->n_kv_heads || p->n_heads > 65535u) {
    set_error("paged_attention: layer outside the pool, or n_heads no multiple of n_kv_heads");
    return SYN_ERR_INVALID_ARG;
  }
  // (kernels look two rounds of tiles past a length, and count rows, in 32 bits)
  if (p->n_seqs > 65535u || p->max_len > 0x7fff0000u || p->n_tokens > 0x7fffffffu ||
      (p->n_tokens && p->max_new > p->n_tokens) || (uint64_t)p->max_new * p->n_heads > 0x3fffffffu) {
    set_error("paged_attention: more than 65535 sequences, 2^31 - 2^16 positions or 2^30 - 1 query rows of "
              "a sequence, or max_new above n_tokens");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->ldq < p->n_heads * hd || p->ldo < p->n_heads * hd || p->ld_table < cdiv(p->max_len, pages->page_size)) {
    set_error("paged_attention: rows or page tables shorter than the heads or the lengths");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  if (!p->n_seqs || !p->max_new || !p->n_tokens) return SYN_OK;
  if (!make_plan(*pages, *p).seqs) {
    set_error("paged_attention: a sequence of more rows than a launch takes");
    return SYN_ERR_INVALID_ARG;
  }
  return SYN_OK;
}

template <class T, int NC, int RW>
void launch_rows(size_t wgs, const PagedArgs &a, const KvPool<T> &pool, hipStream_t s) {
  const dim3 grid((unsigned)wgs), block(64 * kWaves);
  if (pool.hd == 32 * NC)
    hipLaunchKernelGGL((k_attend_new<T, NC, true, RW>), grid, block, 0, s, a, pool);
  else
    hipLaunchKernelGGL((k_attend_new<T, NC, false, RW>), grid, block, 0, s, a, pool);
}
template <class T, int NC>
syn_status_t launch(const Plan &w, const PagedArgs &a, const KvPool<T> &pool, hipStream_t s) {
  const size_t wgs = w.wgs(a.n_seqs, pool.nkv);
  if (w.rw == 1)
    launch_rows<T, NC, 1>(wgs, a, pool, s);
  else if (w.rw == 4)
    launch_rows<T, NC, 4>(wgs, a, pool, s);
  else if constexpr (Rows<T, NC, true, true>::kRing == 4)
    launch_rows<T, NC, 2>(wgs, a, pool, s);
  SYN_LAUNCH_CHECK();
  if (w.parts == 1) return SYN_OK;
  const size_t rows = (size_t)a.n_seqs * a.max_new * a.nh;
  if (w.parts <= kFewParts)
    hipLaunchKernelGGL((k_join_few<8 * NC>), dim3((unsigned)cdiv(rows, 256 / (8 * NC))), dim3(256), 0, s, a,
                       pool.hd, (uint32_t)rows);
  else
    hipLaunchKernelGGL((k_join_new<8 * NC>), dim3((unsigned)rows), dim3(256), 0, s, a, pool.hd);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

// sequences first .. first + n - 1 of a call
PagedArgs some_of(const PagedArgs &a, int hd, size_t first, size_t n) {
  PagedArgs b = a;
  b.n_seqs = (int)n;
  b.len += first;
  if (b.table) b.table += first * a.ld_table;
  if (b.start) {
    b.start += first;
  } else {
    const size_t rows = first * a.max_new, parts = rows * a.nh * a.parts;
    b.q += rows * a.ldq;
    b.out += rows * a.ldo;
    if (a.parts > 1) b.po += parts * hd, b.pml += parts * 2;
  }
  return b;
}

}  // namespace

}  // namespace syn

using namespace syn;

extern "C" syn_status_t syn_hip_paged_attention_workspace(const syn_hip_kv_pages *pages,
                                                          const syn_hip_paged_attention_params *p,
                                                          size_t *bytes) {
  if (!bytes) return SYN_ERR_NULL_PTR;
  SYN_TRY(check(pages, p));
  *bytes = 0;
  if (!p->n_seqs || !p->max_new || !p->n_tokens) return SYN_OK;
  const Plan w = make_plan(*pages, *p);
  *bytes = w.po_bytes + w.pml_bytes;
  return SYN_OK;
}

extern "C" syn_status_t syn_hip_paged_attention(const syn_hip_kv_pages *pages,
                                                const syn_hip_paged_attention_params *p, const float *d_q,
                                                const int32_t *d_start, const int32_t *d_len,
                                                const int32_t *d_table, float *d_out, void *d_workspace,
                                                size_t workspace_bytes, void *stream) {
  SYN_TRY(check(pages, p));
  if (!d_start && (uint64_t)p->n_seqs * p->max_new != p->n_tokens) {
    set_error("paged_attention: without d_start every sequence has max_new tokens");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  if (!p->n_seqs || !p->max_new || !p->n_tokens) return SYN_OK;
  if (!d_q || !d_out || !d_len || (p->max_len && !d_table)) return SYN_ERR_NULL_PTR;
  const Plan w = make_plan(*pages, *p);
  const size_t need = w.po_bytes + w.pml_bytes;
  if (need && !d_workspace) return SYN_ERR_NULL_PTR;
  if (need && (!aligned16(d_workspace) || workspace_bytes < need)) {
    set_error("paged_attention: workspace unaligned or too small");
    return SYN_ERR_INVALID_ARG;
  }
  SYN_TRY(ensure_init());
  PagedArgs a{};
  a.q = d_q;
  a.out = d_out;
  a.ldq = p->ldq;
  a.ldo = p->ldo;
  a.nh = (int)p->n_heads;
  a.rep = (int)(p->n_heads / pages->n_kv_heads);
  a.scale = (p->scale != 0.0f ? p->scale : 1.0f / sqrtf((float)pages->head_dim)) * kLog2e;
  a.parts = w.parts;
  a.po = static_cast<float *>(d_workspace);
  a.pml = reinterpret_cast<float *>(static_cast<uint8_t *>(d_workspace) + w.po_bytes);
  a.q16 = aligned16(d_q) && p->ldq % 4 == 0;
  a.start = d_start;
  a.len = d_len;
  a.table = d_table;
  a.ld_table = p->ld_table;
  a.n_seqs = (int)p->n_seqs;
  a.n_tokens = (int)p->n_tokens;
  a.max_new = (int)p->max_new;
  a.max_len = (int)p->max_len;
  a.window = p->window < p->max_len ? (int)p->window : 0;
  a.chunk = w.chunk;
  a.blocks = w.blocks;
  a.solo = w.solo;
  hipStream_t s = pick_stream(stream);
  return kv_dispatch(pages->dtype, [&](auto t) -> syn_status_t {
    using T = decltype(t);
    const KvPool<T> pool = kv_pool<T>(*pages, p->layer);
    for (size_t i = 0; i < p->n_seqs; i += w.seqs) {
      const PagedArgs b = some_of(a, pool.hd, i, std::min<size_t>(w.seqs, p->n_seqs - i));
      SYN_TRY(w.nc == 2 ? (launch<T, 2>(w, b, pool, s))
                        : (w.nc == 4 ? (launch<T, 4>(w, b, pool, s)) : (launch<T, 8>(w, b, pool, s))));
    }
    return SYN_OK;
  });
}
