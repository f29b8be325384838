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
// accumulators; an f32 pool takes the f32 matrix instructions.  f16 has 40
// binary orders where f32 has 277, so weights far below a row's maximum, which
// are all that counts where its value is zero, are lifted into f16's range by
// powers of two and summed apart.
//
// What bounds it (a large copy reaches 4.8 TB/s here, a stream of reads alone
// more, large products 1115 TFLOP/s in f16 and 152 in f32): up to 16 rows of a
// kv head, bytes: 64 sequences of 4000 positions, 8 kv heads of 128, f16, 191
// us, 5.5 TB/s; a shared prefix of 4 * 32768 under 4 to 16 rows 99 to 101 us,
// 5.4 to 5.3 TB/s.  32 rows 5.0, 64 rows 4.6 TB/s and 290 TFLOP/s of the
// formula, 580 in matrix instructions with the operands' second parts; 128 rows
// 380 and 760.  f32, 64 rows: 3.0 TB/s, 97 TFLOP/s, the matrix instructions.
// Short calls are latency: 4 sequences of 113 positions 7.5 us.
#include <algorithm>
#include <cmath>

#include "attend_rows.hpp"

namespace syn {

namespace {

struct AttnArgs : RowArgs {
  const int32_t *ptable, *plen, *table, *slen;
  size_t ld_ptable, ld_table;
  int group_size, n_seqs, max_prefix, max_suffix;
  // the split: positions of a part (a multiple of kTile), parts of
  // the longest prefix and suffix
  int pchunk, schunk, npp, nsp, prefix_wgs;
  int prw, srw;  // tiles of 16 rows of a prefix and of a suffix workgroup: 1, 2 or 4
  bool joined, solo;  // solo: a wave for a sequence's rows
};

// Joined: a workgroup has both runs of a sequence's rows whole.  Else the
// first workgroups have the parts of the prefixes, the others those of the
// suffixes.  Solo: a wave has what else a sequence's workgroup has.
template <class T, int NC, bool FULL>
__global__ void __launch_bounds__(64 * kWaves, (kResident<T, NC, FULL>)) k_attend(AttnArgs a, KvPool<T> pool) {
  using W = Rows<T, NC, FULL>;
  __shared__ __align__(16) uint8_t lds[W::kLdsBytes];
  __shared__ float ml[kWaves * 16 * 2];
  const bool prefix = (int)blockIdx.x < a.prefix_wgs;
  const int i = prefix ? blockIdx.x : blockIdx.x - a.prefix_wgs;
  const int members = prefix ? a.group_size : 1;  // sequences whose rows go together
  const int RW = prefix ? a.prw : a.srw;
  const int all = members * a.rep, blocks = (all + RW * 16 - 1) / (RW * 16);
  const int parts = a.joined ? 1 : (prefix ? a.npp : a.nsp);
  // workgroup i runs on XCD i % 8: the blocks of rows that read the same
  // positions come 8 apart and share that XCD's L2
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool solo = !prefix && a.solo;  // nothing below waits for the other waves then
  const int j = i >> 3, block = j % blocks;
  int unit = (j / blocks) * 8 + (i & 7);
  if (solo) unit = unit * kWaves + wave;
  const int head = unit % pool.nkv, u = unit / pool.nkv;
  const int part = u % parts, owner = u / parts;  // group or sequence
  if (owner * members >= a.n_seqs) return;
  const int seq0 = owner * members, row0 = block * RW * 16, rows = min(RW * 16, all - row0);
  const int group = prefix ? owner : owner / a.group_size;
  const int plen = prefix || a.joined ? clamped(a.plen, group, a.max_prefix) : 0;
  const int slen = prefix ? 0 : clamped(a.slen, seq0, a.max_suffix);
  Run r{prefix ? a.ptable + (size_t)group * a.ld_ptable : a.table + (size_t)seq0 * a.ld_table, 0, slen, 0};
  int at = -1;
  if (!a.joined) {
    const int len = prefix ? plen : slen, chunk = prefix ? a.pchunk : a.schunk;
    r.from = part * chunk;
    r.to = r.from + min(chunk, len - r.from);  // (the sum of the two may pass 2^31)
    at = prefix ? part : a.npp + part;
    if (r.from >= len) {  // nothing here: no rows to write, a sum of 0
      for (int k = solo ? (int)threadIdx.x & 63 : (int)threadIdx.x; k < rows; k += 64 * kWaves) {
        const int row = row0 + k, member = row / a.rep;
        const size_t p = ((size_t)(seq0 + member) * a.nh + (size_t)head * a.rep + (row - member * a.rep)) *
                             a.parts + at;
        a.pml[p * 2] = kNegInf;
        a.pml[p * 2 + 1] = 0.0f;
      }
      return;
    }
  }
  const size_t head_bytes = (size_t)pool.hd * pool.ps * sizeof(T);
  const HeadBase hb{reinterpret_cast<const uint8_t *>(pool.k) + head * head_bytes,
                    reinterpret_cast<const uint8_t *>(pool.v) + head * head_bytes,
                    (uint32_t)(pool.nkv * head_bytes)};
  const bool wide = pool.ps >= kTile;
  uint32_t ok = 0;
  if (RW == 4)
    ok = wide ? W::template start_shared<true, 1>(pool, hb, r, lds)
              : W::template start_shared<false, 1>(pool, hb, r, lds);
  if constexpr (W::kRing == 4)
    if (RW == 2)
      ok = wide ? W::template start_shared<true, 2>(pool, hb, r, lds)
                : W::template start_shared<false, 2>(pool, hb, r, lds);
  W w;
  const int tile = wave & (RW - 1);
  w.load_queries(a, pool.hd, seq0, head, row0 + tile * 16, row0 + rows - 1);
  if (RW == 1) {
    // joined: the prefix first, its next tile's wave begins the suffix
    for (int k = a.joined ? 0 : 1; k < 2; k++) {
      Run x = r;
      if (k == 0) x = Run{a.ptable + (size_t)group * a.ld_ptable, 0, plen, 0};
      if (k == 1 && a.joined) x.first = (plen + kTile - 1) / kTile;
      if (wide)
        w.template run_alone<true>(pool, hb, x, solo ? 1 : kWaves);
      else
        w.template run_alone<false>(pool, hb, x, solo ? 1 : kWaves);
    }
    if (solo) {
      w.finish_alone(a, pool.hd, seq0, head, row0, rows, at);
      return;
    }
  } else if (RW == 4) {
    if (wide)
      w.template run_shared<true, 1>(pool, hb, r, lds, ok);
    else
      w.template run_shared<false, 1>(pool, hb, r, lds, ok);
  } else if constexpr (W::kRing == 4) {
    if (wide)
      w.template run_shared<true, 2>(pool, hb, r, lds, ok);
    else
      w.template run_shared<false, 2>(pool, hb, r, lds, ok);
  }
  w.finish(a, pool.hd, seq0, head, row0, rows, RW, at, reinterpret_cast<float *>(lds), ml);
}

template <int LANES> __global__ void __launch_bounds__(256) k_join_parts(RowArgs a, int hd) {
  join_parts<LANES>(a, hd, blockIdx.x);
}

// ---------------------------------------------------------------- host
struct Plan {
  bool joined, solo;
  int nc, prw, srw;
  int pchunk, schunk, npp, nsp;
  size_t prefix_wgs, wgs, rows, po_bytes, pml_bytes;
};

Plan make_plan(const syn_hip_kv_pages &pg, const syn_hip_prefix_attention_params &p) {
  Plan w{};
  const int hd = (int)pg.head_dim, nkv = (int)pg.n_kv_heads, rep = (int)p.n_heads / nkv;
  w.nc = hd <= 64 ? 2 : (hd <= 128 ? 4 : 8);
  w.rows = (size_t)p.n_groups * p.group_size * p.n_heads;
  // Two tiles of rows need a ring of four tiles of positions; where it holds
  // two, their blocks read K and V once each, the second time from L2.
  const bool small = w.nc * (pg.dtype == SYN_HIP_KV_F32 ? 2 : 1) <= 4;
  auto tiles = [&](size_t rows) { return rows <= 16 ? 1 : (rows <= 32 ? (small ? 2 : 1) : 4); };
  const size_t seqs = (size_t)p.n_groups * p.group_size;
  // One launch, each sequence's rows whole, where a second launch would cost
  // more than the prefix read again for every sequence (from L2): 24 heads of
  // 128, 8 sequences, f16: 200 positions 7.2 us against 10.5 in parts, 600 9.0
  // against 10.6, 900 10.9 against 10.7, 1600 14.0 against 11.2; 128 sequences of
  // 200 15.0 against 18.4, of 400 20.4 against 18.8.  An f32 tile has twice the
  // bytes and four times the matrix instructions' time: 200 positions 10.4 us
  // against 11.6, 500 17.8 against 11.7.
  const size_t whole = pg.dtype == SYN_HIP_KV_F32 ? 2 : (seqs * nkv <= 512 ? 8 : 4);
  w.joined = (size_t)p.max_prefix + p.max_suffix <= whole * kTile * kWaves;
  w.prw = tiles((size_t)p.group_size * rep);
  w.srw = w.joined ? 1 : tiles(rep);
  const size_t sblocks = cdiv(rep, 16 * w.srw), sunits = seqs * nkv;
  // Parts of about equal work for as many workgroups as the chip holds at
  // once, four a CU, two, or one.  (512 workgroups of 64 dims in 16 bits,
  // 48 sequences of 1500 positions over a shared 8200: 45 us, 1024: 38.7 in bf16,
  // 37.8 in f16; of 128 dims, 64 sequences over four prefixes of 32768: 111 and
  // 119.)
  const size_t want = w.nc == 8 ? 256 : (w.nc == 4 || pg.dtype == SYN_HIP_KV_F32 ? 512 : 1024);
  const size_t ptiles = cdiv(p.max_prefix, kTile), stiles = cdiv(p.max_suffix, kTile);
  // Many short runs of a sequence's own: a wave for each, where the rounds of
  // workgroups with their latency (of about kFix tiles) come to less so (246
  // sequences of 20 positions, 8 kv heads of 128, f32: 19 us against 36 with
  // four waves; 100 over shared prefixes of 559: 32 and 48).
  constexpr size_t kFix = 6;
  auto alone = [&](size_t units, size_t tiles) {
    return w.srw == 1 && cdiv(cdiv(units, kWaves) * sblocks, want) * (kFix + tiles) <
                             cdiv(units * sblocks, want) * (kFix + cdiv(tiles, kWaves));
  };
  auto groups_of = [&](size_t units) { return round_up(w.solo ? cdiv(units, kWaves) : units, 8) * sblocks; };
  if (w.joined) {
    w.solo = alone(sunits, ptiles + stiles);
    w.wgs = groups_of(sunits);
    return w;
  }
  const size_t pblocks = cdiv((size_t)p.group_size * rep, 16 * w.prw), punits = (size_t)p.n_groups * nkv;
  const size_t total = punits * pblocks * ptiles + sunits * sblocks * stiles;
  auto cut = [&](size_t tiles, size_t each, size_t grain, int *chunk, int *n) {
    const size_t k = cdiv(tiles, round_up(each, grain));  // as many parts, of equal length
    each = k ? round_up(cdiv(tiles, k), grain) : 0;
    *chunk = (int)(each * kTile);
    *n = each ? (int)cdiv(tiles, each) : 0;
  };
  // Waves that share tiles take them all, so a part may be short: two tiles (160
  // rows of f16 over 4001 positions 25.6 us, 26.8 with four, 24.7 with one; up to
  // 64 rows over 300 to 4001 the three are alike).
  constexpr size_t kGrain = 2;
  for (size_t per = std::max<size_t>(1, cdiv(total, want));; per += kGrain + per / 16) {
    cut(ptiles, per, w.prw == 1 ? kWaves : kGrain, &w.pchunk, &w.npp);
    cut(stiles, per, kWaves, &w.schunk, &w.nsp);
    w.solo = alone(sunits * w.nsp, std::min<size_t>(stiles, w.schunk / kTile));
    w.prefix_wgs = round_up(punits * w.npp, 8) * pblocks;
    const size_t suffix_wgs = groups_of(sunits * w.nsp);
    w.wgs = w.prefix_wgs + suffix_wgs;
    // A second round for an eighth or more of them costs more than longer parts
    // (24 sequences of 16 heads of 64 over eight prefixes of 3876: 18.0 us, 15.5
    // so), and so do 1.5 of them a CU (52 of 16 heads of 128, f32, over four of
    // 6918: 384 workgroups 82 us, 256 64); suffixes count by their length.
    // Where they alone make rounds, the order hides it.
    constexpr size_t kCus = 256;
    const bool uneven = w.prefix_wgs > kCus && 4 * round_up(w.prefix_wgs, kCus) > 5 * w.prefix_wgs;
    auto waves_take = [&](int chunk, int rw) { return kFix + cdiv((size_t)chunk / kTile * rw, kWaves); };
    const size_t stiles_part = std::min<size_t>(stiles, w.schunk / kTile);
    const size_t suffix = suffix_wgs * (w.solo ? kFix + stiles_part : waves_take(w.schunk, w.srw)) /
                          waves_take(w.pchunk, w.prw);
    if (w.npp <= 1 || (w.prefix_wgs + suffix <= want + want / 8 && !uneven) || 2 * suffix > want) break;
  }
  const size_t n = w.rows * (size_t)(w.npp + w.nsp);
  w.po_bytes = round_up(n * hd * 4, 16);
  w.pml_bytes = round_up(n * 8, 16);
  return w;
}

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
  // (kernels look two rounds of tiles past a length, in 32 bits)
  constexpr uint32_t kMaxLength = 0x7fff0000u;
  if (rows > 65535u || p->max_prefix > kMaxLength || p->max_suffix > kMaxLength) {
    set_error("prefix_attention: more than 65535 sequences or 2^31 - 2^16 positions");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->ldq < p->n_heads * hd || p->ldo < p->n_heads * hd ||
      p->ld_prefix_table < cdiv(p->max_prefix, pages->page_size) ||
      p->ld_table < cdiv(p->max_suffix, pages->page_size)) {
    set_error("prefix_attention: rows or page tables shorter than the heads or the lengths");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  const Plan w = make_plan(*pages, *p);
  if (w.wgs > kMaxThreads / (64 * kWaves) || w.rows > kMaxThreads / 256) {
    set_error("prefix_attention: more workgroups than a launch takes");
    return SYN_ERR_INVALID_ARG;
  }
  return SYN_OK;
}

template <class T, int NC>
syn_status_t launch(const Plan &w, const AttnArgs &a, const KvPool<T> &pool, hipStream_t s) {
  const dim3 grid((unsigned)w.wgs), block(64 * kWaves);
  if (pool.hd == 32 * NC)
    hipLaunchKernelGGL((k_attend<T, NC, true>), grid, block, 0, s, a, pool);
  else
    hipLaunchKernelGGL((k_attend<T, NC, false>), grid, block, 0, s, a, pool);
  SYN_LAUNCH_CHECK();
  if (w.joined) return SYN_OK;
  const dim3 rows((unsigned)w.rows);
  if (NC == 2)
    hipLaunchKernelGGL(k_join_parts<16>, rows, dim3(256), 0, s, a, pool.hd);
  else if (NC == 4)
    hipLaunchKernelGGL(k_join_parts<32>, rows, dim3(256), 0, s, a, pool.hd);
  else
    hipLaunchKernelGGL(k_join_parts<64>, rows, dim3(256), 0, s, a, pool.hd);
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
  a.parts = w.npp + w.nsp;
  a.nsp = w.nsp;
  a.prefix_wgs = (int)w.prefix_wgs;
  a.prw = w.prw;
  a.srw = w.srw;
  a.joined = w.joined;
  a.solo = w.solo;
  a.q16 = aligned16(d_q) && p->ldq % 4 == 0;
  a.po = static_cast<float *>(d_workspace);
  a.pml = reinterpret_cast<float *>(static_cast<uint8_t *>(d_workspace) + w.po_bytes);
  hipStream_t s = pick_stream(stream);
  return kv_dispatch(pages->dtype, [&](auto t) -> syn_status_t {
    using T = decltype(t);
    const KvPool<T> pool = kv_pool<T>(*pages, p->layer);
    if (w.nc == 2) return launch<T, 2>(w, a, pool, s);
    if (w.nc == 4) return launch<T, 4>(w, a, pool, s);
    return launch<T, 8>(w, a, pool, s);
  });
}
