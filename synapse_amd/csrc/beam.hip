// Beam search's choice over beams and vocabulary, and the states that follow
// it.
#include "kv_pages.hpp"

namespace syn {

namespace {

// ---------------------------------------------------------------- choice
// The order of continuations: larger value first, then the lower index.
struct Cand {
  float v;
  int i;
};
__device__ __forceinline__ bool before(float av, int ai, float bv, int bi) {
  return av > bv || (av == bv && ai < bi);
}

// what the first kernel leaves of a row: its n_select best logits, largest
// logit and log of the sum of exp(logit - largest)
struct RowStat {
  double logsum;
  float top;
  int pad;
};

struct SelectArgs {
  const float *logits, *scores;
  const int32_t *finished;
  int32_t *parent, *finished_out;
  uint32_t *token;
  float *score;
  Cand *cand;     // [rows][n_select]
  RowStat *stat;  // [rows]
  size_t ld;
  int vocab, n_beams, n_select, eos, pad;
};

__device__ __forceinline__ float masked(float x) {
  return x != x ? -__builtin_inff() : x;
}

constexpr int kRowNT = 1024;
__global__ void __launch_bounds__(kRowNT) k_beam_rows(SelectArgs a) {
  __shared__ float rv[16];
  __shared__ int ri[16];
  __shared__ double rs[16];
  const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab;
  Cand *out = a.cand + (size_t)row * a.n_select;
  if (!isfinite(a.scores[row])) {  // no continuation: every one -inf
    for (int i = tid; i < a.n_select; i += kRowNT)
      out[i] = Cand{-__builtin_inff(), i < V ? i : -1};
    if (tid == 0) a.stat[row] = RowStat{0.0, 0.0f, 0};
    return;
  }
  if (a.finished && a.finished[row]) {
    for (int i = tid; i < a.n_select; i += kRowNT) {
      const int t = i == 0 ? a.pad : (i - 1 < a.pad ? i - 1 : i);
      out[i] = Cand{i == 0 ? 0.0f : -__builtin_inff(), t < V ? t : -1};
    }
    if (tid == 0) a.stat[row] = RowStat{0.0, 0.0f, 0};
    return;
  }
  const float *x = a.logits + (size_t)row * a.ld;
  float pv = __builtin_inff();
  int pi = -1;
  float top = 0.0f;
  for (int r = 0; r < a.n_select; r++) {
    float bv = -__builtin_inff();
    int bi = 0x7fffffff;
    for (int i = tid; i < V; i += kRowNT) {
      const float v = masked(x[i]);
      if (before(pv, pi, v, i) && before(v, i, bv, bi)) bv = v, bi = i;
    }
    for (int o = 32; o > 0; o >>= 1) {
      const float v = __shfl_xor(bv, o);
      const int i = __shfl_xor(bi, o);
      if (before(v, i, bv, bi)) bv = v, bi = i;
    }
    if ((tid & 63) == 0) rv[tid >> 6] = bv, ri[tid >> 6] = bi;
    __syncthreads();
    bv = rv[0], bi = ri[0];
    for (int w = 1; w < 16; w++)
      if (before(rv[w], ri[w], bv, bi)) bv = rv[w], bi = ri[w];
    __syncthreads();
    if (r == 0) top = bv;
    if (tid == 0) out[r] = Cand{bv, bi == 0x7fffffff ? -1 : bi};
    pv = bv;
    pi = bi;
  }
  double s = 0.0;
  for (int i = tid; i < V; i += kRowNT) {
    const float v = masked(x[i]);
    s += v == top ? 1.0 : (double)expf(v - top);
  }
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((tid & 63) == 0) rs[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.0;
    for (int w = 0; w < 16; w++) s += rs[w];
    a.stat[row] = RowStat{log(s), top, 0};
  }
}

// one workgroup a group: the n_select best of the rows' candidates
__global__ void __launch_bounds__(256) k_beam_merge(SelectArgs a) {
  __shared__ double val[kMaxBeams * kMaxSelect];
  __shared__ double rv[4];
  __shared__ int ri[4];
  const int g = blockIdx.x, tid = threadIdx.x, W = a.n_beams, n = a.n_select;
  const size_t row0 = (size_t)g * W;
  const Cand *c = a.cand + row0 * n;
  for (int j = tid; j < W * n; j += 256) {
    const int b = j / n;
    const RowStat st = a.stat[row0 + b];
    const float sc = a.scores[row0 + b], x = c[j].v;
    const double d = x == st.top ? 0.0 : (double)x - (double)st.top;
    double v = (double)sc + (d - st.logsum);
    if (x == -__builtin_inff()) v = -__builtin_inf();
    if (c[j].i < 0) v = __builtin_nan("");
    val[j] = v;
  }
  __shared__ int done[kMaxBeams];
  for (int b = tid; b < W; b += 256) done[b] = a.finished ? a.finished[row0 + b] != 0 : 0;
  __syncthreads();
  // candidates of a row are in order already, so among equal values the lower
  // j is the lower (beam, token)
  double pv = __builtin_inf();
  int pj = -1;
  for (int r = 0; r < n; r++) {
    double bv = -__builtin_inf();
    int bj = 0x7fffffff;
    for (int j = tid; j < W * n; j += 256) {
      const double v = val[j];
      if ((v < pv || (v == pv && j > pj)) && (v > bv || (v == bv && j < bj))) bv = v, bj = j;
    }
    for (int o = 32; o > 0; o >>= 1) {
      const double v = __shfl_xor(bv, o);
      const int j = __shfl_xor(bj, o);
      if (v > bv || (v == bv && j < bj)) bv = v, bj = j;
    }
    if ((tid & 63) == 0) rv[tid >> 6] = bv, ri[tid >> 6] = bj;
    __syncthreads();
    bv = rv[0], bj = ri[0];
    for (int w = 1; w < 4; w++)
      if (rv[w] > bv || (rv[w] == bv && ri[w] < bj)) bv = rv[w], bj = ri[w];
    __syncthreads();
    if (tid == 0) {
      const int b = bj / n;
      const size_t o = (size_t)g * n + r;
      a.parent[o] = b;
      a.token[o] = (uint32_t)c[bj].i;
      a.score[o] = (float)bv;
      if (a.finished_out) a.finished_out[o] = done[b] || c[bj].i == a.eos;
    }
    pv = bv;
    pj = bj;
  }
}

syn_status_t check_select(const syn_hip_beam_select_params *p) {
  if (!p) return SYN_ERR_NULL_PTR;
  if (!p->n_beams || p->n_beams > kMaxBeams || !p->n_select || p->n_select > kMaxSelect) {
    set_error("beam_select: 1 to 64 beams and 1 to 128 continuations");
    return SYN_ERR_INVALID_ARG;
  }
  if (!p->vocab || p->vocab > 0x7fffff00u || (uint64_t)p->n_select > p->n_beams * (uint64_t)p->vocab ||
      (uint64_t)p->n_groups * p->n_beams > 0x7fffffffu) {
    set_error("beam_select: fewer continuations than n_select, or too many rows");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->ld_logits < p->vocab) {
    set_error("beam_select: rows of logits shorter than the vocabulary");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  return SYN_OK;
}

struct SelectSpace {
  size_t stat, cand, total;
};
SelectSpace select_space(const syn_hip_beam_select_params &p) {
  const size_t rows = (size_t)p.n_groups * p.n_beams;
  SelectSpace s;
  s.stat = 0;
  s.cand = round_up(rows * sizeof(RowStat), 16);
  s.total = s.cand + round_up(rows * p.n_select * sizeof(Cand), 16);
  return s;
}

// ---------------------------------------------------------------- reordering
// One workgroup moves 64 units (of U bytes) of every row of a group: a unit's
// rows are all read before any is written, so the move is in place.
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

// grid (layer * kv head, row): the parent's part of a page into the spare page
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

// grid (columns / 64, group), after the copies
__global__ void __launch_bounds__(64) k_reorder_tables(PagesArgs a) {
  __shared__ int32_t stage[kMaxBeams][64];
  const int l = threadIdx.x, g = blockIdx.y, W = a.W;
  const size_t col = (size_t)blockIdx.x * 64 + l;
  size_t full;
  int rest;
  held(a, g, &full, &rest);
  if (col > full || col >= a.ld_table) return;
  const int32_t *par = a.parent + (size_t)g * W;
  int32_t *t = a.table + (size_t)g * W * a.ld_table + col;
  if (col < full) {
    for (int b = 0; b < W; b++) {
      const int p = par[b];
      stage[b][l] = t[((uint32_t)p < (uint32_t)W ? p : b) * a.ld_table];
    }
    for (int b = 0; b < W; b++) t[b * a.ld_table] = stage[b][l];
  } else if (rest) {
    for (int b = 0; b < W; b++) {
      const int p = par[b];
      if (p == b || (uint32_t)p >= (uint32_t)W) continue;
      const int32_t mine = t[b * a.ld_table];
      t[b * a.ld_table] = a.spare[(size_t)g * W + b];
      a.spare[(size_t)g * W + b] = mine;
    }
  }
}

syn_status_t check_beams(size_t n_groups, size_t n_beams, const char *who) {
  if (!n_beams || n_beams > kMaxBeams || n_groups > 65535u / n_beams) {
    set_error(std::string(who) + ": 1 to 64 beams, at most 65535 rows");
    return SYN_ERR_INVALID_ARG;
  }
  return SYN_OK;
}

}  // namespace

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
                     reinterpret_cast<Cand *>(ws + sp.cand),
                     reinterpret_cast<RowStat *>(ws + sp.stat), p->ld_logits, (int)p->vocab,
                     (int)p->n_beams, (int)p->n_select, p->eos, p->pad};
  hipStream_t s = pick_stream(stream);
  hipLaunchKernelGGL(k_beam_rows, dim3(p->n_groups * p->n_beams), dim3(kRowNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_beam_merge, dim3(p->n_groups), dim3(256), 0, s, a);
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
  if (n_buffers > 65535u || row_bytes > (size_t)1 << 36) {
    set_error("beam_reorder_rows: at most 65535 buffers of rows up to 64 GiB");
    return SYN_ERR_INVALID_ARG;
  }
  if (!n_groups || !row_bytes || !n_buffers) return SYN_OK;
  if (!d_parent || !d_rows) return SYN_ERR_NULL_PTR;
  SYN_TRY(ensure_init());
  const size_t all = reinterpret_cast<uintptr_t>(d_rows) | row_bytes | row_stride |
                     (n_buffers > 1 ? buffer_stride : 0);
  const size_t unit = all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1), units = row_bytes / unit;
  if (cdiv(units, 64) > 0x7fffffffu) {
    set_error("beam_reorder_rows: rows too long for their alignment");
    return SYN_ERR_INVALID_ARG;
  }
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
  if ((uint64_t)pages->n_layers * pages->n_kv_heads > 0x7fffffffu || ld_table > 0x7fffffffu) {
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
                     dim3(64), 0, s, a);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // extern "C"
