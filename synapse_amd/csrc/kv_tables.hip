// Page tables of a paged cache: pages taken and given back, sequences that
// continue another one's pages, live pages moved to another pool.
//
// A page's count is the number of table entries that name it, and a page of
// count 0 is free, so there is no list of free pages to keep in order: whoever
// needs pages gets the free ones of lowest number, the rows in order and the
// columns of a row in order, whatever order the workgroups run in.
#include <algorithm>

#include "kv_pages.hpp"
#include "wave_ops.hpp"

namespace syn {

namespace {

constexpr int kNT = 256;
constexpr int kPer = 16;              // pages of a thread
constexpr int kChunk = kNT * kPer;    // pages of a workgroup
constexpr uint32_t kMaxTablePages = 1u << 24;

struct TableArgs {
  int32_t *table, *held, *refs;
  const int32_t *len, *parent;
  size_t ld;
  uint32_t n_pages;
  int n_seqs, chunks, ps, ps_shift;
  int32_t *need;    // [n_seqs] pages that a row takes
  int32_t *before;  // [n_seqs + 1] those of the rows before it
  int32_t *count;   // [chunks] free (or live) pages of a chunk
  __device__ __forceinline__ bool has(int page) const { return (uint32_t)page < n_pages; }
  __device__ __forceinline__ int holds(int row) const {
    return (int)min((size_t)max(0, held[row]), ld);
  }
  __device__ __forceinline__ int pages_of(int n) const { return (n >> ps_shift) + ((n & (ps - 1)) != 0); }
};

// a page loses one of the entries that name it (a count that the caller has
// left at 0 stays there)
__device__ __forceinline__ void drop(const TableArgs &a, int page) {
  if (a.has(page) && atomicSub(a.refs + page, 1) <= 0) atomicAdd(a.refs + page, 1);
}

// A wave's row: what it gives back.  Lanes take the columns in turn.
__device__ __forceinline__ void give_back(const TableArgs &a, int row, int from, int to) {
  int32_t *t = a.table + (size_t)row * a.ld;
  for (int c = from + (int)(threadIdx.x & 63); c < to; c += 64) {
    drop(a, t[c]);
    t[c] = -1;
  }
}

__device__ __forceinline__ void resize_row(const TableArgs &a, int row) {
  const int len = a.len[row], held = a.holds(row);
  const int want = len < 0 ? held : (int)min((size_t)a.pages_of(len), a.ld);
  give_back(a, row, want, held);
  if ((threadIdx.x & 63) == 0) {
    if (len >= 0) a.held[row] = min(held, want);
    a.need[row] = max(0, want - held);
  }
}

// The parent of a row that continues another one, which must stay what it is;
// -1: the row stays.
__device__ __forceinline__ int parent_of(const TableArgs &a, int row) {
  const int p = a.parent[row];
  return p != row && (uint32_t)p < (uint32_t)a.n_seqs && a.parent[p] == p ? p : -1;
}
// the positions that it takes over
__device__ __forceinline__ long long taken_over(const TableArgs &a, int row, int parent) {
  return min((long long)max(0, a.len[row]), (long long)a.holds(parent) << a.ps_shift);
}

__device__ __forceinline__ void fork_row(const TableArgs &a, int row) {
  const int lane = threadIdx.x & 63, held = a.holds(row), p = parent_of(a, row);
  if (p < 0) {
    if (lane == 0) a.need[row] = 0;
    return;
  }
  give_back(a, row, 0, held);
  const long long n = taken_over(a, row, p);
  const int full = (int)(n >> a.ps_shift);
  int32_t *t = a.table + (size_t)row * a.ld;
  const int32_t *from = a.table + (size_t)p * a.ld;
  for (int c = lane; c < full; c += 64) {
    const int page = from[c];
    if (a.has(page)) atomicAdd(a.refs + page, 1);
    t[c] = page;
  }
  if (lane == 0) {
    a.held[row] = full;
    a.need[row] = (n & (a.ps - 1)) != 0;
  }
}

template <bool FORK> __global__ void __launch_bounds__(kNT) k_rows(TableArgs a) {
  const int row = blockIdx.x * (kNT / 64) + (threadIdx.x >> 6);
  if (row >= a.n_seqs) return;
  if (FORK)
    fork_row(a, row);
  else
    resize_row(a, row);
}

// sum over the workgroup's lower threads; all: the whole sum
template <int NT> __device__ __forceinline__ int sum_before(int x, int *all) {
  __shared__ int w[NT / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = wave_before(x);
  __syncthreads();
  if (lane == 63) w[wave] = s + x;
  __syncthreads();
  int t = 0;
  for (int i = 0; i < NT / 64; i++) {
    if (i < wave) s += w[i];
    t += w[i];
  }
  *all = t;
  return s;
}

// the wanted pages among a thread's: bit j for page first + j
template <bool LIVE> __device__ __forceinline__ uint32_t wanted(const TableArgs &a, uint32_t first) {
  uint32_t on = 0;
#pragma unroll
  for (int j = 0; j < kPer; j++)
    if (first + j < a.n_pages) {
      const int n = a.refs[first + j];
      on |= (LIVE ? n > 0 : n == 0) ? 1u << j : 0u;
    }
  return on;
}

// workgroup 0: the rows' needs added up; the others: a chunk's wanted pages
template <bool LIVE> __global__ void __launch_bounds__(kNT) k_count(TableArgs a) {
  const int tid = threadIdx.x;
  int all;
  if (blockIdx.x == 0) {
    if (LIVE) return;
    int base = 0;
    for (int r0 = 0; r0 < a.n_seqs; r0 += kNT) {
      const int r = r0 + tid, n = r < a.n_seqs ? a.need[r] : 0;
      const int s = sum_before<kNT>(n, &all);
      if (r < a.n_seqs) a.before[r] = base + s;
      base += all;
    }
    if (tid == 0) a.before[a.n_seqs] = base;
    return;
  }
  const uint32_t chunk = blockIdx.x - 1;
  (void)sum_before<kNT>(__popc(wanted<LIVE>(a, chunk * kChunk + tid * kPer)), &all);
  if (tid == 0) a.count[chunk] = all;
}

// wanted pages of the chunks before this one, and of all
__device__ __forceinline__ int chunks_before(const TableArgs &a, int chunk, int *all) {
  int below = 0, total = 0, sum;
  for (int c = threadIdx.x; c < a.chunks; c += kNT) {
    const int n = a.count[c];
    total += n;
    below += c < chunk ? n : 0;
  }
  (void)sum_before<kNT>(total, all);
  (void)sum_before<kNT>(below, &sum);
  return sum;
}

// The i-th free page goes to the i-th place that needs one.
__global__ void __launch_bounds__(kNT) k_take(TableArgs a) {
  const int chunk = blockIdx.x, tid = threadIdx.x;
  int free, in;
  const int base = chunks_before(a, chunk, &free);
  const int needed = a.before[a.n_seqs];
  if (chunk == 0)
    for (int r = tid; r < a.n_seqs; r += kNT)
      a.held[r] += max(0, min(a.need[r], free - a.before[r]));
  if (base >= needed) return;
  const uint32_t first = chunk * (uint32_t)kChunk + tid * kPer;
  uint32_t on = wanted<false>(a, first);
  int rank = base + sum_before<kNT>(__popc(on), &in);
  for (; on && rank < needed; on &= on - 1, rank++) {
    const int page = (int)first + __ffs(on) - 1;
    int lo = 0, hi = a.n_seqs;  // the last row with before[row] <= rank
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.before[mid] <= rank)
        lo = mid;
      else
        hi = mid;
    }
    // (rows that need none have the same sum as the row after them)
    const int len = a.len[lo], i = rank - a.before[lo];
    const int end = a.parent ? (int)(taken_over(a, lo, parent_of(a, lo)) >> a.ps_shift) + 1
                             : (int)min((size_t)a.pages_of(len), a.ld);
    a.table[(size_t)lo * a.ld + (end - a.need[lo] + i)] = page;
    a.refs[page] = 1;
  }
}

// ---------------------------------------------------------------- copies
struct CopyArgs {
  const uint8_t *k, *v;
  uint8_t *to_k, *to_v;
  uint32_t n_pages, to_pages;
  int n_layers, nkv, hd, ps, esz;
};

// grid (layer * kv head, row), after k_take: the part of the parent's last page
// that the row takes over, whole groups of 8 positions.
__global__ void __launch_bounds__(kNT) k_copy_tails(TableArgs a, CopyArgs c) {
  const int row = blockIdx.y, p = parent_of(a, row);
  if (p < 0) return;
  const long long n = taken_over(a, row, p);
  const int rest = (int)(n & (a.ps - 1));
  const size_t full = (size_t)(n >> a.ps_shift);
  if (rest == 0 || (size_t)a.holds(row) <= full) return;
  const int src = a.table[(size_t)p * a.ld + full], dst = a.table[(size_t)row * a.ld + full];
  if (!a.has(src) || !a.has(dst)) return;
  const int n8 = (rest + 7) >> 3;
  const int layer = blockIdx.x / c.nkv, h = blockIdx.x - layer * c.nkv;
  const size_t head = (size_t)c.hd * c.ps * c.esz, off = (size_t)layer * c.n_pages;
  const size_t so = ((off + src) * c.nkv + h) * head, to = ((off + dst) * c.nkv + h) * head;
  const int v16 = n8 * c.hd * c.esz / 2;  // 16-byte units: 8 elements of each dim, whole groups
  for (int i = threadIdx.x; i < v16; i += kNT)
    *reinterpret_cast<uint4 *>(c.to_v + to + (size_t)i * 16) =
        *reinterpret_cast<const uint4 *>(c.v + so + (size_t)i * 16);
  const int run = n8 * 4 * c.esz;  // 16-byte units of n8 * 8 positions at 8 dims
  const size_t pitch = (size_t)c.ps * 8 * c.esz;
  for (int i = threadIdx.x; i < run * (c.hd >> 3); i += kNT) {
    const int d8 = i / run;
    const size_t o = d8 * pitch + (size_t)(i - d8 * run) * 16;
    *reinterpret_cast<uint4 *>(c.to_k + to + o) = *reinterpret_cast<const uint4 *>(c.k + so + o);
  }
}

struct MoveArgs {
  int32_t *number, *order;  // new number of a page; page of a number
  int32_t *to_table, *to_held, *to_refs, *live;
  size_t to_ld;
};

// The live pages numbered; the other pool's counts.
__global__ void __launch_bounds__(kNT) k_number(TableArgs a, CopyArgs c, MoveArgs m) {
  const int chunk = blockIdx.x, tid = threadIdx.x;
  int live, in;
  const int base = chunks_before(a, chunk, &live);
  if (chunk == 0 && tid == 0) *m.live = live;
  for (uint32_t p = live + chunk * kNT + tid; p < c.to_pages; p += gridDim.x * kNT) m.to_refs[p] = 0;
  if (chunk >= a.chunks) return;
  const uint32_t first = chunk * (uint32_t)kChunk + tid * kPer;
  const uint32_t on = wanted<true>(a, first);
  int rank = base + sum_before<kNT>(__popc(on), &in);
  for (int j = 0; j < kPer; j++) {
    if (first + j >= a.n_pages) break;
    const bool is = on >> j & 1, fits = (uint32_t)rank < c.to_pages;
    m.number[first + j] = is && fits ? rank : -1;
    if (is && fits) {
      m.order[rank] = (int)first + j;
      m.to_refs[rank] = a.refs[first + j];
    }
    rank += is;
  }
}

// grid (columns / 256, row)
__global__ void __launch_bounds__(kNT) k_rename(TableArgs a, MoveArgs m) {
  const size_t col = (size_t)blockIdx.x * kNT + threadIdx.x;
  const int row = blockIdx.y, held = a.holds(row);
  if (col == 0) m.to_held[row] = held;
  if (col >= m.to_ld) return;
  int to = -1;
  if (col < (size_t)held) {
    const int page = a.table[(size_t)row * a.ld + col];
    if (a.has(page)) to = m.number[page];
  }
  m.to_table[(size_t)row * m.to_ld + col] = to;
}

constexpr int kSlice = 32768;  // bytes that a workgroup moves at a time

// Pages of every layer, keys then values, in slices.
__global__ void __launch_bounds__(kNT) k_move_pages(CopyArgs c, MoveArgs m) {
  const size_t bytes = (size_t)c.nkv * c.hd * c.ps * c.esz;  // of a page
  const uint32_t slices = (uint32_t)((bytes + kSlice - 1) / kSlice);
  const uint64_t pages = min((uint32_t)*m.live, c.to_pages), items = pages * 2 * c.n_layers * slices;
  for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const uint32_t slice = (uint32_t)(i % slices), page = (uint32_t)(i / slices % pages);
    const uint32_t kind = (uint32_t)(i / slices / pages), layer = kind >> 1;
    const size_t at = (size_t)slice * kSlice;
    const uint8_t *src = (kind & 1 ? c.v : c.k) + ((size_t)layer * c.n_pages + m.order[page]) * bytes + at;
    uint8_t *dst = (kind & 1 ? c.to_v : c.to_k) + ((size_t)layer * c.to_pages + page) * bytes + at;
    const int n = (int)min((size_t)kSlice, bytes - at) / 16;
    for (int u = threadIdx.x; u < n; u += kNT)
      reinterpret_cast<uint4 *>(dst)[u] = reinterpret_cast<const uint4 *>(src)[u];
  }
}

// ---------------------------------------------------------------- host
struct Space {
  size_t need, before, count, number, order, total;
  int chunks;
};
Space space_of(const syn_hip_kv_tables &t) {
  Space s;
  s.chunks = (int)cdiv(t.n_pages, kChunk);
  s.need = 0;
  s.before = s.need + (size_t)t.n_seqs * 4;
  s.count = s.before + ((size_t)t.n_seqs + 1) * 4;
  s.number = s.count + (size_t)s.chunks * 4;
  s.order = s.number + (size_t)t.n_pages * 4;
  s.total = round_up(s.order + (size_t)t.n_pages * 4, 16);
  return s;
}

syn_status_t check_tables(const syn_hip_kv_tables *t, const char *who, bool buffers) {
  if (!t) return SYN_ERR_NULL_PTR;
  if (t->page_size < 8 || t->page_size > kKvMaxPage || (t->page_size & (t->page_size - 1))) {
    set_error(std::string(who) + ": page_size must be a power of two from 8 to 1024");
    return SYN_ERR_INVALID_ARG;
  }
  if (!t->n_pages || t->n_pages > kMaxTablePages || t->n_seqs > 65535u ||
      // (needs and their sums are 32 bits)
      (uint64_t)t->n_seqs * t->ld_table > 0x7fffffffu) {
    set_error(std::string(who) + ": 1 to 2^24 pages, at most 65535 rows and 2^31 - 1 entries");
    return SYN_ERR_INVALID_ARG;
  }
  if (buffers && t->n_seqs && (!t->refs || !t->held || (t->ld_table && !t->table))) return SYN_ERR_NULL_PTR;
  return SYN_OK;
}

syn_status_t check_space(const Space &s, const void *ws, size_t bytes, const char *who) {
  if (!ws) return SYN_ERR_NULL_PTR;
  if (!aligned16(ws) || bytes < s.total) {
    set_error(std::string(who) + ": workspace unaligned or too small");
    return SYN_ERR_INVALID_ARG;
  }
  return SYN_OK;
}

syn_status_t check_pool(const syn_hip_kv_pages *pages, const syn_hip_kv_tables *t, const char *who) {
  SYN_TRY(check_pages(pages, who));
  if (pages->page_size != t->page_size || pages->n_pages != t->n_pages) {
    set_error(std::string(who) + ": pool and tables differ in pages or their size");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  if ((uint64_t)pages->n_layers * pages->n_kv_heads > kMaxThreads / kNT) {
    set_error(std::string(who) + ": too many layers or heads");
    return SYN_ERR_INVALID_ARG;
  }
  return SYN_OK;
}

TableArgs table_args(const syn_hip_kv_tables &t, const int32_t *parent, const int32_t *len, void *ws) {
  const Space s = space_of(t);
  uint8_t *w = static_cast<uint8_t *>(ws);
  TableArgs a{};
  a.table = t.table;
  a.held = t.held;
  a.refs = t.refs;
  a.len = len;
  a.parent = parent;
  a.ld = t.ld_table;
  a.n_pages = t.n_pages;
  a.n_seqs = (int)t.n_seqs;
  a.chunks = s.chunks;
  a.ps = (int)t.page_size;
  a.ps_shift = 31 - __builtin_clz(t.page_size);
  a.need = reinterpret_cast<int32_t *>(w + s.need);
  a.before = reinterpret_cast<int32_t *>(w + s.before);
  a.count = reinterpret_cast<int32_t *>(w + s.count);
  return a;
}

template <bool FORK> syn_status_t launch_take(const TableArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(k_rows<FORK>, dim3((unsigned)cdiv(a.n_seqs, kNT / 64)), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_count<false>, dim3(a.chunks + 1), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_take, dim3(a.chunks), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

bool overlap(const void *a, const void *b, size_t na, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

}  // namespace

}  // namespace syn

using namespace syn;

extern "C" {

syn_status_t syn_hip_kv_tables_workspace(const syn_hip_kv_tables *t, size_t *bytes) {
  if (!bytes) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_tables(t, "kv_tables", false));
  *bytes = space_of(*t).total;
  return SYN_OK;
}

syn_status_t syn_hip_kv_resize(const syn_hip_kv_tables *t, const int32_t *d_len, void *d_workspace,
                               size_t workspace_bytes, void *stream) {
  SYN_TRY(check_tables(t, "kv_resize", true));
  if (t->n_seqs == 0) return SYN_OK;
  if (!d_len) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_space(space_of(*t), d_workspace, workspace_bytes, "kv_resize"));
  SYN_TRY(ensure_init());
  return launch_take<false>(table_args(*t, nullptr, d_len, d_workspace), pick_stream(stream));
}

syn_status_t syn_hip_kv_fork(const syn_hip_kv_pages *pages, const syn_hip_kv_tables *t,
                             const int32_t *d_parent, const int32_t *d_len, void *d_workspace,
                             size_t workspace_bytes, void *stream) {
  SYN_TRY(check_tables(t, "kv_fork", true));
  SYN_TRY(check_pool(pages, t, "kv_fork"));
  if (t->n_seqs == 0) return SYN_OK;
  if (!d_parent || !d_len) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_space(space_of(*t), d_workspace, workspace_bytes, "kv_fork"));
  SYN_TRY(ensure_init());
  hipStream_t s = pick_stream(stream);
  const TableArgs a = table_args(*t, d_parent, d_len, d_workspace);
  SYN_TRY(launch_take<true>(a, s));
  uint8_t *k = static_cast<uint8_t *>(pages->k), *v = static_cast<uint8_t *>(pages->v);
  const CopyArgs c{k, v, k, v, pages->n_pages, pages->n_pages, (int)pages->n_layers,
                   (int)pages->n_kv_heads, (int)pages->head_dim, (int)pages->page_size,
                   (int)kv_elem_bytes(pages->dtype)};
  hipLaunchKernelGGL(k_copy_tails, dim3(pages->n_layers * pages->n_kv_heads, t->n_seqs), dim3(kNT), 0, s,
                     a, c);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

syn_status_t syn_hip_kv_compact(const syn_hip_kv_pages *from, const syn_hip_kv_tables *t,
                                const syn_hip_kv_pages *to, const syn_hip_kv_tables *u,
                                int32_t *d_live, void *d_workspace, size_t workspace_bytes,
                                void *stream) {
  SYN_TRY(check_tables(t, "kv_compact", true));
  SYN_TRY(check_tables(u, "kv_compact", true));
  SYN_TRY(check_pool(from, t, "kv_compact"));
  SYN_TRY(check_pool(to, u, "kv_compact"));
  if (from->dtype != to->dtype || from->page_size != to->page_size || from->n_layers != to->n_layers ||
      from->n_kv_heads != to->n_kv_heads || from->head_dim != to->head_dim || t->n_seqs != u->n_seqs ||
      u->ld_table < t->ld_table) {
    set_error("kv_compact: pools of other pages, or tables of other rows or fewer columns");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  const size_t fb = kv_pool_bytes(*from), tb = kv_pool_bytes(*to);
  if (overlap(from->k, to->k, fb, tb) || overlap(from->k, to->v, fb, tb) ||
      overlap(from->v, to->k, fb, tb) || overlap(from->v, to->v, fb, tb) ||
      (t->n_seqs && (t->table == u->table || t->held == u->held || t->refs == u->refs))) {
    set_error("kv_compact: the pools, or their tables, are not apart");
    return SYN_ERR_INVALID_ARG;
  }
  if (t->n_seqs == 0) return SYN_OK;
  if (!d_live) return SYN_ERR_NULL_PTR;
  const Space sp = space_of(*t);
  SYN_TRY(check_space(sp, d_workspace, workspace_bytes, "kv_compact"));
  SYN_TRY(ensure_init());
  hipStream_t s = pick_stream(stream);
  const TableArgs a = table_args(*t, nullptr, nullptr, d_workspace);
  const CopyArgs c{static_cast<uint8_t *>(from->k), static_cast<uint8_t *>(from->v),
                   static_cast<uint8_t *>(to->k), static_cast<uint8_t *>(to->v), from->n_pages,
                   to->n_pages, (int)from->n_layers, (int)from->n_kv_heads, (int)from->head_dim,
                   (int)from->page_size, (int)kv_elem_bytes(from->dtype)};
  uint8_t *w = static_cast<uint8_t *>(d_workspace);
  const MoveArgs m{reinterpret_cast<int32_t *>(w + sp.number), reinterpret_cast<int32_t *>(w + sp.order),
                   u->table, u->held, u->refs, d_live, u->ld_table};
  hipLaunchKernelGGL(k_count<true>, dim3(a.chunks + 1), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_number, dim3(a.chunks), dim3(kNT), 0, s, a, c, m);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_rename, dim3((unsigned)std::max<size_t>(1, cdiv(u->ld_table, kNT)), t->n_seqs),
                     dim3(kNT), 0, s, a, m);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_move_pages, dim3(2048), dim3(kNT), 0, s, c, m);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // extern "C"
