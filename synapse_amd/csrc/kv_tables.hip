// Page tables of a paged cache: pages taken and given back, sequences that
// continue another one's pages, live pages moved to another pool.
//
// A page's count is the number of table entries that name it, and a page of
// count 0 is free, so there is no list of free pages to keep in order: whoever
// needs pages gets the free ones of lowest number, the rows in order and the
// columns of a row in order, whatever order the workgroups run in.
//
// Pages that are copied are bound by their bytes: all of a pool of 480 live pages
// of 28 layers to another, 7 GB read and written, 1367 us, 5.2 TB/s (a large copy
// reaches 4.7); the last pages of 96 rows that continue 32 others 111 us, 4.2 TB/s
// of what HBM has to read (a parent's page once) and write.  The tables are a few
// dependent loads: 16 rows 4 us, 1024 rows over 262144 pages 3 + 2.5 + 7.5.
#include <algorithm>

#include "kv_pages.hpp"
#include "wave_ops.hpp"

namespace syn {

namespace {

constexpr int kNT = 256;
constexpr int kPoolNT = 1024;           // of a workgroup that looks through a chunk of the pool
constexpr int kPer = 4;                 // pages of a thread
constexpr int kChunk = kPoolNT * kPer;  // pages of a workgroup
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
  int32_t *col;     // [n_seqs] the column that a row's first one goes to
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
    a.col[row] = held;
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
    a.col[row] = full;
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
  const int upto = wave_upto(x);
  int s = wave_shifted(upto);
  __syncthreads();
  if (lane == 63) w[wave] = upto;
  __syncthreads();
  int t = 0;
  for (int i = 0; i < NT / 64; i++) {
    if (i < wave) s += w[i];
    t += w[i];
  }
  *all = t;
  return s;
}

// the wanted pages among a thread's: bit j for page first + j (PER of them, a
// multiple of 4; counts are read where the atomics are)
template <bool LIVE, int PER>
__device__ __forceinline__ uint32_t wanted(const int32_t *refs, uint32_t first, uint32_t n_pages) {
  uint32_t on = 0;
  int n[PER];
  if (first + PER <= n_pages && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < PER; j += 4) {
      const i32x4 x = *reinterpret_cast<const i32x4 *>(refs + first + j);
#pragma unroll
      for (int k = 0; k < 4; k++) n[j + k] = x[k];
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; j++) n[j] = first + j < n_pages ? refs[first + j] : -1;
  }
#pragma unroll
  for (int j = 0; j < PER; j++) on |= (LIVE ? n[j] > 0 : n[j] == 0) ? 1u << j : 0u;
  return on;
}

// the last row with before[row] <= rank (rows that need none have the same sum as
// the row after them)
__device__ __forceinline__ int row_of(const int32_t *before, int n, int rank) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (before[mid] <= rank)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// workgroup 0: the rows' needs added up; the others: a chunk's wanted pages
template <bool LIVE> __global__ void __launch_bounds__(kPoolNT) k_count(TableArgs a) {
  const int tid = threadIdx.x;
  int all;
  if (blockIdx.x == 0) {
    if (LIVE) return;
    const int each = (a.n_seqs + kPoolNT - 1) / kPoolNT, r0 = min(tid * each, a.n_seqs), r1 = min(r0 + each, a.n_seqs);
    int sum = 0;
    for (int r = r0; r < r1; r++) sum += a.need[r];
    int at = sum_before<kPoolNT>(sum, &all);
    for (int r = r0; r < r1; r++) {
      a.before[r] = at;
      at += a.need[r];
    }
    if (tid == 0) a.before[a.n_seqs] = all;
    return;
  }
  const uint32_t chunk = blockIdx.x - 1;
  (void)sum_before<kPoolNT>(__popc(wanted<LIVE, kPer>(a.refs, chunk * kChunk + tid * kPer, a.n_pages)), &all);
  if (tid == 0) a.count[chunk] = all;
}

// wanted pages of the chunks before this one, and of all
__device__ __forceinline__ int chunks_before(const TableArgs &a, int chunk, int *all) {
  int below = 0, total = 0, sum;
  for (int c = threadIdx.x; c < a.chunks; c += kPoolNT) {
    const int n = a.count[c];
    total += n;
    below += c < chunk ? n : 0;
  }
  (void)sum_before<kPoolNT>(total, all);
  (void)sum_before<kPoolNT>(below, &sum);
  return sum;
}

constexpr int kLdsRows = 4096;  // rows whose sums a workgroup searches in LDS

// The i-th free page goes to the i-th place that needs one: a chunk's free pages
// are listed in LDS, so that each thread has one of them in turn.
__global__ void __launch_bounds__(kPoolNT) k_take(TableArgs a) {
  __shared__ uint16_t list[kChunk];
  __shared__ int32_t sums[kLdsRows];
  const int chunk = blockIdx.x, tid = threadIdx.x;
  int free, in;
  const int base = chunks_before(a, chunk, &free);
  const int needed = a.before[a.n_seqs];
  if (chunk == 0)
    for (int r = tid; r < a.n_seqs; r += kPoolNT) {
      const int n = max(0, min(a.need[r], free - a.before[r]));
      if (n) a.held[r] += n;
    }
  if (base >= needed) return;
  const uint32_t on = wanted<false, kPer>(a.refs, chunk * (uint32_t)kChunk + tid * kPer, a.n_pages);
  int rank = sum_before<kPoolNT>(__popc(on), &in);
  for (uint32_t m = on; m; m &= m - 1) list[rank++] = (uint16_t)(tid * kPer + __ffs(m) - 1);
  const bool lds = a.n_seqs <= kLdsRows;
  if (lds)
    for (int r = tid; r < a.n_seqs; r += kPoolNT) sums[r] = a.before[r];
  __syncthreads();
  const int most = min(in, needed - base);
  for (int i = tid; i < most; i += kPoolNT) {
    const int row = row_of(lds ? sums : a.before, a.n_seqs, base + i);
    const int page = chunk * kChunk + list[i];
    a.table[(size_t)row * a.ld + a.col[row] + (base + i - a.before[row])] = page;
    a.refs[page] = 1;
  }
}

// ---- the whole of it by one workgroup, where little is to be done: a launch and
// five steps with a barrier between, their entries dealt to all threads.  (Two calls
// for 16 rows of 44 entries: 8.1 us, by the launches above 20.  128 rows of 24
// entries that all change: 16 us in the kernel, 14.5 in the three.)  The bound on
// entries is for calls that change all of them; most change few.
constexpr int kSmallNT = 1024;
constexpr int kSmallRows = 1024, kSmallEntries = 16384;
constexpr uint32_t kSmallPages = 65536;

template <bool FORK> __global__ void __launch_bounds__(kSmallNT) k_tables_small(TableArgs a) {
  // entries that a row gives back, shares, and takes: sums over the rows before
  __shared__ int32_t back[kSmallRows], share[FORK ? kSmallRows : 1], take[kSmallRows];
  __shared__ int32_t first[kSmallRows], col[kSmallRows], from[FORK ? kSmallRows : 1];
  const int tid = threadIdx.x, n = a.n_seqs;
  int n_back = 0, n_share = 0, n_take = 0, keep = 0, parent = -1;
  bool changed = false;
  if (tid < n) {
    const int held = a.holds(tid);
    if (FORK) {
      parent = parent_of(a, tid);
      if (parent >= 0) {
        const long long m = taken_over(a, tid, parent);
        n_back = held;
        n_share = keep = (int)(m >> a.ps_shift);
        n_take = (m & (a.ps - 1)) != 0;
        first[tid] = 0;
        changed = true;
      }
      from[tid] = parent;
    } else {
      const int len = a.len[tid], want = len < 0 ? held : (int)min((size_t)a.pages_of(len), a.ld);
      keep = min(held, want);
      n_back = held - keep;
      n_take = want - keep;
      first[tid] = keep;
      changed = len >= 0;
    }
    col[tid] = keep;
  }
  int all_back, all_share = 0, all_take;
  const int b0 = sum_before<kSmallNT>(n_back, &all_back), t0 = sum_before<kSmallNT>(n_take, &all_take);
  if (tid < n) back[tid] = b0, take[tid] = t0;
  if (FORK) {
    const int s0 = sum_before<kSmallNT>(n_share, &all_share);
    if (tid < n) share[tid] = s0;
  }
  __syncthreads();
  for (int e = tid; e < all_back; e += kSmallNT) {
    const int row = row_of(back, n, e);
    int32_t *t = a.table + (size_t)row * a.ld + first[row] + (e - back[row]);
    drop(a, *t);
    *t = -1;
  }
  if (FORK) {
    __syncthreads();
    for (int e = tid; e < all_share; e += kSmallNT) {
      const int row = row_of(share, n, e), c = e - share[row];
      const int page = a.table[(size_t)from[row] * a.ld + c];
      if (a.has(page)) atomicAdd(a.refs + page, 1);
      a.table[(size_t)row * a.ld + c] = page;
    }
  }
  // every count has changed where it is read next (an agent's fence would write
  // the L2 back and drop it)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int given = 0;
  constexpr int kEach = 8;
  for (uint32_t p0 = 0; p0 < a.n_pages && given < all_take; p0 += kSmallNT * kEach) {
    int in;
    const uint32_t p = p0 + tid * kEach;
    uint32_t on = wanted<false, kEach>(a.refs, p, a.n_pages);
    int rank = given + sum_before<kSmallNT>(__popc(on), &in);
    for (; on && rank < all_take; on &= on - 1, rank++) {
      const int page = (int)p + __ffs(on) - 1, row = row_of(take, n, rank);
      a.table[(size_t)row * a.ld + col[row] + (rank - take[row])] = page;
      a.refs[page] = 1;
    }
    given += in;
  }
  if (changed) a.held[tid] = keep + max(0, min(n_take, given - t0));
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
  // 16-byte units of 8 elements: V whole groups of 8 positions of every dim, K n8 * 8
  // positions of every 8 dims
  const int units = n8 * c.hd * c.esz / 2, run = n8 * 4 * c.esz;
  const size_t pitch = (size_t)c.ps * 8 * c.esz;
  auto at = [&](int i) {
    if (i < units) return (size_t)i * 16;
    const int k = i - units, d8 = k / run;
    return d8 * pitch + (size_t)(k - d8 * run) * 16;
  };
  constexpr int kAtOnce = 4;
  for (int i0 = threadIdx.x; i0 < 2 * units; i0 += kAtOnce * kNT) {
    u32x4 x[kAtOnce];
    size_t o[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      const int i = min(i0 + j * kNT, 2 * units - 1);
      o[j] = at(i);
      x[j] = *reinterpret_cast<const u32x4 *>((i < units ? c.v : c.k) + so + o[j]);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      const int i = i0 + j * kNT;
      if (i < 2 * units) *reinterpret_cast<u32x4 *>((i < units ? c.to_v : c.to_k) + to + o[j]) = x[j];
    }
  }
}

struct MoveArgs {
  int32_t *number, *order;  // new number of a page; page of a number
  int32_t *to_table, *to_held, *to_refs, *live;
  size_t to_ld;
};

// The live pages numbered; the other pool's counts.
__global__ void __launch_bounds__(kPoolNT) k_number(TableArgs a, CopyArgs c, MoveArgs m) {
  const int chunk = blockIdx.x, tid = threadIdx.x;
  int live, in;
  const int base = chunks_before(a, chunk, &live);
  if (chunk == 0 && tid == 0) *m.live = live;
  for (uint32_t p = live + chunk * kPoolNT + tid; p < c.to_pages; p += gridDim.x * kPoolNT) m.to_refs[p] = 0;
  if (chunk >= a.chunks) return;
  const uint32_t first = chunk * (uint32_t)kChunk + tid * kPer;
  const uint32_t on = wanted<true, kPer>(a.refs, first, a.n_pages);
  int rank = base + sum_before<kPoolNT>(__popc(on), &in);
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

// The same and the tables by one workgroup, where little is to be done.
__global__ void __launch_bounds__(kSmallNT) k_rename_small(TableArgs a, CopyArgs c, MoveArgs m) {
  const int tid = threadIdx.x;
  constexpr int kEach = 8;
  int live = 0, in;
  for (uint32_t p0 = 0; p0 < a.n_pages; p0 += kSmallNT * kEach) {
    const uint32_t p = p0 + tid * kEach;
    const uint32_t on = wanted<true, kEach>(a.refs, p, a.n_pages);
    int rank = live + sum_before<kSmallNT>(__popc(on), &in);
#pragma unroll
    for (int j = 0; j < kEach; j++) {
      if (p + j >= a.n_pages) break;
      const bool is = on >> j & 1, fits = (uint32_t)rank < c.to_pages;
      m.number[p + j] = is && fits ? rank : -1;
      if (is && fits) {
        m.order[rank] = (int)(p + j);
        m.to_refs[rank] = a.refs[p + j];
      }
      rank += is;
    }
    live += in;
  }
  if (tid == 0) *m.live = live;
  for (uint32_t p = live + tid; p < c.to_pages; p += kSmallNT) m.to_refs[p] = 0;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the numbers are read below
  __syncthreads();
  for (int r = tid; r < a.n_seqs; r += kSmallNT) m.to_held[r] = a.holds(r);
  const uint32_t entries = (uint32_t)(a.n_seqs * m.to_ld);
  for (uint32_t e = tid; e < entries; e += kSmallNT) {
    const uint32_t row = e / (uint32_t)m.to_ld, col = e - row * (uint32_t)m.to_ld;
    int to = -1;
    if ((int)col < a.holds((int)row)) {
      const int page = a.table[(size_t)row * a.ld + col];
      if (a.has(page)) to = m.number[page];
    }
    m.to_table[e] = to;
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

constexpr int kSlice = 16384;  // bytes that a workgroup moves at a time

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
    constexpr int kAtOnce = kSlice / 16 / kNT;  // all of a slice in flight
    u32x4 x[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++)
      x[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src) + min((int)threadIdx.x + j * kNT, n - 1));
#pragma unroll
    for (int j = 0; j < kAtOnce; j++)
      if ((int)threadIdx.x + j * kNT < n)
        __builtin_nontemporal_store(x[j], reinterpret_cast<u32x4 *>(dst) + threadIdx.x + j * kNT);
  }
}

// ---------------------------------------------------------------- host
struct Space {
  size_t need, before, count, col, number, order, total;
  int chunks;
};
Space space_of(const syn_hip_kv_tables &t) {
  Space s;
  s.chunks = (int)cdiv(t.n_pages, kChunk);
  s.need = 0;
  s.before = s.need + (size_t)t.n_seqs * 4;
  s.count = s.before + ((size_t)t.n_seqs + 1) * 4;
  s.col = s.count + (size_t)s.chunks * 4;
  s.number = s.col + (size_t)t.n_seqs * 4;
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
  a.col = reinterpret_cast<int32_t *>(w + s.col);
  return a;
}

template <bool FORK> syn_status_t launch_take(const TableArgs &a, hipStream_t s) {
  if (a.n_seqs <= kSmallRows && a.n_pages <= kSmallPages && a.n_seqs * a.ld <= kSmallEntries) {
    hipLaunchKernelGGL(k_tables_small<FORK>, dim3(1), dim3(kSmallNT), 0, s, a);
    SYN_LAUNCH_CHECK();
    return SYN_OK;
  }
  hipLaunchKernelGGL(k_rows<FORK>, dim3((unsigned)cdiv(a.n_seqs, kNT / 64)), dim3(kNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_count<false>, dim3(a.chunks + 1), dim3(kPoolNT), 0, s, a);
  SYN_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_take, dim3(a.chunks), dim3(kPoolNT), 0, s, a);
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
  if (std::max(from->n_pages, to->n_pages) <= kSmallPages && t->n_seqs * u->ld_table <= kSmallEntries) {
    hipLaunchKernelGGL(k_rename_small, dim3(1), dim3(kSmallNT), 0, s, a, c, m);
    SYN_LAUNCH_CHECK();
  } else {
    hipLaunchKernelGGL(k_count<true>, dim3(a.chunks + 1), dim3(kPoolNT), 0, s, a);
    SYN_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_number, dim3(a.chunks), dim3(kPoolNT), 0, s, a, c, m);
    SYN_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_rename, dim3((unsigned)std::max<size_t>(1, cdiv(u->ld_table, kNT)), t->n_seqs),
                       dim3(kNT), 0, s, a, m);
    SYN_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(k_move_pages, dim3(2048), dim3(kNT), 0, s, c, m);
  SYN_LAUNCH_CHECK();
  return SYN_OK;
}

}  // extern "C"
