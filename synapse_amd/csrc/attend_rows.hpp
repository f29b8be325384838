// Attention of a few query rows over a paged cache: a wave's 16 rows of a kv
// head over runs of positions, the waves of a workgroup that share them, and the
// join of a split run's parts (prefix_attention.hip, paged_attention.hip).
#pragma once

#include "kv_pages.hpp"
#include "lds_dma.hpp"

namespace syn {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kWaves = 4;
constexpr int kTile = 32;  // positions a wave takes at a time

// The query rows of a token or of several, and where their results go.
struct RowArgs {
  const float *q;
  float *out;
  size_t ldq, ldo;
  int nh, rep;
  float scale;  // times log2(e): exponentials are powers of two
  // parts of query row (token, head) are po[(token * nh + head) * parts +
  // part][hd], pml[..][2] (max, sum)
  int parts;
  float *po, *pml;
  bool q16;  // rows of queries are 16-byte aligned
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
  // A weight is 2^kBias where its score is the reference maximum, and at most
  // 2^(kBias + kSlack), within f16.  From kLeast = 2^kLeastLog on, two parts
  // hold it to 2^-22 of itself (f16's steps end at 2^-24); a smaller one
  // takes part in multiples of kLift (add_small), up to 2^15 again.
  static constexpr float kBias = 12.0f, kSlack = 3.0f;
  static constexpr float kLeastLog = -3.0f, kLeast = 0.125f, kLift = 262144.0f;
  static __device__ __forceinline__ V load(const _Float16 *p) {
    return *reinterpret_cast<const V *>(p);
  }
  // both parts to nearest: together within 2^-22 of x, or within 2^-25
  static __device__ __forceinline__ void split(const float *x, V *p) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f16x2 h = __builtin_convertvector((f32x2{x[j], x[j + 1]}), f16x2);
      const f16x2 r = __builtin_convertvector((f32x2{__builtin_fmaf((float)h[0], -1.0f, x[j]),
                                                     __builtin_fmaf((float)h[1], -1.0f, x[j + 1])}), f16x2);
      p[0][j] = h[0], p[0][j + 1] = h[1], p[1][j] = r[0], p[1][j + 1] = r[1];
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
  static constexpr float kBias = 0.0f, kSlack = 8.0f;
  static __device__ __forceinline__ V load(const __bf16 *p) {
    return *reinterpret_cast<const V *>(p);
  }
  static __device__ __forceinline__ void split(const float *x, V *p) {
    // the upper 16 bits of x and of what is left, twice: 24 bits in three parts
    uint32_t u[3][8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float r = x[j];
#pragma unroll
      for (int k = 0; k < 3; k++) {
        u[k][j] = __float_as_uint(r) & 0xffff0000u;
        r -= __uint_as_float(u[k][j]);
      }
    }
#pragma unroll
    for (int k = 0; k < 3; k++) {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = __builtin_amdgcn_perm(u[k][2 * j + 1], u[k][2 * j], 0x07060302u);
      p[k] = __builtin_bit_cast(V, w);
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
  static constexpr float kBias = 0.0f, kSlack = 8.0f;
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

// over the four groups of 16 lanes: a swap of halves (of odd and even groups)
// of x with itself leaves each lane its own value and its partner's
template <class Op> __device__ __forceinline__ float over_groups(float x, Op op) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(op(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_max(float x) {
  return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float groups_sum(float x) {
  return over_groups(x, [](float a, float b) { return a + b; });
}

// Positions from .. to of a page table, dealt to the waves by tiles, the first
// to wave `first`.
struct Run {
  const int32_t *table;
  int from, to, first;
};

// A kv head's K and V of page 0, and the bytes from page to page.
struct HeadBase {
  const uint8_t *k, *v;
  uint32_t page_bytes;
};

// One wave's part of the work: 16 query rows of a kv head.  FULL: hd is 32 NC.
// CAUSAL: a row sees positions of its own, lo to lim (see()), of those that the
// run has.  RING: tiles that the ring in LDS holds, if not as many as below.
template <class T, int NC, bool FULL, bool CAUSAL = false, int RING = 0> struct Rows {
  using F = Frag<T>;
  using V = typename F::V;
  static constexpr int DT = 2 * NC;           // tiles of 16 dims (hd <= 32 NC)
  static constexpr int kFrags = 4 * NC;       // operand fragments of a tile of positions: K, then V
  static constexpr int kLoads = kFrags * (int)sizeof(V) / 16;  // 1 KiB direct loads of a tile
  static constexpr int kTileBytes = kLoads * 1024;
  // tiles that the ring in LDS holds: 32 to 64 KiB, 128 where a tile has 64
  static constexpr int kRing = RING ? RING : (kTileBytes <= 16384 ? 4 : 2);
  // V asked for when the scores are formed, where registers are short
  static constexpr bool kLate = sizeof(V) != 16 || (RING == 3 && F::kParts == 3);
  static constexpr int kLd = 32 * NC + 4;     // f32 rows on different banks
  static constexpr int kJoinBytes = kWaves * 16 * kLd * 4;
  static constexpr int kLdsBytes = kRing * kTileBytes > kJoinBytes ? kRing * kTileBytes : kJoinBytes;
  V q[NC][F::kParts];
  f32x4 o[DT];
  float m, l, unscale;
  int lim, lo;             // CAUSAL: what the lane's row sees
  int all_from, all_to;    // what all rows of the wave see

  // The rows' queries times scale, each row for an f16 pool times the power of
  // two that puts its largest element into [2^11, 2^12): an element is held to
  // 2^-22 of itself, or 2^-36 of the row's largest.  Rows past the last repeat it.
  __device__ __forceinline__ void load_queries(const RowArgs &a, int hd, int seq0, int head, int row,
                                               int last) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int r = min(row + n, last), member = r / a.rep;
    const float *src = a.q + (size_t)(seq0 + member) * a.ldq +
                       (size_t)(head * a.rep + (r - member * a.rep)) * hd;
    float x[NC][8], top = 0.0f;
    if (a.q16) {
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(src + min((c * 4 + g) * 8, hd - 8));
        const f32x4 u = p[0], v = p[1];
#pragma unroll
        for (int j = 0; j < 4; j++) x[c][j] = u[j], x[c][j + 4] = v[j];
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) x[c][j] = src[min((c * 4 + g) * 8, hd - 8) + j];
    }
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[c][j] = (c * 4 + g) * 8 < hd ? x[c][j] * a.scale : 0.0f;
        top = fmaxf(top, fabsf(x[c][j]));
      }
    unscale = 1.0f;
    if constexpr (F::kParts == 2) {
      top = groups_max(top);
      int e = top > 0.0f && top < __builtin_huge_valf() ? 11 - ilogbf(top) : 0;
      e = min(max(e, -120), 120);  // a power of two within f32's own range either way
      const float up = __builtin_ldexpf(1.0f, e);
      unscale = __builtin_ldexpf(1.0f, -e);
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) x[c][j] *= up;
    }
#pragma unroll
    for (int c = 0; c < NC; c++) F::split(x[c], q[c]);
    m = kNegInf;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f32x4{0, 0, 0, 0};
  }

  // ---- a tile's operands: lane (g, n) has K of the position group n / 4 and
  // V of group g, of the four groups of 8 positions.  Positions past the end
  // are read at the last group there is.  Pages are looked up by scalar loads
  // (k0 is the same for the whole wave), which do not queue with the K and V
  // in flight; WIDE: a page holds whole tiles, so one serves all groups.
  struct Where {
    int p0, p1, p2, p3;  // pages of the groups
    __device__ __forceinline__ int of(int group) const {
      const int a = p0, b = p1, c = p2, d = p3;  // values, not places: kept in registers
      const int lo = group & 1 ? b : a, hi = group & 1 ? d : c;
      return group & 2 ? hi : lo;
    }
  };
  static __device__ __forceinline__ int spot(int k0, int group, int to) {
    return min(k0 + 8 * group, (to - 1) & ~7);
  }
  template <bool WIDE>
  static __device__ __forceinline__ Where look_up(const KvPool<T> &pool, const Run &r, int k0) {
    const auto *t = (const __attribute__((address_space(4))) int32_t *)(uintptr_t)r.table;
    const int p = t[(uint32_t)spot(k0, 0, r.to) >> pool.ps_shift];
    if (WIDE) return Where{p, p, p, p};
    return Where{p, t[(uint32_t)spot(k0, 1, r.to) >> pool.ps_shift],
                 t[(uint32_t)spot(k0, 2, r.to) >> pool.ps_shift],
                 t[(uint32_t)spot(k0, 3, r.to) >> pool.ps_shift]};
  }
  // which of the groups' pages are pages, a bit each
  template <bool WIDE>
  static __device__ __forceinline__ uint32_t found(const KvPool<T> &pool, const Where &w) {
    if (WIDE) return pool.has(w.p0) ? 15u : 0u;
    return (pool.has(w.p0) ? 1u : 0u) | (pool.has(w.p1) ? 2u : 0u) | (pool.has(w.p2) ? 4u : 0u) |
           (pool.has(w.p3) ? 8u : 0u);
  }
  // The addresses of a tile: K at k + koff (dims of a fragment) and V at v +
  // voff; a tile that one page holds whole has wave-uniform k and v.
  struct Tile {
    const uint8_t *k, *v;
  };
  template <bool WIDE>
  static __device__ __forceinline__ Tile tile_of(const KvPool<T> &pool, const HeadBase &hb, const Run &r,
                                                 int k0, const Where &w) {
    if (WIDE && k0 + kTile <= r.to) {
      const uint64_t page = (uint64_t)(uint32_t)(pool.has(w.p0) ? w.p0 : 0) * hb.page_bytes;
      const uint32_t slot = k0 & (pool.ps - 1);
      return Tile{hb.k + page + slot * (8 * (uint32_t)sizeof(T)),
                  hb.v + page + (slot >> 3) * (uint32_t)(pool.hd * 8 * (int)sizeof(T))};
    }
    // the offsets below are those of group n / 4 (K) and g (V) of a whole tile
    const int n4 = (threadIdx.x & 15) >> 2, g = (threadIdx.x & 63) >> 4;
    const int pk = w.of(n4), pv = w.of(g);
    const int sk = (spot(k0, n4, r.to) & (pool.ps - 1)) - 8 * n4;
    const int sv = ((spot(k0, g, r.to) & (pool.ps - 1)) >> 3) - g;
    return Tile{hb.k + (uint64_t)(uint32_t)(pool.has(pk) ? pk : 0) * hb.page_bytes +
                    (int64_t)(sk * 8 * (int)sizeof(T)),
                hb.v + (uint64_t)(uint32_t)(pool.has(pv) ? pv : 0) * hb.page_bytes +
                    (int64_t)(sv * (pool.hd * 8 * (int)sizeof(T)))};
  }
  // bytes to fragment f: K of half f % 2 at dims 32 (f / 2); V of dims 16 f
  static __device__ __forceinline__ uint32_t koff(const KvPool<T> &pool, int f) {
    const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
    const int d8 = FULL ? (f >> 1) * 4 + g : min((f >> 1) * 4 + g, (pool.hd >> 3) - 1);
    return (uint32_t)((d8 * pool.ps + 8 * (n >> 2) + (n & 3) +
                       (f & 1) * 4) * 8 * (int)sizeof(T));
  }
  static __device__ __forceinline__ uint32_t voff(const KvPool<T> &pool, int f) {
    const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
    const int d = FULL ? f * 16 + n : min(f * 16 + n, pool.hd - 1);
    return (uint32_t)((g * (FULL ? 32 * NC : pool.hd) + d) * 8 * (int)sizeof(T));
  }
  // the positions 8g .. 8g+7 whose weights this lane holds, a bit each
  static __device__ __forceinline__ uint32_t which(int k0, int to, uint32_t ok) {
    const int g = (threadIdx.x & 63) >> 4, left = ok >> g & 1 ? to - (k0 + 8 * g) : 0;
    return left >= 8 ? 0xff : (left <= 0 ? 0 : (1u << left) - 1);
  }

  __device__ __forceinline__ void see(int lo_, int lim_, int all_from_, int all_to_) {
    lo = lo_;
    lim = lim_;
    all_from = all_from_;
    all_to = all_to_;
  }
  // those of the positions 8g .. 8g+7 that the lane's row sees, a bit each
  __device__ __forceinline__ uint32_t seen(int k0) const {
    const int p = k0 + 8 * (int)((threadIdx.x & 63) >> 4), up = lim - p, down = lo - p;
    const uint32_t below = up >= 8 ? 0xff : (up <= 0 ? 0 : (1u << up) - 1);
    return below & (down <= 0 ? 0xff : (down >= 8 ? 0 : 0xffu << down));
  }

  // those of the positions 8g .. 8g+7 at which some dim of V is not finite, a bit each
  static __device__ __forceinline__ uint32_t odd(const V *v) {
    constexpr int kWords = (int)sizeof(V) / 4, kEach = kWords == 4 ? 2 : 1;
    // elements without their signs, the largest of all dims (above another in a word)
    uint32_t hi[kWords] = {}, lo[kWords] = {};
#pragma unroll
    for (int d = 0; d < DT; d++) {
      uint32_t w[kWords];
      __builtin_memcpy(w, &v[d], sizeof(V));
#pragma unroll
      for (int k = 0; k < kWords; k++) {
        hi[k] = max(hi[k], w[k] & 0x7fffffffu);
        if (kEach == 2) lo[k] = max(lo[k], w[k] << 16 & 0x7fffffffu);
      }
    }
    constexpr uint32_t kInf = F::kParts == 2 ? 0x7c000000u : 0x7f800000u;
    uint32_t on = 0;
#pragma unroll
    for (int k = 0; k < kWords; k++)
      on |= (hi[k] >= kInf ? 1u << (kEach * k + kEach - 1) : 0u) | (kEach == 2 && lo[k] >= kInf ? 1u << 2 * k : 0u);
    // over the 16 lanes of the group, each of which has other dims
    auto with = [&](int x) { on |= (uint32_t)x; };
    with(__builtin_amdgcn_update_dpp(0, (int)on, 0xb1, 0xf, 0xf, false));
    with(__builtin_amdgcn_update_dpp(0, (int)on, 0x4e, 0xf, 0xf, false));
    with(__builtin_amdgcn_update_dpp(0, (int)on, 0x141, 0xf, 0xf, false));
    with(__builtin_amdgcn_update_dpp(0, (int)on, 0x140, 0xf, 0xf, false));
    return on;
  }

  // ---- the two products of a tile
  __device__ __forceinline__ void scores(const V *k, f32x4 *s) const {
    s[0] = s[1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NC; c++) {
      s[0] = F::mma(k[2 * c], q[c], s[0]);
      s[1] = F::mma(k[2 * c + 1], q[c], s[1]);
    }
    // Read the sums before the next branch: where a conditional region lies
    // between, the compiler pads the matrix instruction's latency on the
    // longer way only.
    asm volatile("" : "+v"(s[0]), "+v"(s[1]));
  }
  __device__ __forceinline__ void weigh(const f32x4 *s, V *v, int k0, int to, uint32_t ok) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = s[0][j], x[j + 4] = s[1][j];
    const bool cut = k0 + kTile > to || ok != 15;
    if (cut || (CAUSAL && (k0 + kTile > all_to || k0 < all_from))) {
      uint32_t there = which(k0, to, ok);
      const uint32_t mine = CAUSAL ? there & seen(k0) : there;
      bool clear = !CAUSAL || cut;
      if constexpr (CAUSAL) {
        // A value that is not finite is none of the rows' that do not see it; those
        // that do are NaN.
        const uint32_t none = odd(v) & there;
        if (__any(none)) {
          if (none & mine) l = __builtin_nanf("");
          there &= ~none;
          clear = true;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[j] = mine >> j & 1 ? x[j] : kNegInf;
        if (!clear) continue;
#pragma unroll
        for (int d = 0; d < DT; d++)  // what is not there may hold anything: 0 times NaN is NaN
          if (!(there >> j & 1)) F::clear(v[d], j);
      }
    }
    float top = fmaxf(x[0], x[1]);
#pragma unroll
    for (int j = 2; j < 8; j += 2) top = fmaxf(fmaxf(x[j], x[j + 1]), top);
    top = groups_max(top) * unscale;
    // weights are relative to m, a maximum of earlier: the accumulators are
    // rescaled only when a score is 2^kSlack times above it
    if (__any(top > m + F::kSlack)) {
      const float up = fmaxf(m, top);
      const float back = __builtin_amdgcn_exp2f(m - (up == kNegInf ? 0.0f : up));
      m = up;
      l *= back;
#pragma unroll
      for (int d = 0; d < DT; d++) o[d] *= back;
    }
    const float ref = F::kBias - (m == kNegInf ? 0.0f : m);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = __builtin_fmaf(x[j], unscale, ref);
    bool small = false;
    if constexpr (F::kParts == 2) {
      float least = fminf(x[0], x[1]);
#pragma unroll
      for (int j = 2; j < 8; j += 2) least = fminf(fminf(x[j], x[j + 1]), least);
      small = __any(least < F::kLeastLog);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = __builtin_amdgcn_exp2f(x[j]);
    l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    float y[8];  // the weights below kLeast
    if constexpr (F::kParts == 2)
      if (small)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          y[j] = x[j] < F::kLeast ? x[j] : 0.0f;
          x[j] = x[j] < F::kLeast ? 0.0f : x[j];
        }
    V p[F::kParts];
    F::split(x, p);
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = F::mma(v[d], p, o[d]);
    if constexpr (F::kParts == 2)
      if (small) {
#pragma unroll
        for (int d = 0; d < DT; d++) asm volatile("" : "+v"(o[d]));  // as in scores()
        add_small(y, v);
      }
  }
  // Weights of which two parts would keep few bits or none: lifted until they are
  // not, their products are added to the sums in f32.  (At most nine rounds: no
  // weight is below 2^-149.)  Calls without such weights pay for the test and the
  // registers: at 128 dims 1 % (four prefixes of 32768 under 64 rows 109.8 us,
  // 108.7 without) to 7 % (two of 8000 under 128 rows 38.8, 36.4), at 64, where a CU
  // then holds three workgroups and not four, 10 % (48 sequences over 8200: 37.9,
  // 34.4).  Scores spread over 36 binary orders, where most tiles come here, take
  // 215 us where 109 do without.
  __device__ __forceinline__ void add_small(float *y, const V *v) {
    float back = 1.0f;
    bool left = false;
#pragma unroll
    for (int j = 0; j < 8; j++) left |= y[j] > 0.0f;
    while (__any(left)) {
      float z[8];
      left = false;
      back *= 1.0f / F::kLift;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        y[j] *= F::kLift;
        z[j] = y[j] < F::kLeast ? 0.0f : y[j];
        y[j] = y[j] < F::kLeast ? y[j] : 0.0f;
        left |= y[j] > 0.0f;
      }
      V p[F::kParts];
      F::split(z, p);
#pragma unroll
      for (int d = 0; d < DT; d++) {
        f32x4 t = F::mma(v[d], p, f32x4{0, 0, 0, 0});
        asm volatile("" : "+v"(t));
#pragma unroll
        for (int k = 0; k < 4; k++) o[d][k] = __builtin_fmaf(t[k], back, o[d][k]);
      }
    }
  }

  // ---- 16 rows in all: `waves` waves (a power of two) take the tiles of a run
  // in turn, K and V in registers.  One set of them: the next tile's K is
  // requested when this one's scores are formed, its V when this one's product
  // is.
  template <bool WIDE>
  __device__ __forceinline__ void run_alone(const KvPool<T> &pool, const HeadBase &hb, const Run &r,
                                            int waves) {
    const int kStep = kTile * waves;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int k0 = r.from + ((wave - r.first) & (waves - 1)) * kTile;
    if (k0 >= r.to) return;
    // (FULL: the fragments' offsets are even steps from the first)
    const uint32_t k_first = koff(pool, 0), v_first = voff(pool, 0);
    const uint32_t k_step = 32 * (uint32_t)(pool.ps * (int)sizeof(T));
    uint32_t ko[FULL ? 1 : 2 * NC], vo[FULL ? 1 : DT];
    if constexpr (!FULL)
#pragma unroll
      for (int f = 0; f < 2 * NC; f++) ko[f] = koff(pool, f), vo[f] = voff(pool, f);
    auto k_load = [&](const uint8_t *k, int f) {
      const uint8_t *at;
      if constexpr (FULL)
        at = k + k_first + (f >> 1) * k_step + (f & 1) * (32 * (int)sizeof(T));
      else
        at = k + ko[f];
      return F::load(reinterpret_cast<const T *>(at));
    };
    auto v_load = [&](const uint8_t *v, int d) {
      const uint8_t *at;
      if constexpr (FULL)
        at = v + v_first + d * (128 * (int)sizeof(T));
      else
        at = v + vo[d];
      return F::load(reinterpret_cast<const T *>(at));
    };
    V kf[2 * NC], vf[DT];
    Where w = look_up<WIDE>(pool, r, k0);
    uint32_t ok = found<WIDE>(pool, w);
    {
      const Tile t = tile_of<WIDE>(pool, hb, r, k0, w);
#pragma unroll
      for (int f = 0; f < 2 * NC; f++) kf[f] = k_load(t.k, f);
#pragma unroll
      for (int d = 0; d < DT; d++) vf[d] = v_load(t.v, d);
    }
    w = look_up<WIDE>(pool, r, k0 + kStep);
    for (;;) {
      const int k1 = k0 + kStep;
      f32x4 s[2];
      scores(kf, s);
      Tile t;
      if (k1 < r.to) {
        t = tile_of<WIDE>(pool, hb, r, k1, w);
#pragma unroll
        for (int f = 0; f < 2 * NC; f++) kf[f] = k_load(t.k, f);
      }
      weigh(s, vf, k0, r.to, ok);
      if (k1 >= r.to) break;
#pragma unroll
      for (int d = 0; d < DT; d++) vf[d] = v_load(t.v, d);
      ok = found<WIDE>(pool, w);
      w = look_up<WIDE>(pool, r, k1 + kStep);
      k0 = k1;
    }
  }

  // ---- 16 rows to each of kWaves / KW waves: every wave reads every tile (KW
  // 1) or every other (KW 2), so the tiles go through a ring in LDS, in
  // fragment order, by direct loads that run kRing / KW - 1 steps ahead.  (Two
  // tiles of rows a wave, with half the reads of LDS, took 120.8 us where this
  // takes 117.4, at 64 rows over 4 * 32768 positions of 8 heads of 128 in f16,
  // and 176 where 122 in bf16, whose three parts then leave the registers.)
  static constexpr int kHalves = (int)sizeof(V) / 16;  // 16-byte loads of a fragment
  static constexpr int kShare = kLoads / kWaves;       // direct loads of a tile by one wave: K, then V
  template <bool WIDE>
  static __device__ __forceinline__ void issue(const KvPool<T> &pool, const HeadBase &hb, const Run &r, int k0,
                                        uint32_t lds, const Where &w, const uint32_t *off) {
    const Tile t = tile_of<WIDE>(pool, hb, r, k0, w);
#pragma unroll
    for (int i = 0; i < kShare; i++)
      kr_dma((i < kShare / 2 ? t.k : t.v) + off[i], lds + i * kWaves * 1024);
  }
  // the direct loads of a wave's share of a tile
  static __device__ __forceinline__ void share(const KvPool<T> &pool, uint32_t *off) {
    static_assert(kLoads % (2 * kWaves) == 0, "K and V in whole shares");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kShare; i++) {
      const int b = i * kWaves + wave, f = b / kHalves;
      off[i] = (i < kShare / 2 ? koff(pool, f) : voff(pool, f - 2 * NC)) + (b % kHalves) * 16;
    }
  }
  static __device__ __forceinline__ uint32_t ring_base(uint8_t *ring) {
    return __builtin_amdgcn_readfirstlane(lds_addr_of(ring) + (threadIdx.x >> 6) * 1024);
  }
  // the first steps' loads; returns found() of their tiles: 4 bits a tile, 8 a
  // step, the first lowest
  template <bool WIDE, int KW>
  static __device__ __forceinline__ uint32_t start_shared(const KvPool<T> &pool, const HeadBase &hb,
                                                          const Run &r, uint8_t *ring) {
    constexpr int S = kRing / KW, kAhead = S - 1, kStep = KW * kTile;
    static_assert(8 * kAhead < 32, "found() of a ring in a word");
    const int n = (r.to - r.from + kStep - 1) / kStep;
    const uint32_t base = ring_base(ring);
    uint32_t off[kShare], ok = 0;
    share(pool, off);
#pragma unroll
    for (int i = 0; i < kAhead; i++)
      if (i < n)
#pragma unroll
        for (int t = 0; t < KW; t++) {
          const int kt = r.from + i * kStep + t * kTile;
          const Where w = look_up<WIDE>(pool, r, kt);
          ok |= found<WIDE>(pool, w) << (8 * i + 4 * t);
          issue<WIDE>(pool, hb, r, kt, base + (i * KW + t) * kTileBytes, w, off);
        }
    return ok;
  }
  template <bool WIDE, int KW>
  __device__ __forceinline__ void run_shared(const KvPool<T> &pool, const HeadBase &hb, const Run &r,
                                             uint8_t *ring, uint32_t ok) {
    constexpr int S = kRing / KW, kAhead = S - 1, kStep = KW * kTile;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t base = ring_base(ring);
    const int n = (r.to - r.from + kStep - 1) / kStep;
    const int mine = KW == 1 ? 0 : wave / (kWaves / KW);  // tile of a step
    uint32_t off[kShare];
    share(pool, off);
    int get = 0, put = kAhead;  // places in the ring
    for (int i = 0; i < n; i++) {
      const int k0 = r.from + i * kStep, k2 = k0 + kAhead * kStep;
      const Where w0 = look_up<WIDE>(pool, r, k2), w1 = KW == 2 ? look_up<WIDE>(pool, r, k2 + kTile) : w0;
      // step i has landed, and every wave is done with step i - 1
      if (i + kAhead <= n)
        kr_publish<(kAhead - 1) * KW * kShare>();
      else
        kr_publish<0>();
      const int kt = k0 + mine * kTile;
      const uint32_t here = ok >> (4 * mine) & 15;
      const bool on = KW == 1 || kt < r.to;
      V kf[2 * NC], vf[DT];
      const uint8_t *f = ring + (get * KW + mine) * kTileBytes;
      auto frag = [&](int j) {
        if constexpr (sizeof(V) == 16) {
          return reinterpret_cast<const V *>(f)[j * 64 + lane];
        } else {  // two halves of 16 bytes a lane
          const f32x4 *h = reinterpret_cast<const f32x4 *>(f) + j * 128 + lane;
          return V{h[0], h[64]};
        }
      };
      if (on) {
#pragma unroll
        for (int j = 0; j < 2 * NC; j++) kf[j] = frag(j);
        // all of the tile is asked for before the first product waits (V of an
        // f32 pool after it: two workgroups a CU need the registers)
        if constexpr (!kLate)
#pragma unroll
          for (int j = 0; j < DT; j++) vf[j] = frag(2 * NC + j);
        __builtin_amdgcn_sched_barrier(0);
      }
      ok >>= 8;
      if (i + kAhead < n) {
        issue<WIDE>(pool, hb, r, k2, base + put * KW * kTileBytes, w0, off);
        if (KW == 2)
          issue<WIDE>(pool, hb, r, k2 + kTile, base + (put * KW + 1) * kTileBytes, w1, off);
        ok |= (found<WIDE>(pool, w0) | (KW == 2 ? found<WIDE>(pool, w1) << 4 : 0)) << (8 * (kAhead - 1));
      }
      if (on) {
        f32x4 s[2];
        scores(kf, s);
        if constexpr (kLate)
#pragma unroll
          for (int j = 0; j < DT; j++) vf[j] = frag(2 * NC + j);
        weigh(s, vf, kt, r.to, here);
      }
      get = get + 1 == S ? 0 : get + 1;
      put = put + 1 == S ? 0 : put + 1;
    }
  }

  // A wave's own results to the output, or to its part of the workspace.
  __device__ __forceinline__ void finish_alone(const RowArgs &a, int hd, int seq0, int head, int row0,
                                               int rows, int part) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const float sum = groups_sum(l);
    if (n >= rows) return;
    const int row = row0 + n, member = row / a.rep;
    const size_t qh = (size_t)head * a.rep + (row - member * a.rep), seq = seq0 + member;
    float *out = a.out + seq * a.ldo + qh * hd;
    const size_t at = part < 0 ? 0 : (seq * a.nh + qh) * a.parts + part;
#pragma unroll
    for (int d = 0; d < DT; d++) {
      const int c = d * 16 + g * 4;
      if (c >= hd) continue;
      if (part < 0) {
#pragma unroll
        for (int k = 0; k < 4; k++) out[c + k] = sum == 0.0f ? 0.0f : o[d][k] / sum;
      } else {
        *reinterpret_cast<f32x4 *>(a.po + at * hd + c) = o[d];
      }
    }
    if (part >= 0 && g == 0) a.pml[at * 2] = m, a.pml[at * 2 + 1] = sum;
  }

  // The results of the waves that share rows joined, in the order of the
  // waves; a row's goes to the output, or to its part of the workspace.  RW
  // tiles of rows: wave w has tile w % RW.
  __device__ __forceinline__ void finish(const RowArgs &a, int hd, int seq0, int head, int row0, int rows,
                                         int RW, int part, float *buf, float *ml) {
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4, wave = tid >> 6;
    constexpr int kCols = 8 * NC;  // of four dims
    const float sum = groups_sum(l);
    __syncthreads();
    if (g == 0) ml[(wave * 16 + n) * 2] = m, ml[(wave * 16 + n) * 2 + 1] = sum;
#pragma unroll
    for (int d = 0; d < DT; d++)
      *reinterpret_cast<f32x4 *>(buf + (wave * 16 + n) * kLd + d * 16 + g * 4) = o[d];
    __syncthreads();
    for (int i = tid; i < rows * kCols; i += 64 * kWaves) {
      const int r = i / kCols, c = i % kCols;
      if (4 * c >= hd) continue;
      float ls = 0.0f, mx = kNegInf;
      f32x4 x{0, 0, 0, 0};
      for (int w = r; w < kWaves * 16; w += RW * 16) mx = fmaxf(mx, ml[w * 2]);
      for (int w = r; w < kWaves * 16; w += RW * 16) {
        const float mw = ml[w * 2];
        // (a wave with no position has sums of 0, or of NaN if its scores were)
        const float f = mw == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mw - mx);
        const f32x4 y = *reinterpret_cast<const f32x4 *>(buf + w * kLd + 4 * c);
        ls = __builtin_fmaf(ml[w * 2 + 1], f, ls);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = __builtin_fmaf(y[k], f, x[k]);
      }
      const int row = row0 + r, member = row / a.rep;
      const size_t qh = (size_t)head * a.rep + (row - member * a.rep), seq = seq0 + member;
      if (part < 0) {
        float *out = a.out + seq * a.ldo + qh * hd + 4 * c;
#pragma unroll
        for (int k = 0; k < 4; k++) out[k] = ls == 0.0f ? 0.0f : x[k] / ls;
      } else {
        const size_t at = (seq * a.nh + qh) * a.parts + part;
        *reinterpret_cast<f32x4 *>(a.po + at * hd + 4 * c) = x;
        if (c == 0) a.pml[at * 2] = mx, a.pml[at * 2 + 1] = ls;
      }
    }
  }
};

__device__ __forceinline__ int clamped(const int32_t *len, int i, int most) {
  const auto *t = (const __attribute__((address_space(4))) int32_t *)(uintptr_t)len;  // a scalar load
  return most ? max(0, min(t[i], most)) : 0;
}

// workgroups of a CU that share its registers
template <class T, int NC, bool FULL> constexpr int kResident = NC == 8 || (NC * sizeof(T) == 16 && !FULL) ? 1 : 2;

// One workgroup a query row: its lanes hold four dims of several parts at
// once (LANES to a part), the first of them asked for before their weights
// are known; the sums are joined in a fixed order.
template <int LANES>
__device__ __forceinline__ void join_parts(const RowArgs &a, int hd, size_t row) {
  __shared__ float xs[4][4 * LANES];
  constexpr int kSub = 64 / LANES, kU = 4, kStep = 4 * kSub;  // parts of a wave, and of all four, at once
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = wave * kSub + lane / LANES, c4 = 4 * (lane % LANES);
  const int n = a.parts;
  const float *ml = a.pml + row * n * 2, *po = a.po + row * n * hd + min(c4, hd - 4);
  f32x4 x{0, 0, 0, 0}, y[kU];
  auto ask = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kU; u++)
      y[u] = *reinterpret_cast<const f32x4 *>(po + (size_t)min(i0 + u * kStep + sub, n - 1) * hd);
  };
  ask(0);
  float top = kNegInf;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, ml[2 * i]);
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  float l = 0.0f;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = min(i0 + lane, n - 1);
    const float lp = i0 + lane < n ? ml[2 * i + 1] : 0.0f;
    const float f = lp == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[2 * i] - top);
    l += lp * f;
    const int most = min(64, n - i0);
    for (int k = 0; k < most; k += kU * kStep) {
      if (i0 + k) ask(i0 + k);
#pragma unroll
      for (int u = 0; u < kU; u++) {
        const int at = k + u * kStep + sub;
        const float fu = __shfl(f, at & 63);
        // (a part with no position has left its row unwritten)
        if (at < most && fu != 0.0f)
#pragma unroll
          for (int c = 0; c < 4; c++) x[c] = __builtin_fmaf(y[u][c], fu, x[c]);
      }
    }
  }
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
#pragma unroll
  for (int o = LANES; o < 64; o *= 2)
#pragma unroll
    for (int c = 0; c < 4; c++) x[c] += __shfl_xor(x[c], o);
  if (lane < LANES) *reinterpret_cast<f32x4 *>(&xs[wave][c4]) = x;
  __syncthreads();
  if (tid < hd) {
    const size_t seq = row / a.nh, head = row - seq * a.nh;
    const float v = (xs[0][tid] + xs[1][tid]) + (xs[2][tid] + xs[3][tid]);
    a.out[seq * a.ldo + head * hd + tid] = l == 0.0f ? 0.0f : v / l;
  }
}

}  // namespace

}  // namespace syn
