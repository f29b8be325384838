// Keys and values into a paged cache, with head norms and position rotation on
// the way: y = x * gain / sqrt(mean x^2 + eps) per head, then each pair (a, b)
// of the first rotary_dim dims turned by its position's angle, f32 throughout,
// rounded once (to nearest even) where a 16-bit pool stores it.
#include <algorithm>

#include "kv_pages.hpp"

namespace syn {

namespace {

constexpr int kTok = 16;  // tokens of a workgroup: V needs 8 in a row for a whole write
constexpr int kThreads = 256;

struct AppendArgs {
  const float *q, *k, *v, *qn, *kn, *cs, *sn;
  const int32_t *pos, *seq, *index, *table;
  float *qo;
  size_t ldq, ldk, ldv, ldo, ld_table;
  int n_tokens, nh, n_seqs, rd, interleaved, n_pos;
  float eps;
  bool vec_in, vec_out, vec_rot, vec_gain;  // 16-byte rows of q, k, v; of q_out; of the tables (half of rd too); gains
};

// four consecutive floats
__device__ __forceinline__ f32x4 load4(const float *p, bool vec) {
  if (vec) return *reinterpret_cast<const f32x4 *>(p);
  return f32x4{p[0], p[1], p[2], p[3]};
}
// sum over the 16 lanes of a token
__device__ __forceinline__ float row_sum(float x) {
  auto add = [&](int y) { x += __int_as_float(y); };
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xb1, 0xf, 0xf, false));   // lane ^ 1
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4e, 0xf, 0xf, false));   // lane ^ 2
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, false));  // 7 - lane
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xf, 0xf, false));  // 15 - lane
  return x;
}

// A workgroup takes 16 tokens and every gridDim.y-th head (queries, keys, then
// values): 16 threads a token, each four dims of every 64.  A thread's angles
// are the same for all heads and stay in registers; the other half of a pair
// comes from the token's row in LDS, which only its own wave writes.  The next
// head is requested before this one is worked on.  Bound by its bytes, read
// once and written once: 8192 tokens of 32 + 2 * 8 heads of 128 into f16 pages
// 89 us, 4.1 TB/s (a large copy reaches 4.8); 517 tokens of 16 + 2 * 8 heads into
// bf16 8.5 us, three dependent loads (place, page, angles) and one round of heads; 8
// tokens 4.7, a launch.  KD: 64 dims each (hd <= 64 KD).
template <class T, int KD>
__global__ void __launch_bounds__(kThreads) k_kv_append(AppendArgs a, KvPool<T> pool) {
  __shared__ __align__(16) float xs[kTok][64 * KD + 4];
  __shared__ int row_page[kTok], row_slot[kTok], whole[kTok];
  const int tid = threadIdx.x, hd = pool.hd, t = tid >> 4, l = tid & 15;
  const int t0 = blockIdx.x * kTok, nt = min(kTok, a.n_tokens - t0);
  const int heads = a.nh + 2 * pool.nkv;
  const size_t tok = t0 + min(t, nt - 1);  // (threads past the last repeat it and write nothing)

  auto row_of = [&](int head) {
    const bool is_q = head < a.nh, is_k = !is_q && head < a.nh + pool.nkv;
    const float *src = is_q ? a.q : (is_k ? a.k : a.v);
    const size_t ld = is_q ? a.ldq : (is_k ? a.ldk : a.ldv);
    const int h = is_q ? head : (is_k ? head - a.nh : head - a.nh - pool.nkv);
    return src + tok * ld + (size_t)h * hd;
  };
  f32x4 next[KD];
  auto ask = [&](int head) {
    const float *src = row_of(head);
#pragma unroll
    for (int k = 0; k < KD; k++) next[k] = load4(src + min(64 * k + 4 * l, hd - 4), a.vec_in);
  };
  ask(blockIdx.y);

  // the token's place, and its angles
  int pos = a.pos[tok], page = -1, slot = 0;
  {
    const int seq = a.seq ? a.seq[tok] : (int)tok, i = a.index[tok];
    const bool known = (uint32_t)pos < (uint32_t)a.n_pos;
    if (!known || t >= nt) pos = -1;
    const int col = i >> pool.ps_shift;
    if (pos >= 0 && i >= 0 && (size_t)col < a.ld_table && (uint32_t)seq < (uint32_t)a.n_seqs) {
      page = a.table[(size_t)seq * a.ld_table + col];
      if (!pool.has(page)) page = -1;
      slot = i & (pool.ps - 1);
    }
    if (l == 0) row_page[t] = page, row_slot[t] = slot;
  }
  const int half = a.rd >> 1;
  f32x4 c[KD], s[KD];  // of the thread's dims; s negative where the pair's first half is
  const size_t at = (size_t)max(pos, 0) * half;
#pragma unroll
  for (int k = 0; k < KD; k++) {
    c[k] = f32x4{1, 1, 1, 1};
    s[k] = f32x4{0, 0, 0, 0};
    const int d0 = 64 * k + 4 * l;
    if (d0 >= a.rd) continue;
    if (a.vec_rot && !a.interleaved) {
      const int i = d0 < half ? d0 : d0 - half;
      c[k] = load4(a.cs + at + i, true);
      s[k] = load4(a.sn + at + i, true);
      if (d0 < half) s[k] = -s[k];
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int d = d0 + j;
        if (d >= a.rd) break;
        const bool lo = a.interleaved ? !(d & 1) : d < half;
        const int i = a.interleaved ? d >> 1 : (lo ? d : d - half);
        c[k][j] = a.cs[at + i];
        s[k][j] = lo ? -a.sn[at + i] : a.sn[at + i];
      }
    }
  }
  // 8 tokens that fill an aligned group of 8 positions are written together
  const int last = blockIdx.y + (heads - 1 - (int)blockIdx.y) / (int)gridDim.y * (int)gridDim.y;
  const bool has_v = last >= a.nh + pool.nkv;
  if (has_v) __syncthreads();
  if (has_v && tid < kTok) {
    bool w = tid + 8 <= nt && row_page[tid] >= 0 && (row_slot[tid] & 7) == 0;
    for (int j = 1; w && j < 8; j++)
      w = row_page[tid + j] == row_page[tid] && row_slot[tid + j] == row_slot[tid] + j;
    whole[tid] = w;
  }
  if (has_v) __syncthreads();

  for (int head = blockIdx.y; head < heads; head += gridDim.y) {
    const bool is_q = head < a.nh, is_k = !is_q && head < a.nh + pool.nkv;
    f32x4 x[KD];
#pragma unroll
    for (int k = 0; k < KD; k++) x[k] = next[k];
    if (head + (int)gridDim.y < heads) ask(head + gridDim.y);
    if (is_q || is_k) {
      const float *gain = is_q ? a.qn : a.kn;
      if (gain) {
        f32x4 w[KD];
#pragma unroll
        for (int k = 0; k < KD; k++) w[k] = load4(gain + min(64 * k + 4 * l, hd - 4), a.vec_gain);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < KD; k++)
          if (64 * k + 4 * l < hd)
#pragma unroll
            for (int j = 0; j < 4; j++) sum = __builtin_fmaf(x[k][j], x[k][j], sum);
        const float inv = 1.0f / sqrtf(row_sum(sum) / (float)hd + a.eps);
#pragma unroll
        for (int k = 0; k < KD; k++)
#pragma unroll
          for (int j = 0; j < 4; j++) x[k][j] = x[k][j] * w[k][j] * inv;
      }
      if (a.rd) {
        f32x4 y[KD];  // the pairs' other halves
        if (a.interleaved) {
#pragma unroll
          for (int k = 0; k < KD; k++) y[k] = f32x4{x[k][1], x[k][0], x[k][3], x[k][2]};
        } else {
#pragma unroll
          for (int k = 0; k < KD; k++) *reinterpret_cast<f32x4 *>(&xs[t][64 * k + 4 * l]) = x[k];
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int k = 0; k < KD; k++) {
            const int d0 = 64 * k + 4 * l;
            if (a.vec_rot) {
              const int d = d0 < half ? d0 + half : d0 - half;
              y[k] = *reinterpret_cast<const f32x4 *>(&xs[t][d0 < a.rd ? d : 0]);
            } else {
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const int d = d0 + j < half ? d0 + j + half : d0 + j - half;
                y[k][j] = xs[t][d0 + j < a.rd ? d : 0];
              }
            }
          }
          __builtin_amdgcn_wave_barrier();  // (the next head's rows are written behind these reads)
        }
#pragma unroll
        for (int k = 0; k < KD; k++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (64 * k + 4 * l + j < a.rd) x[k][j] = __builtin_fmaf(x[k][j], c[k][j], y[k][j] * s[k][j]);
      }
      if (is_q) {
        float *dst = a.qo + tok * a.ldo + (size_t)head * hd;
        if (pos >= 0)
#pragma unroll
          for (int k = 0; k < KD; k++) {
            const int d = 64 * k + 4 * l;
            if (d >= hd) continue;
            if (a.vec_out)
              *reinterpret_cast<f32x4 *>(dst + d) = x[k];
            else
#pragma unroll
              for (int j = 0; j < 4; j++) dst[d + j] = x[k][j];
          }
      } else if (page >= 0) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        T *dst = pool.k + pool.base(page, head - a.nh);
#pragma unroll
        for (int k = 0; k < KD; k++) {
          const int d = 64 * k + 4 * l;
          if (d >= hd) continue;
          t4 v;
#pragma unroll
          for (int j = 0; j < 4; j++) v[j] = (T)x[k][j];
          *reinterpret_cast<t4 *>(dst + pool.k_at(slot, d)) = v;
        }
      }
    } else {
      // V: positions of a dim are next to each other, so the tokens change
      // places through LDS
#pragma unroll
      for (int k = 0; k < KD; k++) *reinterpret_cast<f32x4 *>(&xs[t][64 * k + 4 * l]) = x[k];
      __syncthreads();
      const int h = head - a.nh - pool.nkv;
      typedef T t8 __attribute__((ext_vector_type(8)));
      for (int d = tid & (64 * KD - 1); d < hd; d += 64 * KD)
        for (int r = tid / (64 * KD); r < kTok; r += kThreads / (64 * KD)) {
          if (row_page[r] < 0) continue;
          T *dst = pool.v + pool.base(row_page[r], h) + pool.v_at(row_slot[r], d);
          const int lead = r - (row_slot[r] & 7);
          if (whole[r]) {
            t8 v;
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (T)xs[r + j][d];
            *reinterpret_cast<t8 *>(dst) = v;
          } else if (lead < 0 || !whole[lead]) {
            *dst = (T)xs[r][d];
          }
        }
      __syncthreads();
    }
  }
}

}  // namespace

syn_status_t check_pages(const syn_hip_kv_pages *p, const char *who) {
  if (!p) return SYN_ERR_NULL_PTR;
  if (p->dtype != SYN_HIP_KV_F32 && p->dtype != SYN_HIP_KV_F16 && p->dtype != SYN_HIP_KV_BF16) {
    set_error(std::string(who) + ": unknown page dtype");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->page_size < 8 || p->page_size > kKvMaxPage || (p->page_size & (p->page_size - 1))) {
    set_error(std::string(who) + ": page_size must be a power of two from 8 to 1024");
    return SYN_ERR_INVALID_ARG;
  }
  if (p->head_dim == 0 || p->head_dim % 8 || p->head_dim > kKvMaxHeadDim) {
    set_error(std::string(who) + ": head_dim must be a multiple of 8 up to 256");
    return SYN_ERR_INVALID_ARG;
  }
  if (!p->n_kv_heads || !p->n_pages || !p->n_layers || p->n_pages > 0x7fffffffu ||
      p->n_kv_heads > 65535u) {
    set_error(std::string(who) + ": pages, layers and kv heads must be at least 1");
    return SYN_ERR_INVALID_ARG;
  }
  // (kernels step through a page's bytes in 32 bits; from page to page in 64)
  if (kv_page_elems(*p) * kv_elem_bytes(p->dtype) > 0x7fffffffu) {
    set_error(std::string(who) + ": pages of at most 2^31 - 1 bytes");
    return SYN_ERR_INVALID_ARG;
  }
  if (!p->k || !p->v) return SYN_ERR_NULL_PTR;
  if (!aligned16(p->k) || !aligned16(p->v)) {
    set_error(std::string(who) + ": page pools must be 16-byte aligned");
    return SYN_ERR_INVALID_ARG;
  }
  return SYN_OK;
}

}  // namespace syn

using namespace syn;

extern "C" syn_status_t syn_hip_kv_append(
    const syn_hip_kv_pages *pages, const syn_hip_kv_append_params *p, size_t n_tokens,
    const float *d_q, const float *d_k, const float *d_v, const float *d_q_norm,
    const float *d_k_norm, const float *d_cos, const float *d_sin, const int32_t *d_pos,
    const int32_t *d_seq, const int32_t *d_index, const int32_t *d_table, float *d_q_out,
    void *stream) {
  if (!p) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_pages(pages, "kv_append"));
  const size_t hd = pages->head_dim, nh = p->n_heads, nkv = pages->n_kv_heads;
  if (p->layer >= pages->n_layers || p->rotary_dim > hd || p->rotary_dim % 2) {
    set_error("kv_append: layer outside the pool, or rotary_dim not even and at most head_dim");
    return SYN_ERR_INVALID_ARG;
  }
  if (cdiv(n_tokens, kTok) > kMaxThreads / kThreads || p->n_seqs > 0x7fffffffu || p->n_positions > 0x7fffffffu ||
      nh + 2 * nkv > 65535u) {
    set_error("kv_append: too many tokens, sequences, positions or heads");
    return SYN_ERR_INVALID_ARG;
  }
  if ((nh && (p->ldq < nh * hd || p->ldo < nh * hd)) || p->ldk < nkv * hd || p->ldv < nkv * hd) {
    set_error("kv_append: row strides shorter than the heads");
    return SYN_ERR_SHAPE_MISMATCH;
  }
  if (n_tokens == 0) return SYN_OK;
  if (!d_k || !d_v || !d_pos || !d_index || !d_table || (nh && (!d_q || !d_q_out)) ||
      (p->rotary_dim && (!d_cos || !d_sin)))
    return SYN_ERR_NULL_PTR;
  if (nh && d_q_out == d_q && p->ldo != p->ldq) {
    set_error("kv_append: d_q_out may be d_q with ldo == ldq only");
    return SYN_ERR_INVALID_ARG;
  }
  // (every token is skipped: the tables have no row that a kernel may read)
  if (p->n_positions == 0) return SYN_OK;
  SYN_TRY(ensure_init());
  AppendArgs a{d_q,      d_k,    d_v,    d_q_norm, d_k_norm, d_cos,       d_sin,
               d_pos,    d_seq,  d_index, d_table, d_q_out,  p->ldq,      p->ldk,
               p->ldv,   p->ldo, p->ld_table, (int)n_tokens, (int)nh, (int)p->n_seqs,
               (int)p->rotary_dim, p->interleaved, (int)p->n_positions, p->eps};
  a.vec_in = aligned16(d_k) && aligned16(d_v) && p->ldk % 4 == 0 && p->ldv % 4 == 0 &&
             (!nh || (aligned16(d_q) && p->ldq % 4 == 0));
  a.vec_out = aligned16(d_q_out) && p->ldo % 4 == 0;
  a.vec_rot = aligned16(d_cos) && aligned16(d_sin) && p->rotary_dim % 8 == 0;
  a.vec_gain = aligned16(d_q_norm) && aligned16(d_k_norm);
  // Workgroups enough to fill the chip, then heads in turn, whose angles are
  // there already (8192 tokens of 48 heads: 89 us with 1024 workgroups, 87 with
  // 2048, 103 with 512, 98 with 4096; 517 of 32: 8.6, 8.7, 9.2, 8.7).
  const size_t tiles = cdiv(n_tokens, kTok), heads = nh + 2 * nkv;
  const dim3 grid((unsigned)tiles, (unsigned)std::min(heads, std::max<size_t>(1, cdiv(1024, tiles))));
  return kv_dispatch(pages->dtype, [&](auto t) -> syn_status_t {
    using T = decltype(t);
    const KvPool<T> pool = kv_pool<T>(*pages, p->layer);
    hipStream_t s = pick_stream(stream);
    if (hd <= 64)
      hipLaunchKernelGGL((k_kv_append<T, 1>), grid, dim3(kThreads), 0, s, a, pool);
    else if (hd <= 128)
      hipLaunchKernelGGL((k_kv_append<T, 2>), grid, dim3(kThreads), 0, s, a, pool);
    else
      hipLaunchKernelGGL((k_kv_append<T, 4>), grid, dim3(kThreads), 0, s, a, pool);
    SYN_LAUNCH_CHECK();
    return SYN_OK;
  });
}
