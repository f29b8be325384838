// Attention of one query token per sequence over a paged cache, for groups of
// sequences that share a prefix.
#include "kv_pages.hpp"

namespace syn {

namespace {

struct AttnArgs {
  const float *q;
  const int32_t *ptable, *plen, *table, *slen;
  float *out;
  size_t ldq, ldo, ld_ptable, ld_table;
  int nh, group_size, max_prefix, max_suffix;
  float scale;
};

// One workgroup per (query head, sequence): 256 positions at a time, running
// maximum and sum.
template <class T>
__global__ void __launch_bounds__(256) k_prefix_attention(AttnArgs a, KvPool<T> pool) {
  __shared__ float qs[kKvMaxHeadDim], p[256];
  __shared__ float red[8];
  const int tid = threadIdx.x, hd = pool.hd;
  const int head = blockIdx.x, row = blockIdx.y, kvh = head / (a.nh / pool.nkv);
  const int group = row / a.group_size;
  for (int d = tid; d < hd; d += 256) qs[d] = a.q[(size_t)row * a.ldq + (size_t)head * hd + d];
  __syncthreads();
  float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
  for (int part = 0; part < 2; part++) {
    const int bound = part ? a.max_suffix : a.max_prefix;
    const int len = bound ? max(0, min(part ? a.slen[row] : a.plen[group], bound)) : 0;
    const int32_t *tab = part ? a.table + (size_t)row * a.ld_table
                              : a.ptable + (size_t)group * a.ld_ptable;
    for (int j0 = 0; j0 < len; j0 += 256) {
      const int j = j0 + tid;
      float s = -__builtin_inff();
      if (j < len) {
        const int page = tab[j >> pool.ps_shift];
        if (pool.has(page)) {
          const T *k = pool.k + pool.base(page, kvh);
          float acc = 0.0f;
          for (int d = 0; d < hd; d++)
            acc = __builtin_fmaf(qs[d], (float)k[pool.k_at(j & (pool.ps - 1), d)], acc);
          s = acc * a.scale;
        }
      }
      float mx = s;
      for (int w = 32; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
      if ((tid & 63) == 0) red[tid >> 6] = mx;
      __syncthreads();
      mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      const float m2 = fmaxf(m, mx);
      const float c = m2 == -__builtin_inff() ? 1.0f : expf(m - m2);
      const float e = m2 == -__builtin_inff() ? 0.0f : expf(s - m2);
      m = m2;
      p[tid] = e;
      float sum = e;
      for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
      if ((tid & 63) == 0) red[4 + (tid >> 6)] = sum;
      __syncthreads();
      l = l * c + (red[4] + red[5] + red[6] + red[7]);
      o *= c;
      if (tid < hd)
        for (int i = 0; i < min(256, len - j0); i++) {
          const int page = tab[(j0 + i) >> pool.ps_shift];
          if (pool.has(page))
            o = __builtin_fmaf(p[i], (float)pool.v[pool.base(page, kvh) +
                                                   pool.v_at((j0 + i) & (pool.ps - 1), tid)], o);
        }
      __syncthreads();
    }
  }
  if (tid < hd) a.out[(size_t)row * a.ldo + (size_t)head * hd + tid] = l == 0.0f ? 0.0f : o / l;
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

}  // namespace

}  // namespace syn

using namespace syn;

extern "C" syn_status_t syn_hip_prefix_attention_workspace(
    const syn_hip_kv_pages *pages, const syn_hip_prefix_attention_params *p, size_t *bytes) {
  if (!bytes) return SYN_ERR_NULL_PTR;
  SYN_TRY(check_attention(pages, p));
  *bytes = 0;
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
  SYN_TRY(ensure_init());
  AttnArgs a{d_q,    d_prefix_table, d_prefix_len,    d_table,     d_len,
             d_out,  p->ldq,         p->ldo,          p->ld_prefix_table, p->ld_table,
             (int)p->n_heads, (int)p->group_size, (int)p->max_prefix, (int)p->max_suffix,
             p->scale != 0.0f ? p->scale : 1.0f / sqrtf((float)pages->head_dim)};
  return kv_dispatch(pages->dtype, [&](auto t) -> syn_status_t {
    using T = decltype(t);
    hipLaunchKernelGGL(k_prefix_attention<T>, dim3(p->n_heads, (unsigned)rows), dim3(256), 0,
                       pick_stream(stream), a, kv_pool<T>(*pages, p->layer));
    SYN_LAUNCH_CHECK();
    return SYN_OK;
  });
}
