// Keys and values into a paged cache, with head norms and position rotation on
// the way: y = x * gain / sqrt(mean x^2 + eps) per head, then each pair (a, b)
// of the first rotary_dim dims turned by its position's angle, f32 throughout,
// rounded once (to nearest even) where a 16-bit pool stores it.
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
};

template <class T>
__global__ void __launch_bounds__(kThreads) k_kv_append(AppendArgs a, KvPool<T> pool) {
  extern __shared__ float xs[];  // [kTok][hd + 4]
  __shared__ float inv[kTok];
  __shared__ int row_pos[kTok], row_page[kTok], row_slot[kTok], whole[kTok];
  const int tid = threadIdx.x, hd = pool.hd, ldx = hd + 4;
  const int t0 = blockIdx.x * kTok, head = blockIdx.y;
  const int nt = min(kTok, a.n_tokens - t0);
  const bool is_q = head < a.nh, is_k = !is_q && head < a.nh + pool.nkv;
  const int h = is_q ? head : (is_k ? head - a.nh : head - a.nh - pool.nkv);
  const float *src = is_q ? a.q : (is_k ? a.k : a.v);
  const size_t lds = is_q ? a.ldq : (is_k ? a.ldk : a.ldv);

  if (tid < kTok) {
    int pos = -1, page = -1, slot = 0;
    if (tid < nt) {
      const int t = t0 + tid;
      pos = a.pos[t];
      if ((uint32_t)pos >= (uint32_t)a.n_pos) pos = -1;
      const int seq = a.seq ? a.seq[t] : t, i = a.index[t];
      const int col = i >> pool.ps_shift;
      if (pos >= 0 && i >= 0 && (size_t)col < a.ld_table && (uint32_t)seq < (uint32_t)a.n_seqs) {
        page = a.table[(size_t)seq * a.ld_table + col];
        if (!pool.has(page)) page = -1;
        slot = i & (pool.ps - 1);
      }
    }
    row_pos[tid] = pos;
    row_page[tid] = page;
    row_slot[tid] = slot;
  }
  for (int i = tid; i < nt * hd; i += kThreads) {
    const int t = i / hd, d = i - t * hd;
    xs[t * ldx + d] = src[(size_t)(t0 + t) * lds + (size_t)h * hd + d];
  }
  __syncthreads();

  const float *gain = is_q ? a.qn : (is_k ? a.kn : nullptr);
  if (gain) {
    // 16 threads a token
    const int t = tid >> 4, l = tid & 15;
    float s = 0.0f;
    if (t < nt)
      for (int d = l; d < hd; d += 16) s = __builtin_fmaf(xs[t * ldx + d], xs[t * ldx + d], s);
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (l == 0) inv[t] = 1.0f / sqrtf(s / (float)hd + a.eps);
    __syncthreads();
    for (int i = tid; i < nt * hd; i += kThreads) {
      const int tt = i / hd, d = i - tt * hd;
      xs[tt * ldx + d] = xs[tt * ldx + d] * gain[d] * inv[tt];
    }
    __syncthreads();
  }

  const int half = a.rd >> 1;
  auto turned = [&](int t, int d) {
    const float x = xs[t * ldx + d];
    if (d >= a.rd) return x;
    const bool lo = a.interleaved ? !(d & 1) : d < half;
    const int i = a.interleaved ? d >> 1 : (lo ? d : d - half);
    const float y = xs[t * ldx + (a.interleaved ? d ^ 1 : (lo ? d + half : d - half))];
    const size_t at = (size_t)row_pos[t] * half + i;
    const float c = a.cs[at], s = a.sn[at];
    return __builtin_fmaf(x, c, lo ? -(y * s) : y * s);
  };

  if (is_q) {
    for (int i = tid; i < nt * hd; i += kThreads) {
      const int t = i / hd, d = i - t * hd;
      if (row_pos[t] >= 0) a.qo[(size_t)(t0 + t) * a.ldo + (size_t)h * hd + d] = turned(t, d);
    }
  } else if (is_k) {
    const int n8 = hd >> 3;  // consecutive threads write consecutive positions
    for (int i = tid; i < nt * n8; i += kThreads) {
      const int t = i % nt, c = i / nt;
      if (row_page[t] < 0) continue;
      T *dst = pool.k + pool.base(row_page[t], h) + pool.k_at(row_slot[t], c * 8);
      for (int j = 0; j < 8; j++) dst[j] = (T)turned(t, c * 8 + j);
    }
  } else {
    // 8 tokens that fill an aligned group of 8 positions are written together
    if (tid < kTok) {
      bool w = tid + 8 <= nt && row_page[tid] >= 0 && (row_slot[tid] & 7) == 0;
      for (int j = 1; w && j < 8; j++)
        w = row_page[tid + j] == row_page[tid] && row_slot[tid + j] == row_slot[tid] + j;
      whole[tid] = w;
    }
    __syncthreads();
    for (int i = tid; i < nt * hd; i += kThreads) {
      const int t = i / hd, d = i - t * hd;
      if (row_page[t] < 0) continue;
      T *dst = pool.v + pool.base(row_page[t], h) + pool.v_at(row_slot[t], d);
      const int lead = t - (row_slot[t] & 7);
      if (whole[t]) {
        for (int j = 0; j < 8; j++) dst[j] = (T)xs[(t + j) * ldx + d];
      } else if (lead < 0 || !whole[lead]) {
        *dst = (T)xs[t * ldx + d];
      }
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
  if (n_tokens > 0x7fffffffu || p->n_seqs > 0x7fffffffu || p->n_positions > 0x7fffffffu ||
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
  SYN_TRY(ensure_init());
  const AppendArgs a{d_q,      d_k,    d_v,    d_q_norm, d_k_norm, d_cos,       d_sin,
                     d_pos,    d_seq,  d_index, d_table, d_q_out,  p->ldq,      p->ldk,
                     p->ldv,   p->ldo, p->ld_table, (int)n_tokens, (int)nh, (int)p->n_seqs,
                     (int)p->rotary_dim, p->interleaved, (int)p->n_positions, p->eps};
  const dim3 grid((unsigned)cdiv(n_tokens, kTok), (unsigned)(nh + 2 * nkv));
  const size_t shm = kTok * (hd + 4) * sizeof(float);
  return kv_dispatch(pages->dtype, [&](auto t) -> syn_status_t {
    using T = decltype(t);
    hipLaunchKernelGGL(k_kv_append<T>, grid, dim3(kThreads), shm, pick_stream(stream), a,
                       kv_pool<T>(*pages, p->layer));
    SYN_LAUNCH_CHECK();
    return SYN_OK;
  });
}
