// Paged key/value pools (syn_hip_kv_pages): layout, argument checks and the
// operators' launches, shared by the C entry points and the decoders.
#pragma once

#include "common.hpp"

namespace syn {

// A page holds page_size positions of one layer, every kv head:
//   K: [kv head][hd / 8][page_size][8]   - 8 dims of a position are one 16-byte
//      (16-bit types) load, and 16 positions at the same dims are contiguous:
//      the A operand of v_mfma_f32_16x16x32 straight from memory;
//   V: [kv head][page_size / 8][hd][8]   - 8 positions of a dim are one load,
//      16 dims contiguous: V transposed, the A operand of the second product.
// Both products then read global memory in whole 256-byte runs and need no
// transposition through LDS.
template <class T> struct KvPool {
  T *k, *v;            // of the layer
  uint32_t n_pages;
  int nkv, hd, ps, ps_shift;
  __device__ __forceinline__ bool has(int page) const { return (uint32_t)page < n_pages; }
  // element offset of (page, head)
  __device__ __forceinline__ size_t base(int page, int head) const {
    return ((size_t)page * nkv + head) * ((size_t)hd * ps);
  }
  __device__ __forceinline__ size_t k_at(int slot, int d) const {
    return ((size_t)(d >> 3) * ps + slot) * 8 + (d & 7);
  }
  __device__ __forceinline__ size_t v_at(int slot, int d) const {
    return ((size_t)(slot >> 3) * hd + d) * 8 + (slot & 7);
  }
};

constexpr uint32_t kKvMaxHeadDim = 256;
constexpr uint32_t kKvMaxPage = 1024;
constexpr size_t kMaxThreads = 0xffffffffu;  // of a launch, in one dimension
constexpr uint32_t kMaxBeams = 64;
constexpr uint32_t kMaxSelect = 128;

// SYN_OK when the pool's description is one that the kernels take
syn_status_t check_pages(const syn_hip_kv_pages *p, const char *who);

inline size_t kv_elem_bytes(int32_t dtype) { return dtype == SYN_HIP_KV_F32 ? 4 : 2; }
inline size_t kv_page_elems(const syn_hip_kv_pages &p) {
  return (size_t)p.n_kv_heads * p.page_size * p.head_dim;
}
// K or V bytes of the whole pool
inline size_t kv_pool_bytes(const syn_hip_kv_pages &p) {
  return kv_elem_bytes(p.dtype) * p.n_layers * p.n_pages * kv_page_elems(p);
}

template <class T> KvPool<T> kv_pool(const syn_hip_kv_pages &p, uint32_t layer) {
  const size_t off = (size_t)layer * p.n_pages * kv_page_elems(p);
  return KvPool<T>{static_cast<T *>(p.k) + off, static_cast<T *>(p.v) + off, p.n_pages,
                   (int)p.n_kv_heads, (int)p.head_dim, (int)p.page_size,
                   31 - __builtin_clz(p.page_size)};
}

// fn(T{}) for the pool's element type
template <class F> syn_status_t kv_dispatch(int32_t dtype, F fn) {
  switch (dtype) {
    case SYN_HIP_KV_F32: return fn(float{});
    case SYN_HIP_KV_F16: return fn(_Float16{});
    default: return fn(__bf16{});
  }
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace syn
