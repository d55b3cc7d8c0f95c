// Shared by the operators over a paged KV cache (paged.cu, paged_attn.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/myos_cuda.h"

namespace myos {

// myos_paged_kv as the kernels take it.
template <class KT>
struct PagedKv {
  KT* k;
  KT* v;
  int64_t page_stride, head_stride, slot_stride;  // elements
  uint32_t num_pages, page_size, heads, d;
};

template <class KT>
inline PagedKv<KT> paged_view(const myos_paged_kv* kv) {
  PagedKv<KT> p;
  p.k = static_cast<KT*>(kv->k);
  p.v = static_cast<KT*>(kv->v);
  p.page_stride = (int64_t)kv->page_stride;
  p.head_stride = (int64_t)kv->head_stride;
  p.slot_stride = (int64_t)kv->slot_stride;
  p.num_pages = kv->num_pages;
  p.page_size = kv->page_size;
  p.heads = kv->num_kv_heads;
  p.d = kv->head_dim;
  return p;
}

// The header's rules for a cache; MYOS_OK or the status to return.
int paged_check(const myos_paged_kv* kv);

inline bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace myos
