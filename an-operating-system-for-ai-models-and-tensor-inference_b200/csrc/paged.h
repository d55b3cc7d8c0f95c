// Shared by the operators over a paged KV cache (paged.cu, paged_attn.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

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

// Raises a kernel's dynamic shared-memory limit, once per device; `done` is the
// kernel's own mask of devices.
inline cudaError_t raise_smem_limit(const void* kernel, size_t bytes, std::atomic<uint64_t>* done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (bit && (done->load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_release);
  else cudaGetLastError();
  return e;
}

// Launches with a programmatic edge to the previous kernel of the stream: the
// blocks are placed while its last ones run, and wait for its end and its
// memory (pdl_wait) before their first global access. cluster: blocks of one
// thread-block cluster.
template <class... P, class... A>
inline cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, size_t smem,
                              cudaStream_t st, int cluster, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) cudaGetLastError();  // reported here, not by a later call
  return e;
}

// Multiprocessors of the current device (148 where it cannot be asked).
int sm_count();

inline bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace myos
