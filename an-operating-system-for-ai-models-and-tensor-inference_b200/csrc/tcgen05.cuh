// The fifth-generation tensor cores' instructions, and the tensor copies that feed
// them: thin wrappers of the PTX.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace myos {

// Brings a map (a kernel's parameter) to the copy engine.
MYOS_DEV void tma_ahead(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
MYOS_DEV void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// The same for one block of a pair: bar (a cluster address) may be the other's.
MYOS_DEV void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// One lane of a whole warp, the same each time.
MYOS_DEV bool one_lane() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

// Tensor memory: `columns` (a power of two, 32 .. 512) of 128 lanes x 32 bits, its
// address into *dst (shared memory). One whole warp each.
template <bool PAIR>
MYOS_DEV void tmem_alloc(uint32_t* dst, uint32_t columns) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <bool PAIR>
MYOS_DEV void tmem_free(uint32_t base, uint32_t columns) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}

MYOS_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
MYOS_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// An operand in shared memory: rows of 128 bytes along k in the copy engine's
// 128-byte swizzle, groups of 8 rows 1024 bytes apart, the first at a multiple of
// 1024. 32 bytes further along k: + 2. Of a pair: at the same place in both blocks.
MYOS_DEV uint64_t tc_operand(const void* p) {
  constexpr uint64_t kForm = (uint64_t)1 << 16 | (uint64_t)(1024 / 16) << 32 | (uint64_t)1 << 46 |
                             (uint64_t)2 << 61;
  return kForm | (smem_u32(p) >> 4);
}

// D[m, n] 32-bit integers = (accumulate ? D : 0) + A[m, 32] B[n, 32], signed bytes.
MYOS_DEV constexpr uint32_t tc_i8_shape(uint32_t m, uint32_t n) {
  return 2u << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | (m >> 4) << 24;
}
// PAIR: each block of the pair holds half of A's rows, half of B's, and half of D's;
// one of the two issues.
template <bool PAIR>
MYOS_DEV void tc_mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"((uint32_t)accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"((uint32_t)accumulate)
        : "memory");
}
// An arrival at bar (of a pair: in both blocks) once the products issued so far are
// done.
template <bool PAIR>
MYOS_DEV void tc_commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
            smem_u32(bar))
        : "memory");
}

// 16 columns of this warp's 32 lanes (lane 32 * (warp % 4) of the address).
MYOS_DEV void tmem_load16(uint32_t at, int* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(at));
}
MYOS_DEV void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

MYOS_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// All threads of the cluster meet; in two parts, with work between them.
MYOS_DEV void cluster_enter() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
MYOS_DEV void cluster_leave() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
MYOS_DEV void cluster_meet() {
  cluster_enter();
  cluster_leave();
}
// The same without an order of memory.
MYOS_DEV void cluster_end() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  cluster_leave();
}
// The address in block `rank` of the cluster of what lies at p in this one.
MYOS_DEV uint32_t cluster_at(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
MYOS_DEV void cluster_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
MYOS_DEV void cluster_store(uint32_t at, int v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

}  // namespace myos
