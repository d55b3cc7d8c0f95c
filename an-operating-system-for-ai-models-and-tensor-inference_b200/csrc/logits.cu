// Logits under the requests' controls (penalties for repeated tokens, biases,
// grammar masks) and the greedy id.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace myos {
namespace {

struct LogitArgs {
  float* out;
  const float* logits;
  int64_t out_stride, logits_stride;
  int vocab;
  int slice, chunk;  // ids of a block, and of a pass over its tables: multiples of 4
  uint32_t* ids;
  myos_logit_controls_args c;
};

// A row is shared by a cluster of blocks, a slice of the vocabulary each. A
// slice goes by in chunks whose history and biases are first sorted into tables
// in shared memory, one word an id, by integer atomics (the result does not
// depend on their order); a chunk's logits are loaded before that, kGroups
// 16-byte groups a thread, so the tables are built while they come. The blocks'
// best ids meet in the first block's shared memory.
constexpr int kThreads = 512, kGroups = 4, kMaxChunk = kThreads * kGroups * 4;
constexpr int kMaxCluster = 8;
constexpr uint32_t kSeen = 0x80000000u;  // in the prompt; the low bits count the output

// x under the penalties: each step rounded, as a chain of elementwise passes
// would round it.
MYOS_DEV float penalised(float x, uint32_t said, float rep, float freq, float pres, bool has_rep) {
  if (has_rep) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
  const uint32_t times = said & ~kSeen;
  x = __fsub_rn(x, __fmul_rn(freq, (float)times));
  return times ? __fsub_rn(x, pres) : x;
}

// The first maximum: the larger value, on a tie the lower id.
MYOS_DEV void better(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) {
    v = ov;
    i = oi;
  }
}

__global__ void __launch_bounds__(kThreads, 2) k_logit_controls(const LogitArgs a) {
  extern __shared__ __align__(16) uint32_t tables[];
  __shared__ float best_v[32];
  __shared__ int best_i[32];
  __shared__ unsigned long long found[kMaxCluster];
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  if (a.ids && ranks > 1)  // the first block's memory is written to below: it has to have started
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int64_t row = blockIdx.x / ranks;
  const myos_logit_controls_args& c = a.c;
  const float* x = a.logits + row * a.logits_stride;
  float* y = a.out ? a.out + row * a.out_stride : nullptr;
  // Ids count from `shift` on, so that groups of four lie on 16 bytes of x.
  const int shift = (int)((uintptr_t)x >> 2 & 3);
  const bool together = y && (((uintptr_t)x ^ (uintptr_t)y) & 15) == 0;
  const bool in_place = y == x;

  const bool pen = c.history && (c.repetition || c.frequency || c.presence);
  int hist = 0, prompt = 0;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (pen) {
    hist = (int)c.history_width;
    if (c.history_lens) hist = min(hist, max(c.history_lens[row], 0));
    if (c.prompt_lens) prompt = c.prompt_lens[row];
    if (c.repetition) rep = c.repetition[row];
    if (c.frequency) freq = c.frequency[row];
    if (c.presence) pres = c.presence[row];
  }
  const int32_t* said_ids = pen ? c.history + row * (int64_t)c.history_stride : nullptr;
  int e0 = 0, e1 = 0;
  if (c.bias_starts) {
    e0 = min(max(c.bias_starts[row], 0), (int)c.num_bias);
    e1 = min(max(c.bias_starts[row + 1], 0), (int)c.num_bias);
  }
  const bool has_bias = e1 > e0;
  const uint32_t* mask = nullptr;
  if (c.mask) {
    const int64_t g = c.mask_rows ? c.mask_rows[row] : row;
    if (g >= 0 && g < (int64_t)c.num_masks) mask = c.mask + g * (int64_t)c.mask_stride;
  }
  uint32_t* said = tables;
  uint32_t* bias = tables + (pen ? a.chunk : 0);

  float bv = -INFINITY;
  int bi = 0;
  const int s0 = rank * a.slice, s1 = min(s0 + a.slice, a.vocab + shift);
#pragma unroll 1
  for (int base = s0; base < s1; base += a.chunk) {
    const int n = min(a.chunk, s1 - base);  // shifted ids base .. base + n
    const uint32_t first = (uint32_t)(base - shift);
    float4 v[kGroups];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int at = 4 * (tid + k * kThreads), i = base + at - shift;  // ids i .. i + 3
      v[k] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (at >= n) continue;
      if (i >= 0 && i + 3 < a.vocab) {
        v[k] = *reinterpret_cast<const float4*>(x + i);
      } else {
        if (i >= 0 && i < a.vocab) v[k].x = x[i];
        if (i + 1 >= 0 && i + 1 < a.vocab) v[k].y = x[i + 1];
        if (i + 2 >= 0 && i + 2 < a.vocab) v[k].z = x[i + 2];
        if (i + 3 >= 0 && i + 3 < a.vocab) v[k].w = x[i + 3];
      }
    }
    if (hist > 0 || has_bias) {
      const uint4 none = make_uint4(0, 0, 0, 0);
      if (base > s0) __syncthreads();
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const int at = 4 * (tid + k * kThreads);
        if (at >= n) break;
        if (pen) *reinterpret_cast<uint4*>(said + at) = none;
        if (has_bias) *reinterpret_cast<uint4*>(bias + at) = none;
      }
      __syncthreads();
#pragma unroll 4
      for (int i = tid; i < hist; i += kThreads) {
        const uint32_t t = (uint32_t)said_ids[i] - first;
        // ids of this chunk; not those below 0, which the first chunk's shift would let in
        if (t >= (uint32_t)n || (uint32_t)said_ids[i] >= (uint32_t)a.vocab) continue;
        if (i >= prompt) atomicAdd(&said[t], 1u);
        else atomicOr(&said[t], kSeen);
      }
      if (has_bias) {
        // the last entry of an id counts: entries leave their number, the largest stays ...
#pragma unroll 1
        for (int e = e0 + tid; e < e1; e += kThreads) {
          const uint32_t t = (uint32_t)c.bias_ids[e] - first;
          if (t < (uint32_t)n && (uint32_t)c.bias_ids[e] < (uint32_t)a.vocab)
            atomicMax(&bias[t], (uint32_t)(e - e0 + 1));
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int at = 4 * (tid + k * kThreads), i = base + at - shift;
      if (at >= n) break;
      float r[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
      if (hist > 0) {
        const uint4 w = *reinterpret_cast<const uint4*>(said + at);
        if ((w.x | w.y | w.z | w.w) != 0) {
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (u[j]) r[j] = penalised(r[j], u[j], rep, freq, pres, c.repetition != nullptr);
        }
      }
      if (has_bias) {
        const uint4 w = *reinterpret_cast<const uint4*>(bias + at);
        if ((w.x | w.y | w.z | w.w) != 0) {
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)  // ... and is looked up here
            if (u[j]) r[j] = __fadd_rn(r[j], c.bias_vals[e0 + u[j] - 1]);
        }
      }
      if (mask) {
        // bits of ids i .. i + 3, which may lie in two words; none of ids out of range is used
        const int w0 = max(i, 0) >> 5, w1 = min(i + 3, a.vocab - 1) >> 5;
        uint32_t bits = mask[w0];
        const uint32_t more = w1 > w0 ? mask[w1] : 0u;
        bits = i >= 0 ? __funnelshift_r(bits, more, i & 31) : bits << -i;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!((bits >> j) & 1u)) r[j] = -INFINITY;
      }
      if (i >= 0 && i + 3 < a.vocab) {
        if (y) {
          const bool same = in_place && __float_as_uint(r[0]) == __float_as_uint(v[k].x) &&
                            __float_as_uint(r[1]) == __float_as_uint(v[k].y) &&
                            __float_as_uint(r[2]) == __float_as_uint(v[k].z) &&
                            __float_as_uint(r[3]) == __float_as_uint(v[k].w);
          if (together) {
            if (!same) *reinterpret_cast<float4*>(y + i) = make_float4(r[0], r[1], r[2], r[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[i + j] = r[j];
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r[j] > bv) {
            bv = r[j];
            bi = i + j;
          }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (i + j < 0 || i + j >= a.vocab) continue;
          if (y) y[i + j] = r[j];
          if (r[j] > bv) {
            bv = r[j];
            bi = i + j;
          }
        }
      }
    }
  }
  if (!a.ids) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
  if (lane == 0) {
    best_v[tid >> 5] = bv;
    best_i[tid >> 5] = bi;
  }
  __syncthreads();
  if (tid < 32) {
    bv = lane < kThreads / 32 ? best_v[lane] : -INFINITY;
    bi = lane < kThreads / 32 ? best_i[lane] : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
  }
  if (ranks > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid == 0) {
      const unsigned long long w = (unsigned long long)__float_as_uint(bv) << 32 | (uint32_t)bi;
      asm volatile(
          "{\n .reg .u32 p;\n mapa.shared::cluster.u32 p, %0, 0;\n"
          " st.shared::cluster.u64 [p], %1;\n}" ::"r"(smem_u32(&found[rank])),
          "l"(w)
          : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0)
      for (uint32_t u = 1; u < ranks; ++u)
        better(bv, bi, __uint_as_float((uint32_t)(found[u] >> 32)), (int)(uint32_t)found[u]);
  }
  if (tid == 0) a.ids[row] = bv == -INFINITY ? 0u : (uint32_t)bi;
}

}  // namespace
}  // namespace myos

using namespace myos;

extern "C" int myos_dev_logit_controls(float* d_out, size_t out_stride, const float* d_logits,
                                       size_t logits_stride, size_t rows, size_t vocab,
                                       const myos_logit_controls_args* c, uint32_t* d_ids,
                                       void* stream) {
  if (rows == 0) return MYOS_OK;
  if (!d_logits || (!d_out && !d_ids)) return MYOS_ERR_ARG;
  if (!aligned(d_logits, 4) || !aligned(d_out, 4) || !aligned(d_ids, 4)) return MYOS_ERR_ARG;
  if (vocab == 0 || vocab > 0x40000000 || rows > 0x0fffffff || logits_stride < vocab ||
      logits_stride > ((size_t)1 << 40) ||
      (d_out && (out_stride < vocab || out_stride > ((size_t)1 << 40))))
    return MYOS_ERR_SHAPE;
  if (d_out == d_logits && rows > 1 && out_stride != logits_stride) return MYOS_ERR_ARG;
  LogitArgs a = {};
  a.out = d_out;
  a.logits = d_logits;
  a.out_stride = (int64_t)out_stride;
  a.logits_stride = (int64_t)logits_stride;
  a.vocab = (int)vocab;
  a.ids = d_ids;
  if (c) {
    const uintptr_t words = (uintptr_t)c->history | (uintptr_t)c->prompt_lens |
                            (uintptr_t)c->history_lens | (uintptr_t)c->repetition |
                            (uintptr_t)c->frequency | (uintptr_t)c->presence |
                            (uintptr_t)c->bias_starts | (uintptr_t)c->bias_ids |
                            (uintptr_t)c->bias_vals | (uintptr_t)c->mask | (uintptr_t)c->mask_rows;
    if ((words & 3) != 0) return MYOS_ERR_ARG;
    if (!c->history && (c->repetition || c->frequency || c->presence)) return MYOS_ERR_ARG;
    if (c->bias_starts && (!c->bias_ids || !c->bias_vals)) return MYOS_ERR_ARG;
    if (c->history && (c->history_width > 0x7fffffff || c->history_stride < c->history_width ||
                       c->history_stride > ((uint64_t)1 << 40)))
      return MYOS_ERR_SHAPE;
    if (c->num_bias > 0x7fffffff) return MYOS_ERR_SHAPE;
    if (c->mask && (c->mask_stride < (vocab + 31) / 32 || c->mask_stride > ((uint64_t)1 << 40) ||
                    c->num_masks > 0x7fffffff || (!c->mask_rows && c->num_masks < rows)))
      return MYOS_ERR_SHAPE;
    a.c = *c;
  }
  // As many blocks a row as keep the device busy, slices of at least 2048 ids;
  // slices and chunks in multiples of four (three ids more: a row's shift).
  const size_t ids_shifted = vocab + 3;
  int cluster = kMaxCluster;
  while (cluster > 1 && (rows * cluster > (size_t)sm_count() * 8 || ids_shifted / cluster < 2048))
    cluster /= 2;
  a.slice = (int)((ids_shifted + cluster - 1) / cluster + 3) & ~3;
  const int passes = (a.slice + kMaxChunk - 1) / kMaxChunk;
  a.chunk = ((a.slice + passes - 1) / passes + 3) & ~3;
  const bool pen = a.c.history && (a.c.repetition || a.c.frequency || a.c.presence);
  const size_t smem = 4 * (size_t)a.chunk * ((pen ? 1 : 0) + (a.c.bias_starts ? 1 : 0));
  static std::atomic<uint64_t> raised{0};
  if (raise_smem_limit((const void*)k_logit_controls, 2 * kMaxChunk * 4, &raised) != cudaSuccess)
    return MYOS_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return counted(cudaLaunchKernelEx(&cfg, k_logit_controls, a)) == cudaSuccess ? MYOS_OK
                                                                               : MYOS_ERR_CUDA;
}
