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
  int slice, chunk, slots;  // ids of a block, and of a pass (multiples of 4); table slots
  uint32_t* ids;
  myos_logit_controls_args c;
};

// A row is shared by a cluster of blocks, a slice of the vocabulary each. A
// block sorts the row's tokens and biases that fall into its slice into a hash
// table in shared memory by integer atomics (the result does not depend on their
// order); then the slice passes once, four ids a thread and load, with nothing
// to wait for between them: out = logits under the mask, and the largest of the
// ids that no token or bias touches; then the touched ids are computed one to a
// thread, over what that pass wrote. A history longer than the table has room
// for is handled in chunks of as many ids as the table has slots, each id in the
// slot of its own number. The blocks' best ids meet in the first block's shared
// memory.
//
// What this replaces: tables of one word an id, chunk by chunk, with the
// penalties in the pass over all ids, 59 instructions an id (64 rows of 152064:
// 52 us), and with the touched ids computed before that pass from lists, 40
// instructions (39 us): zeroing and reading the tables and looking through the
// lists for every chunk cost more than the pass.
#ifndef SLOTS
#define SLOTS 2
#define VT 512
#endif
constexpr int kMaxCluster = 8;
constexpr int kTokens = 4096, kBiases = 1024;  // of a row: room in the table
constexpr int kMaxChunk = 65536;
constexpr uint32_t kSeen = 0x80000000u;  // in the prompt; the low bits count the output
constexpr uint32_t kNoId = 0xffffffffu;

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

template <int kThreads>
__global__ void __launch_bounds__(kThreads) k_logit_controls(const LogitArgs a) {
  extern __shared__ __align__(16) uint32_t tables[];
  __shared__ float best_v[32];
  __shared__ int best_i[32];
  __shared__ unsigned long long found[kMaxCluster];
  __shared__ int listed;
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
  const bool together = (((uintptr_t)x ^ (uintptr_t)y) & 15) == 0;

  int hist = 0, prompt = 0;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (c.history && (c.repetition || c.frequency || c.presence)) {
    hist = (int)c.history_width;
    if (c.history_lens) hist = min(hist, max(c.history_lens[row], 0));
    if (c.prompt_lens) prompt = c.prompt_lens[row];
    if (c.repetition) rep = c.repetition[row];
    if (c.frequency) freq = c.frequency[row];
    if (c.presence) pres = c.presence[row];
  }
  const int32_t* said = c.history + row * (int64_t)c.history_stride;
  int e0 = 0, e1 = 0;
  if (c.bias_starts) {
    e0 = min(max(c.bias_starts[row], 0), (int)c.num_bias);
    e1 = min(max(c.bias_starts[row + 1], 0), (int)c.num_bias);
  }
  const bool touched = hist > 0 || e1 > e0;
  const bool hashed = hist <= kTokens && e1 - e0 <= kBiases;
  const uint32_t* mask = nullptr;
  if (c.mask) {
    const int64_t g = c.mask_rows ? c.mask_rows[row] : row;
    if (g >= 0 && g < (int64_t)c.num_masks) mask = c.mask + g * (int64_t)c.mask_stride;
  }
  // the chunk's mask and touched ids, a bit each (two mask words more than full
  // ones: a chunk may begin inside a word); the table: an id's place in the
  // chunk, the history's word, 1 + its last bias entry; the slots in use
  const uint32_t slots = a.slots;
  const int words = a.chunk / 32 + 2;
  uint32_t* mask_s = tables;
  uint32_t* bits = mask_s + words;
  uint32_t* key = bits + words;
  uint32_t* word = key + slots;
  uint32_t* bias = word + slots;
  uint16_t* used = reinterpret_cast<uint16_t*>(bias + slots);

  float bv = -INFINITY;
  int bi = 0;
  const int s0 = rank * a.slice, s1 = min(s0 + a.slice, a.vocab + shift);
  const int step = hashed || !touched ? a.chunk : min(a.chunk, (int)slots & ~3);
#pragma unroll 1
  for (int base = s0; base < s1; base += step) {
    const int n = min(step, s1 - base);  // shifted ids base .. base + n
    const int first = base - shift;      // the id of the first
    const int word0 = max(first, 0) >> 5;
    if (base > s0) __syncthreads();
    if (mask)
#pragma unroll 1
      for (int k = tid; k < n / 32 + 2; k += kThreads)
        mask_s[k] = (word0 + k) * 32 < a.vocab ? mask[word0 + k] : 0u;
    if (touched) {
#pragma unroll 1
      for (int k = tid; k < (int)slots; k += kThreads) {
        key[k] = kNoId;
        word[k] = 0;
        bias[k] = 0;
      }
#pragma unroll 1
      for (int k = tid; k < n / 32 + 1; k += kThreads) bits[k] = 0;
      if (tid == 0) listed = 0;
      __syncthreads();
      // the slot of an id of this chunk, or -1
      auto slot_of = [&](int32_t id) -> int {
        const uint32_t t = (uint32_t)id - (uint32_t)first;
        if ((uint32_t)id >= (uint32_t)a.vocab || t >= (uint32_t)n) return -1;
        uint32_t h = hashed ? __umulhi(t * 2654435761u, slots) : t;
        for (;;) {
          const uint32_t was = atomicCAS(&key[h], kNoId, t);
          if (was == kNoId) {
            atomicOr(&bits[t >> 5], 1u << (t & 31));
            used[atomicAdd(&listed, 1)] = (uint16_t)h;
            break;
          }
          if (was == t) break;
          if (++h == slots) h = 0;
        }
        return (int)h;
      };
      constexpr int kBatch = 4;
#pragma unroll 1
      for (int i0 = tid; i0 < hist; i0 += kBatch * kThreads) {
        int32_t id[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) id[k] = i0 + k * kThreads < hist ? said[i0 + k * kThreads] : -1;
#pragma unroll 1
        for (int k = 0; k < kBatch; ++k) {
          const int32_t now = id[0];
          id[0] = id[1], id[1] = id[2], id[2] = id[3];
          const int h = slot_of(now);
          if (h < 0) continue;
          if (i0 + k * kThreads < prompt) atomicOr(&word[h], kSeen);
          else atomicAdd(&word[h], 1u);
        }
      }
      // the last entry of an id counts: entries leave their number, the largest stays
#pragma unroll 1
      for (int e = e0 + tid; e < e1; e += kThreads) {
        const int h = slot_of(c.bias_ids[e]);
        if (h >= 0) atomicMax(&bias[h], (uint32_t)(e - e0 + 1));
      }
    }
    if (touched || mask) __syncthreads();

    // ids i .. i + 3 at place `at` of the chunk: the value of an id, edge or not
    auto pass = [&](int at, float (&r)[4]) -> uint32_t {  // the untouched ones
      uint32_t keep = 15u;
      if (touched) keep = ~(bits[at >> 5] >> (at & 31));  // at is a multiple of 4
      if (mask) {
        // their bits may lie in two words; bits of ids out of range are not used
        const int i = first + at, w0 = (max(i, 0) >> 5) - word0;
        const uint32_t m = mask_s[w0];
        const uint32_t m4 = i >= 0 ? __funnelshift_r(m, mask_s[w0 + 1], i & 31) : m << -i;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!((m4 >> j) & 1u)) r[j] = -INFINITY;
      }
      return keep;
    };
    auto take = [&](float v, int i) {  // ids come in rising order
      if (v > bv) {
        bv = v;
        bi = i;
      }
    };
    // groups [g0, g1) lie within the row; at most one before and one behind do not
    const int g0 = first < 0 ? 1 : 0, g1 = min((n + 3) / 4, (a.vocab - first) / 4);
    const float* xc = x + first;
    float* yc = y + first;
    constexpr int kUnroll = 4;
#pragma unroll 1
    for (int gr = g0 + tid; gr < g1; gr += kUnroll * kThreads) {
      float4 v[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (gr + k * kThreads < g1)
          v[k] = *reinterpret_cast<const float4*>(xc + 4 * (gr + k * kThreads));
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        if (gr + k * kThreads >= g1) break;
        const int at = 4 * (gr + k * kThreads);
        float r[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
        const uint32_t keep = pass(at, r);
        if (y) {
          if (together) {
            *reinterpret_cast<float4*>(yc + at) = make_float4(r[0], r[1], r[2], r[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) yc[at + j] = r[j];
          }
        }
        if (fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3])) > bv) {  // NaN is passed over
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (keep >> j & 1u) take(r[j], first + at + j);
        }
      }
    }
    // the groups that reach over the row's ends
    if (tid < 2) {
      const int gr = tid == 0 ? 0 : g1;
      if ((tid == 0 ? g0 == 1 : 4 * g1 < n) && (tid == 0 || g1 >= g0)) {
        float r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = first + 4 * gr + j;
          r[j] = i >= 0 && i < a.vocab ? x[i] : -INFINITY;
        }
        const uint32_t keep = pass(4 * gr, r);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = first + 4 * gr + j;
          if (i < 0 || i >= a.vocab) continue;
          if (y) y[i] = r[j];
          if ((keep >> j & 1u) && (r[j] > bv || (r[j] == bv && i < bi))) {
            bv = r[j];
            bi = i;
          }
        }
      }
    }
    if (!touched) continue;
    __syncthreads();
    // the touched ids, over what the pass wrote (an id that the mask takes out
    // is -inf whatever it was, any other still holds its logit)
#pragma unroll 1
    for (int k = tid; k < listed; k += kThreads) {
      const int h = used[k], i = first + (int)key[h];
      float r = x[i];
      const uint32_t w = word[h], e = bias[h];
      if (w) r = penalised(r, w, rep, freq, pres, c.repetition != nullptr);
      if (e) r = __fadd_rn(r, c.bias_vals[e0 + e - 1]);
      if (mask && !(mask_s[(i >> 5) - word0] >> (i & 31) & 1u)) r = -INFINITY;
      if (y) y[i] = r;
      if (r > bv || (r == bv && i < bi)) {
        bv = r;
        bi = i;
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

template <int kThreads>
cudaError_t launch_controls(LogitArgs a, size_t rows, cudaStream_t st) {
  // As many blocks a row as are resident at once, slices of at least 2048 ids;
  // slices and chunks in multiples of four (three ids more: a row's shift).
  const int ids = a.vocab + 3;
  int cluster = kMaxCluster;
  while (cluster > 1 &&
         (rows * cluster > (size_t)sm_count() * SLOTS || ids / cluster < 2048))
    cluster /= 2;
  a.slice = ((ids + cluster - 1) / cluster + 3) & ~3;
  const int passes = (a.slice + kMaxChunk - 1) / kMaxChunk;
  a.chunk = ((a.slice + passes - 1) / passes + 3) & ~3;
  const bool pen = a.c.history && (a.c.repetition || a.c.frequency || a.c.presence);
  // room for every id that the listed tokens and biases can name, and a quarter more
  size_t room = 0;
  if (pen) room += a.c.history_width < kTokens ? a.c.history_width : kTokens;
  if (a.c.bias_starts) room += a.c.num_bias < kBiases ? a.c.num_bias : kBiases;
  a.slots = room ? (int)((room + room / 4 + 31) & ~(size_t)31) : 0;
  const auto bytes = [](size_t chunk, size_t slots) { return 8 * (chunk / 32 + 2) + 14 * slots; };
  const size_t smem = bytes(a.chunk, a.slots);
  constexpr size_t kMostSlots = (kTokens + kBiases) * 5 / 4;
  static_assert(kMostSlots % 32 == 0 && kMostSlots <= 65536);
  static std::atomic<uint64_t> raised{0};
  const cudaError_t e = raise_smem_limit((const void*)k_logit_controls<kThreads>,
                                         bytes(kMaxChunk, kMostSlots), &raised);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return counted(cudaLaunchKernelEx(&cfg, k_logit_controls<kThreads>, a));
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
  const cudaError_t e = rows * kMaxCluster <= (size_t)sm_count()
                            ? launch_controls<1024>(a, rows, (cudaStream_t)stream)
                            : launch_controls<VT>(a, rows, (cudaStream_t)stream);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}
