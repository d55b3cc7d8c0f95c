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
  uint32_t* ids;
  myos_logit_controls_args c;
};

constexpr int kThreads = 1024, kChunk = 8192;
constexpr uint32_t kSeen = 0x80000000u;  // in the prompt or the output; the low bits count the output

// x under the penalties: each step rounded, as a chain of elementwise passes
// would round it.
MYOS_DEV float penalised(float x, uint32_t said, float rep, float freq, float pres, bool has_rep) {
  if (said == 0) return x;
  if (has_rep) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
  const uint32_t times = said & ~kSeen;
  x = __fsub_rn(x, __fmul_rn(freq, (float)times));
  return times ? __fsub_rn(x, pres) : x;
}

// One block per row; the vocabulary goes by in chunks. For a chunk the row's
// history and biases are sorted into shared tables by integer atomics (the
// result does not depend on their order), then the logits pass once.
__global__ void __launch_bounds__(kThreads) k_logit_controls(LogitArgs a) {
  extern __shared__ uint32_t table[];
  uint32_t* said = table;
  uint32_t* bias = table + kChunk;  // 1 + the last bias entry of the token
  __shared__ float best_v[32];
  __shared__ int best_i[32];
  const int row = blockIdx.x, tid = threadIdx.x;
  const myos_logit_controls_args& c = a.c;
  const float* x = a.logits + row * a.logits_stride;
  float* y = a.out ? a.out + row * a.out_stride : nullptr;
  const bool pen = c.history && (c.repetition || c.frequency || c.presence);
  int64_t hist = 0, prompt = 0;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (pen) {
    hist = (int64_t)c.history_width;
    if (c.history_lens) hist = min(hist, (int64_t)max(c.history_lens[row], 0));
    if (c.prompt_lens) prompt = c.prompt_lens[row];
    if (c.repetition) rep = c.repetition[row];
    if (c.frequency) freq = c.frequency[row];
    if (c.presence) pres = c.presence[row];
  }
  int64_t e0 = 0, e1 = 0;
  if (c.bias_starts) {
    const int64_t n = (int64_t)c.num_bias;
    e0 = min((int64_t)max(c.bias_starts[row], 0), n);
    e1 = min((int64_t)max(c.bias_starts[row + 1], 0), n);
  }
  const uint32_t* mask = nullptr;
  if (c.mask) {
    const int64_t g = c.mask_rows ? c.mask_rows[row] : row;
    if (g >= 0 && g < (int64_t)c.num_masks) mask = c.mask + g * (int64_t)c.mask_stride;
  }
  float bv = -INFINITY;
  int bi = 0;
  for (int base = 0; base < a.vocab; base += kChunk) {
    const int n = min(kChunk, a.vocab - base);
    if (pen)
      for (int i = tid; i < n; i += kThreads) said[i] = 0;
    if (e1 > e0)
      for (int i = tid; i < n; i += kThreads) bias[i] = 0;
    __syncthreads();
    for (int64_t i = tid; i < hist; i += kThreads) {
      const uint32_t t = (uint32_t)c.history[row * (int64_t)c.history_stride + i] - (uint32_t)base;
      if (t >= (uint32_t)n) continue;
      atomicOr(&said[t], kSeen);
      if (i >= prompt) atomicAdd(&said[t], 1u);
    }
    for (int64_t e = e0 + tid; e < e1; e += kThreads) {
      const uint32_t t = (uint32_t)c.bias_ids[e] - (uint32_t)base;
      if (t < (uint32_t)n) atomicMax(&bias[t], (uint32_t)(e - e0 + 1));
    }
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      float v = x[base + i];
      if (pen) v = penalised(v, said[i], rep, freq, pres, c.repetition != nullptr);
      if (e1 > e0 && bias[i]) v = __fadd_rn(v, c.bias_vals[e0 + bias[i] - 1]);
      if (mask && !((mask[(base + i) >> 5] >> ((base + i) & 31)) & 1u)) v = -INFINITY;
      if (y) y[base + i] = v;
      if (v > bv) {
        bv = v;
        bi = base + i;
      }
    }
    __syncthreads();
  }
  if (!a.ids) return;
  // first maximum: the larger value, on a tie the lower id
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, bv, o);
    const int i = __shfl_xor_sync(0xffffffffu, bi, o);
    if (v > bv || (v == bv && i < bi)) {
      bv = v;
      bi = i;
    }
  }
  if ((tid & 31) == 0) {
    best_v[tid >> 5] = bv;
    best_i[tid >> 5] = bi;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w)
      if (best_v[w] > bv || (best_v[w] == bv && best_i[w] < bi)) {
        bv = best_v[w];
        bi = best_i[w];
      }
    a.ids[row] = bv == -INFINITY ? 0u : (uint32_t)bi;
  }
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
  if (vocab == 0 || vocab > 0x40000000 || rows > 0x7fffffff || logits_stride < vocab ||
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
  constexpr int smem = 2 * kChunk * 4;
  static std::atomic<uint64_t> raised{0};
  if (raise_smem_limit((const void*)k_logit_controls, smem, &raised) != cudaSuccess)
    return MYOS_ERR_CUDA;
  k_logit_controls<<<(unsigned)rows, kThreads, smem, (cudaStream_t)stream>>>(a);
  return counted(cudaGetLastError()) == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}
