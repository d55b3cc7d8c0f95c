// Attention of one new token per sequence over a paged KV cache.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace myos {
namespace {

constexpr int kMaxGroup = 8;  // query heads per KV head, as tensor_core::gqa_attn_f32 here

struct PagedAttnArgs {
  float* out;
  float* lse;
  const float* q;
  int64_t out_stride, q_stride;
  int nseq, hq, group;
  const int32_t* table;
  int64_t table_stride, max_blocks;
  const int32_t* kv_lens;
  float scale;
  uint32_t window;
};

MYOS_DEV float load1(const float* p) { return *p; }
MYOS_DEV float load1(const __nv_bfloat16* p) { return bf16_at(reinterpret_cast<const uint16_t*>(p)); }

// One block per (sequence, KV head); warp w takes keys w, w + 8, ...; a lane
// holds dims lane, lane + 32, ... of the group's queries and outputs. Each
// warp keeps its own running maximum and sum of every head; the warps' states
// meet in shared memory at the end.
template <class KT>
__global__ void __launch_bounds__(256) k_paged_attn(PagedAttnArgs a, PagedKv<KT> kv) {
  constexpr int kWarps = 8, kD = 8;
  __shared__ float part[kWarps][256];
  __shared__ float ms[kWarps][kMaxGroup], ls[kWarps][kMaxGroup];
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d = (int)kv.d, G = a.group;
  const int64_t P = kv.page_size;
  const int64_t len = min((int64_t)max(a.kv_lens[b], 0), a.max_blocks * P);
  const int64_t start = a.window > 0 && len > a.window ? len - a.window : 0;
  const float* q = a.q + b * a.q_stride + (int64_t)h * G * d;
  float qr[kMaxGroup][kD], o[kMaxGroup][kD], m[kMaxGroup], l[kMaxGroup];
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < kD; ++i) {
      const int c = lane + 32 * i;
      o[g][i] = 0.f;
      qr[g][i] = g < G && c < d ? q[g * d + c] : 0.f;
    }
  }
  for (int64_t t = start + warp; t < len; t += kWarps) {
    const int32_t page = a.table[b * a.table_stride + t / P];
    if (page < 0 || (uint32_t)page >= kv.num_pages) continue;
    const int64_t at = page * kv.page_stride + h * kv.head_stride + (t % P) * kv.slot_stride;
    float kr[kD], vr[kD];
#pragma unroll
    for (int i = 0; i < kD; ++i) {
      const int c = lane + 32 * i;
      kr[i] = c < d ? load1(kv.k + at + c) : 0.f;
      vr[i] = c < d ? load1(kv.v + at + c) : 0.f;
    }
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) {
      if (g >= G) break;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kD; ++i) s = fmaf(qr[g][i], kr[i], s);
      s = warp_sum(s) * a.scale;
      const float mn = fmaxf(m[g], s);
      const float c = expf(m[g] - mn), p = expf(s - mn);
      m[g] = mn;
      l[g] = l[g] * c + p;
#pragma unroll
      for (int i = 0; i < kD; ++i) o[g][i] = fmaf(p, vr[i], o[g][i] * c);
    }
  }
  for (int g = 0; g < G; ++g) {
    float mg = 0.f, lg = 0.f;
#pragma unroll
    for (int u = 0; u < kMaxGroup; ++u)
      if (u == g) {
        mg = m[u];
        lg = l[u];
#pragma unroll
        for (int i = 0; i < kD; ++i) part[warp][lane + 32 * i] = o[u][i];
      }
    if (lane == 0) {
      ms[warp][g] = mg;
      ls[warp][g] = lg;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ms[w][g]);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < kWarps; ++w) total += ls[w][g] * expf(ms[w][g] - ref);
    const int head = h * G + g;
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
      float s = 0.f;
      for (int w = 0; w < kWarps; ++w) s += part[w][c] * expf(ms[w][g] - ref);
      a.out[b * a.out_stride + (int64_t)head * d + c] = total > 0.f ? s / total : 0.f;
    }
    if (a.lse && threadIdx.x == 0)
      a.lse[(int64_t)b * a.hq + head] = total > 0.f ? top + logf(total) : -INFINITY;
    __syncthreads();
  }
}

template <class KT>
cudaError_t launch(const PagedAttnArgs& a, const myos_paged_kv* kv, cudaStream_t st) {
  k_paged_attn<KT><<<dim3(kv->num_kv_heads, a.nseq), 256, 0, st>>>(a, paged_view<KT>(kv));
  return counted(cudaGetLastError());
}

}  // namespace
}  // namespace myos

using namespace myos;

extern "C" int myos_dev_paged_attn(float* d_out, size_t out_stride, float* d_lse, const float* d_q,
                                   size_t q_stride, size_t nseq, size_t num_q_heads,
                                   const myos_paged_kv* kv, const int32_t* d_block_table,
                                   size_t table_stride, size_t max_blocks,
                                   const int32_t* d_kv_lens, float scale, uint32_t window,
                                   void* d_work, size_t work_bytes, void* stream) {
  if (int st = paged_check(kv)) return st;
  if (nseq == 0) return MYOS_OK;
  if (!d_out || !d_q || !d_block_table || !d_kv_lens || !d_work) return MYOS_ERR_ARG;
  const size_t d = kv->head_dim;
  if (num_q_heads == 0 || num_q_heads % kv->num_kv_heads != 0 ||
      num_q_heads / kv->num_kv_heads > (size_t)kMaxGroup || nseq > 65535 || max_blocks == 0 ||
      max_blocks > 0x7fffffff || table_stride < max_blocks || table_stride > ((size_t)1 << 40) ||
      max_blocks * kv->page_size > 0x7fffffff || q_stride < num_q_heads * d ||
      out_stride < num_q_heads * d || q_stride > ((size_t)1 << 30) ||
      out_stride > ((size_t)1 << 30))
    return MYOS_ERR_SHAPE;
  if (!aligned(d_q, 16) || !aligned(d_out, 16) || q_stride % 4 != 0 || out_stride % 4 != 0 ||
      !aligned(d_lse, 4) || !aligned(d_block_table, 4) || !aligned(d_kv_lens, 4) ||
      !aligned(d_work, 16))
    return MYOS_ERR_ARG;
  if (work_bytes < MYOS_PAGED_WORK_BYTES) return MYOS_ERR_SCRATCH_LIMIT;
  PagedAttnArgs a;
  a.out = d_out;
  a.lse = d_lse;
  a.q = d_q;
  a.out_stride = (int64_t)out_stride;
  a.q_stride = (int64_t)q_stride;
  a.nseq = (int)nseq;
  a.hq = (int)num_q_heads;
  a.group = (int)(num_q_heads / kv->num_kv_heads);
  a.table = d_block_table;
  a.table_stride = (int64_t)table_stride;
  a.max_blocks = (int64_t)max_blocks;
  a.kv_lens = d_kv_lens;
  a.scale = scale;
  a.window = window;
  const cudaError_t e = kv->kv_dtype == MYOS_KV_F32
                            ? launch<float>(a, kv, (cudaStream_t)stream)
                            : launch<__nv_bfloat16>(a, kv, (cudaStream_t)stream);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}
