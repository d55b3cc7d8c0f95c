// Logits under the requests' controls (penalties for repeated tokens, biases,
// grammar masks) and the greedy id.
#include "common.cuh"
#include "cp_async.cuh"
#include "kernels.h"
#include "logits_plan.h"
#include "paged.h"

namespace myos {
namespace {

struct LogitArgs {
  float* out;
  const float* logits;
  int64_t out_stride, logits_stride;
  int vocab;
  int chunk, slots, room;  // ids of a pass (a multiple of kRun), table slots (of 4), list
  uint32_t* ids;
  myos_logit_controls_args c;
};

// A row is shared by a cluster of blocks, every so many-th run of 128 ids each
// (common tokens have low ids: in plain slices the first block had most of the
// work). A block lists the row's tokens and biases among its ids and sorts them
// into a hash table in shared memory by integer atomics (the result does not
// depend on their order); then its ids pass once, four a thread and load, with nothing to wait
// for between them: out = logits under the mask, and the largest of the ids that
// no token or bias touches; then the touched ids are computed one to a thread,
// over what that pass wrote. Where the list runs over, the block's ids go in
// chunks of as many as the table has slots, each id in the slot of its own
// number, and the whole history is looked through for each. The blocks' best ids
// meet in the first block's shared memory.
//
// The list has 5120 entries at most, of tokens, not of distinct ones. A row's
// history passes it from about 5 thousand tokens on where a row has one block, 10
// where it has two, 20 where it has four, sooner where few ids make most of it,
// and from there the time grows with the history times the steps: 64 rows of
// 152064 with 4096, 8192, 16384 and 32768 tokens take 23, 45, 136 and 304 us, 256
// rows with 4096 and 8192 94 and 310 us; 64 rows that each said one token 4096
// times 77 us.
//
// Everything before the pass is latency (row parameters, tokens, table), so it
// is kept off the memory's back: the table is cleared before the launch's
// dependency, the first tokens and logits and the mask are on their way while
// the row's lengths come. 64 rows of 152064 with every control (79 MB): 24 us;
// with tables of one word an id, chunk by chunk, and the penalties in the pass
// over all ids 52 us (59 instructions an id, nearly every warp went through the
// divisions), with the touched ids computed before that pass 39 us. The pass
// itself, without controls, takes 17.9 us; 12 us is the memory's share.
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

template <int kThreads, int kDepth, int kUnroll>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) k_logit_controls(const LogitArgs a) {
  extern __shared__ __align__(16) uint32_t tables[];
  __shared__ float best_v[32];
  __shared__ int best_i[32];
  __shared__ unsigned long long found[kMaxCluster];
  __shared__ int listed, in_use;
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  if (a.ids && ranks > 1)  // the first block's memory is written to below: it has to have started
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int64_t row = blockIdx.x / ranks;
  const myos_logit_controls_args& c = a.c;
  // the chunk's touched ids, a bit each; the table: an id's place among the
  // block's, the history's word, 1 + its last bias entry; the mask's words; the
  // list; the slots in use
  const uint32_t slots = a.slots;
  float4* ring = reinterpret_cast<float4*>(tables) + tid;  // slot t at t * kThreads
  uint32_t* key = tables + kDepth * kThreads * 4;
  uint32_t* word = key + slots;
  uint32_t* bias = word + slots;
  uint32_t* bits = bias + slots;
  uint32_t* mask_s = bits + (slots ? a.chunk / 32 : 0);
  uint2* list = reinterpret_cast<uint2*>(mask_s + (c.mask ? (a.chunk / kRun * kRunWords + 2) & ~1 : 0));
  uint16_t* used = reinterpret_cast<uint16_t*>(list + a.room);
  auto clear_tables = [&]() {
    const uint4 none = make_uint4(0, 0, 0, 0), no_id = make_uint4(kNoId, kNoId, kNoId, kNoId);
#pragma unroll 1
    for (int k = tid; k < (int)slots / 4; k += kThreads) reinterpret_cast<uint4*>(key)[k] = no_id;
    // word, bias and bits lie behind one another
#pragma unroll 1
    for (int k = tid; k < (int)slots / 2 + a.chunk / 128; k += kThreads)
      reinterpret_cast<uint4*>(word)[k] = none;
    if (tid == 0) in_use = 0;
  };
  if (slots) clear_tables();
  if (tid == 0) listed = 0;
  pdl_launch();
  pdl_wait();
  const float* x = a.logits + row * a.logits_stride;
  float* y = a.out ? a.out + row * a.out_stride : nullptr;
  // Ids count from `shift` on, so that groups of four lie on 16 bytes of x.
  const int shift = (int)((uintptr_t)x >> 2 & 3);
  const bool together = (((uintptr_t)x ^ (uintptr_t)y) & 15) == 0;

  int hist = 0, prompt = 0;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  const int32_t* said = c.history + row * (int64_t)c.history_stride;
  // the row's first 4096 tokens on their way before its length is known
  constexpr int kEarly = 4096 / kThreads;
  int32_t early[kEarly];
  if (c.history && (c.repetition || c.frequency || c.presence)) {
#pragma unroll
    for (int k = 0; k < kEarly; ++k)
      early[k] = tid + k * kThreads < (int)c.history_width ? said[tid + k * kThreads] : -1;
    hist = (int)c.history_width;
    if (c.history_lens) hist = min(hist, max(c.history_lens[row], 0));
    if (c.prompt_lens) prompt = c.prompt_lens[row];
    if (c.repetition) rep = c.repetition[row];
    if (c.frequency) freq = c.frequency[row];
    if (c.presence) pres = c.presence[row];
  }
  int e0 = 0, e1 = 0;
  if (c.bias_starts) {
    e0 = min(max(c.bias_starts[row], 0), (int)c.num_bias);
    e1 = min(max(c.bias_starts[row + 1], 0), (int)c.num_bias);
  }
  const int32_t early_bias = e0 + tid < e1 ? c.bias_ids[e0 + tid] : -1;
  const bool touched = slots > 0 && (hist > 0 || e1 > e0);  // the plan has slots for either
  const uint32_t* mask = nullptr;
  if (c.mask) {
    const int64_t g = c.mask_rows ? c.mask_rows[row] : row;
    if (g >= 0 && g < (int64_t)c.num_masks) mask = c.mask + g * (int64_t)c.mask_stride;
  }
  // The block's ids: place l is id (l / kRun * ranks + rank) * kRun + l % kRun - shift.
  const uint32_t log_ranks = __ffs(ranks) - 1;
  const int runs = (a.vocab + shift + kRun - 1) / kRun;
  const int places = (runs - (int)rank + (int)ranks - 1) / (int)ranks * kRun;
  auto id_at = [&](int l) -> int {
    return (((l / kRun) << log_ranks | (int)rank) * kRun | (l & (kRun - 1))) - shift;
  };
  // the first 3 ids of a row may come before it, and any behind it
  const uint32_t whole = a.vocab > 3 ? a.vocab - 3 : 0;  // ids from which four on are in the row

  // the best id so far, and the best whole group of four (its first largest value
  // is looked for once, at the end)
  const bool ids = a.ids != nullptr;
  float bv = -INFINITY, gv = -INFINITY, group[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  int bi = 0, gi = 0;
  auto take = [&](float v, int i) {
    if (v > bv || (v == bv && i < bi)) {
      bv = v;
      bi = i;
    }
  };
  // An id's place among the block's, or -1.
  auto place = [&](int32_t id) -> int {
    const uint32_t t = (uint32_t)id + (uint32_t)shift, run = t / kRun;
    const bool ours = (uint32_t)id < (uint32_t)a.vocab && (run & (ranks - 1)) == rank;
    return ours ? (int)((run >> log_ranks) * kRun + t % kRun) : -1;
  };
  // The row's tokens from i0 on f(id, kSeen or 0, 0) and biases from entry b0 on
  // f(id, 0, 1 + entry), whole warps at a time (id -1: none).
  const int warp_at = tid & ~31;
  auto rest_of_row = [&](int i0, int b0, auto&& f) {
#pragma unroll 1
    for (int i = i0 + warp_at; i < hist; i += kThreads)
      f(i + lane < hist ? said[i + lane] : -1, i + lane < prompt ? kSeen : 0u, 0u);
#pragma unroll 1
    for (int e = e0 + b0 + warp_at; e < e1; e += kThreads)
      f(e + lane < e1 ? c.bias_ids[e + lane] : -1, 0u, (uint32_t)(e + lane - e0 + 1));
  };
  // The pass: a thread's next kAhead groups are always on their way, to its own
  // slots of the ring (long slices) or to registers (kDepth 0), the first ones
  // while the row's tokens are listed and sorted. With four slots 64 rows of
  // 152064 take 23.5 us, with registers for two 25.6; 128 of 151936 36.6 and 38.9;
  // 333 of 32003 29.7 and 33.8. Of few groups the ring's extra steps cost more than
  // its depth gives: 16 rows of 151936 (9 groups a thread) 11.9 and 11.3 us.
  constexpr int kAhead = kDepth > 0 ? kDepth : kUnroll;
  static_assert(4 * kThreads % kRun == 0 && kAhead % kUnroll == 0);
  const int far = (4 * kThreads) << log_ranks;  // ids from a thread's group to its next
  float4 v[kUnroll];
  auto fetch = [&](int at, int l, int i, int n) {
    const bool in = l < n && (uint32_t)i < whole;
    if constexpr (kDepth > 0) {
      if (in) cp_async16(smem_u32(ring + at * kThreads), x + i, true);
      cp_commit();
    } else {
      if (in) v[at] = *reinterpret_cast<const float4*>(x + i);
    }
  };
  auto fetch_first = [&](int base, int n) {
    const int i0 = id_at(base + 4 * tid);
#pragma unroll
    for (int t = 0; t < kAhead; ++t) fetch(t, 4 * (tid + t * kThreads), i0 + t * far, n);
  };
  fetch_first(0, min(a.chunk, places));

  bool hashed = true;
  if (touched) {
    __syncthreads();
    auto note = [&](int32_t id, uint32_t flag, uint32_t e) {
      const int l = place(id);
      const uint32_t who = __ballot_sync(0xffffffffu, l >= 0);
      if (who == 0) return;
      int at = 0;
      if (lane == 0) at = atomicAdd(&listed, __popc(who));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
      if (l >= 0 && at < a.room) list[at] = make_uint2((uint32_t)l | flag, e);
    };
#pragma unroll
    for (int k = 0; k < kEarly; ++k) {
      const int i = tid + k * kThreads;
      if (k * kThreads < hist) note(i < hist ? early[k] : -1, i < prompt ? kSeen : 0u, 0u);
    }
    if (e1 > e0) note(early_bias, 0u, (uint32_t)(tid + 1));
    rest_of_row(kEarly * kThreads, kThreads, note);
    __syncthreads();
    hashed = listed <= a.room;
  }
  const int step = logit_step(hashed, a.chunk, (int)slots);
#pragma unroll 1
  for (int base = 0; base < places; base += step) {
    const int n = min(step, places - base);
    if (base > 0) {
      __syncthreads();
      fetch_first(base, n);
    }
    if (mask) {
      // the mask's words of each run, from the one with its first id on; that id
      // is the word's bit -shift % 32 in every run
      const int all = (a.vocab + 31) / 32;
#pragma unroll 1
      for (int k = tid; k < n / kRun * 8; k += kThreads) {  // eight threads a run
        const int at = k & 7, w = (id_at(base + (k >> 3) * kRun) >> 5) + at;  // -1: before the row
        const bool in = (uint32_t)w < (uint32_t)all;
        if (at < kRunWords)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                           smem_u32(mask_s + (k >> 3) * kRunWords + at)),
                       "l"(mask + (in ? w : 0)), "r"(in ? 4 : 0)
                       : "memory");
      }
    }
    if (touched) {
      if (base > 0) {
        clear_tables();
        __syncthreads();
      }
      // a token (kSeen or 0: of the prompt or the output) or a bias entry of place
      // l, or none (l from n on); a whole warp at a time
      auto enter = [&](uint32_t l, uint32_t flag, uint32_t e) {
        uint32_t h = 0;
        bool fresh_slot = false;
        if (l < (uint32_t)n) {
          h = hashed ? __umulhi(l * 2654435761u, slots) : l;
          for (;;) {
            const uint32_t was = atomicCAS(&key[h], kNoId, l);
            fresh_slot = was == kNoId;
            if (fresh_slot || was == l) break;
            if (++h == slots) h = 0;
          }
          // the last entry of an id counts: entries leave their number, the largest stays
          if (e) atomicMax(&bias[h], e);
          else if (flag) atomicOr(&word[h], kSeen);
          else atomicAdd(&word[h], 1u);
          if (fresh_slot) atomicOr(&bits[l >> 5], 1u << (l & 31));
        }
        const uint32_t who = __ballot_sync(0xffffffffu, fresh_slot);
        if (who == 0) return;
        int at = 0;
        if (lane == 0) at = atomicAdd(&in_use, __popc(who));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
        if (fresh_slot) used[at] = (uint16_t)h;
      };
      if (hashed) {
#pragma unroll 1
        for (int k = warp_at; k < listed; k += kThreads) {
          const uint2 t = k + lane < listed ? list[k + lane] : make_uint2(kNoId, 0u);
          enter(t.x == kNoId ? kNoId : (t.x & ~kSeen) - (uint32_t)base, t.x & kSeen, t.y);
        }
      } else {
        rest_of_row(0, 0, [&](int32_t id, uint32_t flag, uint32_t e) {
          const int l = place(id);
          enter(l >= base ? (uint32_t)(l - base) : kNoId, flag, e);
        });
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (touched || mask) __syncthreads();
    // the mask's bits from place l on, at least four of them
    const int lead = -shift & 31;
    auto allowed = [&](int l) -> uint32_t {
      const int at = (l & (kRun - 1)) + lead;
      const uint32_t* w = mask_s + l / kRun * kRunWords + (at >> 5);
      return __funnelshift_r(w[0], w[1], at & 31);  // a run's last word is not needed at its end
    };

    // A warp's groups are one run of ids, so a thread's place in its run, and with
    // it the bits' position in their words, is the same in all its groups.
    static_assert(kRun == 4 * 32);
    int i = id_at(base + 4 * tid);
    const uint32_t* bits_at = bits + (tid >> 3);
    const uint32_t* mask_at = mask_s + (tid >> 5) * kRunWords + ((4 * lane + lead) >> 5);
    const int bit = 4 * tid & 31, mask_bit = (4 * lane + lead) & 31;
    int slot = 0;
#pragma unroll 1
    for (int l0 = 4 * tid; l0 < n; l0 += 4 * kUnroll * kThreads) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int l = l0 + 4 * k * kThreads;
        if (k > 0 && l >= n) break;
        float4 now;
        if constexpr (kDepth > 0) {
          cp_wait<kDepth - 1>();
          now = ring[(slot + k) * kThreads];
        } else {
          now = v[k];
          fetch(k, l + 4 * kAhead * kThreads, i + kAhead * far, n);
        }
        const uint32_t b4 = touched ? bits_at[k * (kThreads / 8)] >> bit & 15u : 0u;
        if ((uint32_t)i < whole) {
          float r[4] = {now.x, now.y, now.z, now.w};
          if (mask) {
            const uint32_t* w = mask_at + k * (kThreads / 32 * kRunWords);
            const uint32_t m = __funnelshift_r(w[0], w[1], mask_bit);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (!(m >> j & 1u)) r[j] = -INFINITY;
          }
          if (y) {
            if (together) {
              *reinterpret_cast<float4*>(y + i) = make_float4(r[0], r[1], r[2], r[3]);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) y[i + j] = r[j];
            }
          }
          if (b4) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (b4 >> j & 1u) r[j] = -INFINITY;
          }
          const float top = fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));  // NaN is passed over
          if (ids && top > gv) {
            gv = top;
            gi = i;
#pragma unroll
            for (int j = 0; j < 4; ++j) group[j] = r[j];
          }
        } else {  // the group reaches over the row's ends, or lies behind it
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            const int id = i + j;
            if ((uint32_t)id >= (uint32_t)a.vocab) continue;
            float r = x[id];
            if (mask && !(allowed(l + j) & 1u)) r = -INFINITY;
            if (y) y[id] = r;
            if (!(b4 >> j & 1u)) take(r, id);
          }
        }
        if constexpr (kDepth > 0)  // into the slot that has been read
          fetch(slot + k, l + 4 * kAhead * kThreads, i + kAhead * far, n);
        i += far;
      }
      slot = slot + kUnroll < kAhead ? slot + kUnroll : 0;
      bits_at += kUnroll * (kThreads / 8);
      mask_at += kUnroll * (kThreads / 32 * kRunWords);
    }
    if (!touched) continue;
    __syncthreads();
    // the touched ids, over what the pass wrote (an id that the mask takes out
    // is -inf whatever it was, any other still holds its logit)
#pragma unroll 2
    for (int k = tid; k < in_use; k += kThreads) {
      const int h = used[k], l = (int)key[h], i = id_at(base + l);
      float r = x[i];
      const uint32_t w = word[h], e = bias[h];
      if (w) r = penalised(r, w, rep, freq, pres, c.repetition != nullptr);
      if (e) r = __fadd_rn(r, c.bias_vals[e0 + e - 1]);
      if (mask && !(allowed(l) & 1u)) r = -INFINITY;
      if (y) y[i] = r;
      take(r, i);
    }
  }
  if (!ids) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (gv > -INFINITY && group[j] == gv) take(gv, gi + j);
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

template <int kThreads, int kDepth, int kUnroll>
cudaError_t launch_controls(LogitArgs a, size_t rows, int cluster, cudaStream_t st) {
  const bool pen = a.c.history && (a.c.repetition || a.c.frequency || a.c.presence);
  const LogitPlan p = logit_plan(kThreads, kDepth, cluster, a.vocab, rows,
                                 pen ? a.c.history_width : 0, a.c.bias_starts != nullptr,
                                 a.c.num_bias, a.c.mask != nullptr);
  a.chunk = p.chunk;
  a.slots = p.slots;
  a.room = p.room;
  static std::atomic<uint64_t> raised{0};
  const cudaError_t e = raise_smem_limit((const void*)k_logit_controls<kThreads, kDepth, kUnroll>,
                                         logit_smem(kMaxChunk, kMostRoom, true, kThreads, kDepth),
                                         &raised);
  if (e != cudaSuccess) return e;
  return counted(launch_pdl(k_logit_controls<kThreads, kDepth, kUnroll>,
                            dim3((unsigned)(rows * cluster)), kThreads, p.smem, st, cluster, a));
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
    if (c->history && (c->history_width > 0x40000000 || c->history_stride < c->history_width ||
                       c->history_stride > ((uint64_t)1 << 40)))
      return MYOS_ERR_SHAPE;
    if (c->num_bias > 0x40000000) return MYOS_ERR_SHAPE;
    // a block counts the entries of its list in 31 bits
    if (c->bias_starts && (c->repetition || c->frequency || c->presence) &&
        c->history_width + c->num_bias > 0x7fffffff)
      return MYOS_ERR_SHAPE;
    if (c->mask && (c->mask_stride < (vocab + 31) / 32 || c->mask_stride > ((uint64_t)1 << 40) ||
                    c->num_masks > 0x7fffffff || (!c->mask_rows && c->num_masks < rows)))
      return MYOS_ERR_SHAPE;
    a.c = *c;
  }
  // Few rows: larger blocks, as long as their clusters are placed at once, a
  // block to a multiprocessor (with 16 rows of 151936 they are not: 17.4 us, in
  // blocks of 512 12.1, before the pass's later steps). 12 rows take 8.6 us with one
  // group a thread and turn, with two 8.9.
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (rows * kMaxCluster <= (size_t)sm_count() * 2 / 3) {
    e = launch_controls<1024, 0, 1>(a, rows, logit_cluster(rows, a.vocab, 1024, sm_count()), st);
  } else {
    const int cluster = logit_cluster(rows, a.vocab, 512, sm_count());
    e = a.vocab / cluster >= 12 * 4 * 512 ? launch_controls<512, 4, 2>(a, rows, cluster, st)
                                          : launch_controls<512, 0, 2>(a, rows, cluster, st);
  }
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}
