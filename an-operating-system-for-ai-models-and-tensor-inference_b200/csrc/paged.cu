// Serving over a paged KV cache: block tables and slot maps from request
// lengths, and the pass that norms, rotates and stores q, k and v.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace myos {

int paged_check(const myos_paged_kv* kv) {
  if (!kv || !kv->k || !kv->v) return MYOS_ERR_ARG;
  if (kv->kv_dtype != MYOS_KV_F32 && kv->kv_dtype != MYOS_KV_BF16) return MYOS_ERR_ARG;
  if (kv->reserved != 0) return MYOS_ERR_ARG;
  if (kv->num_pages == 0 || kv->num_pages > 0x7fffffffu || kv->page_size == 0 ||
      kv->page_size > 65536 || kv->num_kv_heads == 0 || kv->num_kv_heads > 65535 ||
      kv->head_dim == 0 || kv->head_dim % 8 != 0 || kv->head_dim > 256)
    return MYOS_ERR_SHAPE;
  if (kv->slot_stride < kv->head_dim || kv->head_stride < kv->head_dim ||
      kv->page_stride < kv->head_dim)
    return MYOS_ERR_SHAPE;
  // every element offset fits 62 bits
  const uint64_t most = (uint64_t)1 << 60;
  uint64_t pages, heads, slots;
  if (__builtin_mul_overflow(kv->page_stride, (uint64_t)kv->num_pages, &pages) ||
      __builtin_mul_overflow(kv->head_stride, (uint64_t)kv->num_kv_heads, &heads) ||
      __builtin_mul_overflow(kv->slot_stride, (uint64_t)kv->page_size, &slots) || pages > most ||
      heads > most || slots > most)
    return MYOS_ERR_SHAPE;
  const uint64_t per16 = kv->kv_dtype == MYOS_KV_F32 ? 4 : 8;
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || kv->page_stride % per16 != 0 ||
      kv->head_stride % per16 != 0 || kv->slot_stride % per16 != 0)
    return MYOS_ERR_ARG;
  return MYOS_OK;
}

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

namespace {

// ------------------------------------------------------------------ tables
// Every block runs the prefix sums over all requests itself (8 bytes a request
// from L2), so one launch with no meeting of the blocks does the whole step:
// block i then writes the table entries and rows of its share. A request of one
// or two rows (decode) is written by the thread that scanned it, which has
// looked its last page up meanwhile; the rows of longer ones find their request
// by a binary search. What is left is latency: two loads on one another
// (lengths, then pages), one barrier, the stores. A new page's first slot is a
// row of the step, and that row writes the page's table entry.
struct TablesArgs {
  int32_t* table;
  int64_t table_stride;
  int max_blocks;
  const int32_t *ctx, *add;
  int nseq;
  const int32_t* free_pages;
  int free_cap;
  const int32_t* num_free;
  uint32_t page_size, num_pages;
  int64_t* slots;
  int32_t *positions, *row_seq;
  int max_rows;
  int32_t *kv_lens, *seq_starts, *result;
};

struct Sums {
  int64_t rows, pages;
};
MYOS_DEV Sums warp_scan(Sums v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t r = __shfl_up_sync(0xffffffffu, v.rows, o);
    const int64_t p = __shfl_up_sync(0xffffffffu, v.pages, o);
    if (lane >= o) {
      v.rows += r;
      v.pages += p;
    }
  }
  return v;
}

constexpr int kSmall = 2;  // rows that a request's thread writes itself
constexpr uint32_t kLong = 0x80000000u;

// A request: its first row, the pages taken by the requests before it (-1: it is
// refused), and its length, with kLong where its rows are not written yet.
struct Span {
  int start, first;
  uint32_t ctx;
};
MYOS_DEV uint32_t ceil_div(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

__global__ void __launch_bounds__(1024) k_paged_tables(const TablesArgs a) {
  extern __shared__ Span spans[];
  __shared__ Sums parts[2][32];
  __shared__ int64_t taken_s[32];
  __shared__ int refused_s[32];
  const uint32_t P = a.page_size;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  pdl_launch();
  pdl_wait();
  const int nfree = min(max(*a.num_free, 0), a.free_cap);
  const int64_t room = min((int64_t)a.max_blocks * P, (int64_t)0x7fffffff);  // lengths are int32
  Sums before = {0, 0};  // of the requests of earlier rounds
  int64_t taken = 0;
  int refused = 0, longer = 0;
  // the page of a position of a request with `held` pages and `first` taken before
  auto page_of = [&](int b, uint32_t pg, uint32_t held, int first) -> int32_t {
    return pg < held ? a.table[b * a.table_stride + pg]
                     : a.free_pages[nfree - 1 - first - (int)(pg - held)];
  };
  auto row = [&](int r, int b, uint32_t pos, uint32_t in, int32_t page) {
    a.slots[r] = page >= 0 && (uint32_t)page < a.num_pages ? (int64_t)page * P + in : -1;
    a.positions[r] = (int32_t)pos;
    a.row_seq[r] = b;
  };
#pragma unroll 1
  for (int base = 0, round = 0; base < a.nseq; base += blockDim.x, ++round) {
    const int b = base + threadIdx.x;
    const bool mine = b % (int)(gridDim.x * 32) / 32 == (int)blockIdx.x;  // 32 in turn
    uint32_t ctx = 0, add = 0;
    if (b < a.nseq) {
      ctx = max(a.ctx[b], 0);
      add = max(a.add[b], 0);
    }
    // lengths are below 2^31, their sum below 2^32
    const uint32_t held = ceil_div(ctx, P), all = ceil_div(ctx + add, P);
    const bool fits = (int64_t)ctx + add <= room;
    // the page that a decode row goes to, on its way during the scan
    const bool look = mine && fits && add > 0 && add <= kSmall && ctx % P != 0;
    const int32_t last = look ? a.table[b * a.table_stride + ctx / P] : -1;
    // A request that the row buffer has no room for is behind every admitted one
    // (the rows only grow), so its need may stand in the sum.
    const uint32_t need = add > 0 && fits ? all - held : 0;
    const Sums own = {(int64_t)add, (int64_t)need};
    Sums s = warp_scan(own);
    if (lane == 31) parts[round & 1][warp] = s;
    __syncthreads();
    const Sums upto = warp_scan(lane < nwarps ? parts[round & 1][lane] : Sums{0, 0});
    s.rows += before.rows + (warp ? __shfl_sync(0xffffffffu, upto.rows, max(warp, 1) - 1) : 0);
    s.pages += before.pages + (warp ? __shfl_sync(0xffffffffu, upto.pages, max(warp, 1) - 1) : 0);
    before.rows += __shfl_sync(0xffffffffu, upto.rows, 31);
    before.pages += __shfl_sync(0xffffffffu, upto.pages, 31);
    if (b >= a.nseq) continue;
    const int end = (int)min(s.rows, (int64_t)a.max_rows);
    const int start = (int)min(s.rows - own.rows, (int64_t)a.max_rows);
    const bool ok = add == 0 || (fits && s.rows <= a.max_rows && (need == 0 || s.pages <= nfree));
    const int first = ok ? (int)min(s.pages - own.pages, (int64_t)nfree) : -1;
    if (ok && need > 0) taken = s.pages;  // a later request's is larger
    refused += !ok;
    spans[b] = Span{start, first, ctx | (add > kSmall ? kLong : 0u)};
    longer |= add > kSmall;
    if (!mine) continue;
    a.kv_lens[b] = (int32_t)(ok ? ctx + add : ctx);
    a.seq_starts[b + 1] = end;
    if (b == 0) a.seq_starts[0] = 0;
    if (add == 0 || add > kSmall) continue;
#pragma unroll 1
    for (int r = start; r < end; ++r) {
      if (!ok) {
        row(r, b, 0, 0, -1);
        continue;
      }
      const uint32_t pos = ctx + (r - start), pg = pos / P, in = pos - pg * P;
      const int32_t page = look && pg == ctx / P ? last : page_of(b, pg, held, first);
      if (pg >= held && in == 0) a.table[b * a.table_stride + pg] = page;
      row(r, b, pos, in, page);
    }
  }
  if (blockIdx.x == 0) {
    // the admitted requests' running sum is largest at the last of them
    for (int o = 16; o > 0; o >>= 1) {
      taken = max(taken, __shfl_xor_sync(0xffffffffu, taken, o));
      refused += __shfl_xor_sync(0xffffffffu, refused, o);
    }
    if (lane == 0) {
      taken_s[warp] = taken;
      refused_s[warp] = refused;
    }
  }
  longer = __syncthreads_or(longer);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    for (int w = 1; w < nwarps; ++w) {
      taken = max(taken, taken_s[w]);
      refused += refused_s[w];
    }
    a.result[0] = (int32_t)(nfree - taken);
    a.result[1] = refused;
  }
  const int rows = (int)min(before.rows, (int64_t)a.max_rows);
  if (longer) {
    // rows: of the last request that begins at or before the row (a step past 2^31
    // rows is still below 2^32)
#pragma unroll 2
    for (uint32_t r = blockIdx.x * blockDim.x + threadIdx.x; r < (uint32_t)rows;
         r += gridDim.x * blockDim.x) {
      int lo = 0, hi = a.nseq;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((uint32_t)spans[mid].start <= r) lo = mid;
        else hi = mid;
      }
      const Span sp = spans[lo];
      if (!(sp.ctx & kLong)) continue;
      const uint32_t ctx = sp.ctx & ~kLong, pos = ctx + (r - sp.start), pg = pos / P;
      if (sp.first < 0) {
        row((int)r, lo, 0, 0, -1);
        continue;
      }
      const uint32_t held = ceil_div(ctx, P), in = pos - pg * P;
      const int32_t page = page_of(lo, pg, held, sp.first);
      if (pg >= held && in == 0) a.table[lo * a.table_stride + pg] = page;
      row((int)r, lo, pos, in, page);
    }
  }
  // rows behind the last request's
  for (int64_t r = (int64_t)rows + blockIdx.x * blockDim.x + threadIdx.x; r < a.max_rows;
       r += gridDim.x * blockDim.x)
    row((int)r, -1, 0, 0, -1);
}

// ------------------------------------------------------- norm, rotate, store
// A head is handled by `1 << lanes_log2` >= d / 8 lanes, each with two chunks
// of four values: chunk j and its rotation partner j + rot / 8, or (behind the
// rotated part) two neighbouring chunks. A block takes a row at a time, so a
// lane's cosines and sines serve all the heads it comes to, and its loads of
// kHeads heads are in flight together; of few rows, several blocks take one.
// Bound by memory: 16001 rows of 40/8 heads of 128 with norms into a bf16 cache
// (860 MB) take 139 us, 6.2 TB/s, 0.94 of a copy. Its 63 registers a thread let 8
// blocks of 128 reside; the grid is twice that, 16 a multiprocessor (14: 148 us,
// 32: 142 us; blocks of 256: 147 us). Registers capped for 10 or 12 resident
// blocks: 154 and 187 us; a row's position loaded in its own turn: 156 us; 4
// heads in flight: 167 us.
struct StoreArgs {
  float* q;
  const float* qkv;
  int64_t q_stride, qkv_stride, rows;
  const uint16_t *q_gamma, *k_gamma;
  float eps;
  const float *cos_t, *sin_t;
  int64_t num_pos;
  const int32_t* positions;
  const int64_t* slots;
  int hq, rot, lanes_log2;
};

MYOS_DEV void put4(float* p, const float4& v) { *reinterpret_cast<float4*>(p) = v; }
// bf16 cache: round to nearest even, at most half a step (2^-9 of the value's
// binade) off the f32 value; the cache type asks for it.
MYOS_DEV void put4(__nv_bfloat16* p, const float4& v) {
  __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
  uint2 u;
  u.x = *reinterpret_cast<uint32_t*>(&lo);
  u.y = *reinterpret_cast<uint32_t*>(&hi);
  *reinterpret_cast<uint2*>(p) = u;
}

MYOS_DEV float sq4(const float4& v) { return v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w; }

MYOS_DEV float4 scale4(const float4& v, float inv, const uint16_t* g) {
  const uint2 u = *reinterpret_cast<const uint2*>(g);
  float4 r;
  r.x = __fmul_rn(bf16_lo(u.x), __fmul_rn(v.x, inv));
  r.y = __fmul_rn(bf16_hi(u.x), __fmul_rn(v.y, inv));
  r.z = __fmul_rn(bf16_lo(u.y), __fmul_rn(v.z, inv));
  r.w = __fmul_rn(bf16_hi(u.y), __fmul_rn(v.w, inv));
  return r;
}

MYOS_DEV float rot_lo(float x, float y, float c, float s) {
  return __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
}
MYOS_DEV float rot_hi(float x, float y, float c, float s) {
  return __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
}

constexpr int kStoreThreads = 128;

template <class KT, int kHeads>
__global__ void __launch_bounds__(kStoreThreads) k_paged_store(const StoreArgs a, const PagedKv<KT> kv) {
  const int lanes = 1 << a.lanes_log2, d = (int)kv.d, hk = (int)kv.heads, heads = a.hq + 2 * hk;
  const int j = threadIdx.x & (lanes - 1), per = kStoreThreads >> a.lanes_log2;
  const int step = per * gridDim.y, begin = per * blockIdx.y + (threadIdx.x >> a.lanes_log2);
  const bool on = j < d / 8;
  const int pairs = a.rot / 8;
  const bool turn = j < pairs;
  const int c0 = 4 * (turn ? j : 2 * pairs + 2 * (j - pairs));
  const int c1 = turn ? c0 + 4 * pairs : c0 + 4;
  const bool norm = a.q_gamma || a.k_gamma;
  pdl_launch();
  pdl_wait();
  // a row's slot and position are loaded a row ahead: its cosines need them first
  int64_t next_slot = a.slots[blockIdx.x];
  int next_pos = a.rot > 0 ? a.positions[blockIdx.x] : 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* src = a.qkv + row * a.qkv_stride;
    const int64_t slot = next_slot, pos = next_pos;
    if (row + gridDim.x < a.rows) {
      next_slot = a.slots[row + gridDim.x];
      if (a.rot > 0) next_pos = a.positions[row + gridDim.x];
    }
    float4 cs = make_float4(0.f, 0.f, 0.f, 0.f), sn = cs;
    bool placed = true;
    if (a.rot > 0) {
      placed = pos >= 0 && pos < a.num_pos;
      if (placed && turn && on) {
        cs = *reinterpret_cast<const float4*>(a.cos_t + pos * (a.rot / 2) + c0);
        sn = *reinterpret_cast<const float4*>(a.sin_t + pos * (a.rot / 2) + c0);
      }
    }
    const bool stored = placed && slot >= 0 && slot < (int64_t)kv.num_pages * kv.page_size;
    const int64_t page = stored ? slot / kv.page_size : 0;
    const int64_t at = page * kv.page_stride + (slot - page * kv.page_size) * kv.slot_stride;
    // every lane of a warp goes through the shuffles, with or without a head
    for (int h0 = begin; h0 - begin % per < heads; h0 += kHeads * step) {
      float4 x[kHeads], y[kHeads];
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = h0 + u * step;
        x[u] = y[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on && h < heads) {
          x[u] = *reinterpret_cast<const float4*>(src + h * d + c0);
          y[u] = *reinterpret_cast<const float4*>(src + h * d + c1);
        }
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = h0 + u * step;
        const bool is_q = h < a.hq, is_v = h >= a.hq + hk;
        if (norm) {
          float ss = sq4(x[u]) + sq4(y[u]);
          for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const uint16_t* gamma = is_q ? a.q_gamma : is_v ? nullptr : a.k_gamma;
          if (on && h < heads && gamma) {
            const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)d), a.eps)));
            x[u] = scale4(x[u], inv, gamma + c0);
            y[u] = scale4(y[u], inv, gamma + c1);
          }
        }
        if (!on || h >= heads) continue;
        if (turn && !is_v) {
          const float4 p = x[u], r = y[u];
          x[u].x = rot_lo(p.x, r.x, cs.x, sn.x);
          x[u].y = rot_lo(p.y, r.y, cs.y, sn.y);
          x[u].z = rot_lo(p.z, r.z, cs.z, sn.z);
          x[u].w = rot_lo(p.w, r.w, cs.w, sn.w);
          y[u].x = rot_hi(p.x, r.x, cs.x, sn.x);
          y[u].y = rot_hi(p.y, r.y, cs.y, sn.y);
          y[u].z = rot_hi(p.z, r.z, cs.z, sn.z);
          y[u].w = rot_hi(p.w, r.w, cs.w, sn.w);
        }
        if (is_q) {
          float* dst = a.q + row * a.q_stride + h * d;
          if (!placed) {
            const float n = __int_as_float(0x7fc00000);
            x[u] = y[u] = make_float4(n, n, n, n);
          }
          put4(dst + c0, x[u]);
          put4(dst + c1, y[u]);
        } else if (stored) {
          KT* dst = is_v ? kv.v + at + (h - a.hq - hk) * kv.head_stride
                         : kv.k + at + (h - a.hq) * kv.head_stride;
          put4(dst + c0, x[u]);
          put4(dst + c1, y[u]);
        }
      }
    }
  }
}

template <class KT>
cudaError_t launch_store(const StoreArgs& a, const myos_paged_kv* kv, cudaStream_t st) {
  constexpr int kResident = 16;  // blocks a multiprocessor
  const int64_t most = (int64_t)sm_count() * kResident;
  const int per = kStoreThreads >> a.lanes_log2;
  const int parts = (a.hq + 2 * (int)kv->num_kv_heads + per - 1) / per;
  dim3 grid((unsigned)(a.rows < most ? a.rows : most));
  while ((int)grid.y < parts && grid.x * (grid.y + 1) <= most / 2) ++grid.y;
  return counted(
      launch_pdl(k_paged_store<KT, 2>, grid, kStoreThreads, 0, st, 1, a, paged_view<KT>(kv)));
}

}  // namespace
}  // namespace myos

using namespace myos;

extern "C" {

int myos_dev_paged_tables(int32_t* d_block_table, size_t table_stride, size_t max_blocks,
                          const int32_t* d_ctx_lens, const int32_t* d_new_lens, size_t nseq,
                          const int32_t* d_free_pages, size_t free_cap,
                          const int32_t* d_num_free, uint32_t page_size, uint32_t num_pages,
                          int64_t* d_slots, int32_t* d_positions, int32_t* d_row_seq,
                          size_t max_rows, int32_t* d_kv_lens, int32_t* d_seq_starts,
                          int32_t* d_result, void* stream) {
  if (nseq == 0) return MYOS_OK;
  if (!d_block_table || !d_ctx_lens || !d_new_lens || (!d_free_pages && free_cap > 0) ||
      !d_num_free || (max_rows > 0 && (!d_slots || !d_positions || !d_row_seq)) || !d_kv_lens ||
      !d_seq_starts || !d_result)
    return MYOS_ERR_ARG;
  const uintptr_t words = (uintptr_t)d_block_table | (uintptr_t)d_ctx_lens |
                          (uintptr_t)d_new_lens | (uintptr_t)d_free_pages |
                          (uintptr_t)d_num_free | (uintptr_t)d_positions | (uintptr_t)d_row_seq |
                          (uintptr_t)d_kv_lens | (uintptr_t)d_seq_starts | (uintptr_t)d_result;
  if ((words & 3) != 0 || !aligned(d_slots, 8)) return MYOS_ERR_ARG;
  if (d_kv_lens == d_ctx_lens || d_kv_lens == d_new_lens || d_result == d_num_free ||
      d_result + 1 == d_num_free)
    return MYOS_ERR_ARG;
  if (nseq > 16384 || page_size == 0 || page_size > 65536 || num_pages > 0x7fffffffu ||
      max_blocks == 0 || max_blocks > 0x7fffffff || table_stride < max_blocks ||
      table_stride > ((size_t)1 << 40) || max_rows > 0x7fffffff || free_cap > 0x7fffffff)
    return MYOS_ERR_SHAPE;
  const size_t smem = sizeof(Span) * nseq;
  static std::atomic<uint64_t> raised{0};
  // 48 KB unless it is raised, the kernel's own shared memory (1.4 KB) included
  if (smem > 40 * 1024 &&
      raise_smem_limit((const void*)k_paged_tables, sizeof(Span) * 16384, &raised) != cudaSuccess)
    return MYOS_ERR_CUDA;
  TablesArgs a;
  a.table = d_block_table;
  a.table_stride = (int64_t)table_stride;
  a.max_blocks = (int)max_blocks;
  a.ctx = d_ctx_lens;
  a.add = d_new_lens;
  a.nseq = (int)nseq;
  a.free_pages = d_free_pages;
  a.free_cap = (int)free_cap;
  a.num_free = d_num_free;
  a.page_size = page_size;
  a.num_pages = num_pages;
  a.slots = d_slots;
  a.positions = d_positions;
  a.row_seq = d_row_seq;
  a.max_rows = (int)max_rows;
  a.kv_lens = d_kv_lens;
  a.seq_starts = d_seq_starts;
  a.result = d_result;
  // a small batch in small blocks: the barrier waits for fewer warps
  const int threads = nseq <= 32 && max_rows <= 64 ? 32 : nseq <= 256 && max_rows <= 4096 ? 256 : 1024;
  size_t grid = ((max_rows > nseq ? max_rows : nseq) + threads - 1) / threads;
  if (grid > (size_t)sm_count()) grid = sm_count();
  const cudaError_t e =
      launch_pdl(k_paged_tables, dim3((unsigned)grid), threads, smem, (cudaStream_t)stream, 1, a);
  return counted(e) == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}

int myos_dev_qk_norm_rope_store(float* d_q, size_t q_stride, const float* d_qkv,
                                size_t qkv_stride, size_t rows, size_t num_q_heads,
                                const myos_paged_kv* kv, const void* d_q_gamma,
                                const void* d_k_gamma, float eps, const float* d_cos,
                                const float* d_sin, size_t num_pos, size_t rot_dim,
                                const int32_t* d_positions, const int64_t* d_slots,
                                void* stream) {
  if (int st = paged_check(kv)) return st;
  if (rows == 0) return MYOS_OK;
  if (!d_q || !d_qkv || !d_slots || (rot_dim > 0 && (!d_cos || !d_sin || !d_positions)))
    return MYOS_ERR_ARG;
  const size_t d = kv->head_dim;
  if (num_q_heads == 0 || num_q_heads > 65535 || rot_dim % 8 != 0 || rot_dim > d ||
      rows > 0x7fffffff || num_pos > 0x7fffffff || (rot_dim > 0 && num_pos == 0) ||
      q_stride < num_q_heads * d || qkv_stride < (num_q_heads + 2 * (size_t)kv->num_kv_heads) * d ||
      q_stride > ((size_t)1 << 30) || qkv_stride > ((size_t)1 << 30))
    return MYOS_ERR_SHAPE;
  if (!aligned(d_q, 16) || !aligned(d_qkv, 16) || q_stride % 4 != 0 || qkv_stride % 4 != 0 ||
      !aligned(d_q_gamma, 8) || !aligned(d_k_gamma, 8) || !aligned(d_slots, 8))
    return MYOS_ERR_ARG;
  if (rot_dim > 0 && (!aligned(d_cos, 16) || !aligned(d_sin, 16) || !aligned(d_positions, 4)))
    return MYOS_ERR_ARG;
  if (d_q == d_qkv && rows > 1 && q_stride != qkv_stride) return MYOS_ERR_ARG;
  StoreArgs a;
  a.q = d_q;
  a.qkv = d_qkv;
  a.q_stride = (int64_t)q_stride;
  a.qkv_stride = (int64_t)qkv_stride;
  a.rows = (int64_t)rows;
  a.q_gamma = static_cast<const uint16_t*>(d_q_gamma);
  a.k_gamma = static_cast<const uint16_t*>(d_k_gamma);
  a.eps = eps;
  a.cos_t = d_cos;
  a.sin_t = d_sin;
  a.num_pos = (int64_t)num_pos;
  a.positions = d_positions;
  a.slots = d_slots;
  a.hq = (int)num_q_heads;
  a.rot = (int)rot_dim;
  a.lanes_log2 = 0;
  while ((8u << a.lanes_log2) < d) ++a.lanes_log2;
  const cudaError_t e = kv->kv_dtype == MYOS_KV_F32
                            ? launch_store<float>(a, kv, (cudaStream_t)stream)
                            : launch_store<__nv_bfloat16>(a, kv, (cudaStream_t)stream);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}

// rope.rs:186-194, one row per position: libm in f32, each step rounded.
int myos_rope_table(float* cos_out, float* sin_out, size_t num_pos, size_t rot_dim, float theta) {
  if (!cos_out || !sin_out) return MYOS_ERR_ARG;
  if (rot_dim == 0 || rot_dim % 2 != 0 || rot_dim > 65536 || num_pos > 0x7fffffff)
    return MYOS_ERR_SHAPE;
  const size_t half = rot_dim / 2;
  for (size_t i = 0; i < half; ++i) {
    volatile float exponent = (float)(2 * i) / (float)rot_dim;
    volatile float inv = 1.0f / powf(theta, exponent);
    for (size_t p = 0; p < num_pos; ++p) {
      volatile float angle = (float)p * inv;
      cos_out[p * half + i] = cosf(angle);
      sin_out[p * half + i] = sinf(angle);
    }
  }
  return MYOS_OK;
}

}  // extern "C"
