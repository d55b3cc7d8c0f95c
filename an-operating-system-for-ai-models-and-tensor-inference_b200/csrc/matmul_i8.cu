// The product of 8-bit rows and 8-bit channels with a scale each
// (include/myos_cuda.h, "Projections in 8-bit integers"): out[r][c] =
// (sum_i a[r][i] w[c][i]) a_scales[r] w_scales[c] + bias[c].
//
// The sum is exact in 32-bit integers, so it may be split and joined in any order
// and gives the same bits. Two kernels:
//
// k_few_i8, up to 16 rows: the weights' memory bounds it. mma.sync straight from
// global memory, blocks of 8 to 32 channels, its warps sharing k (1 x 1536 x 151936:
// 37.5 us, 6.2 TB/s, 0.95 of the copy rate; 1 x 1536 x 2048: 2.2 us).
//
// k_matmul_i8, tiles on tcgen05: 128 channels (the tensor core's M, the lanes of its
// memory) by up to 256 rows (its N, the columns). A lane holds one channel, so a
// warp's store of one row is 32 channels side by side, and few rows cost nothing but
// their own columns. Six warps: copies (TMA, 128 bytes of k a stage), products
// (tcgen05, 32 bytes of k each), and four that scale and store while the next tile's
// products go into the other half of the tensor memory. From 65 rows on two blocks
// make a tile of 256 channels, each copying half of the rows. Where tiles are few, a
// cluster shares a tile's k and adds its parts through shared memory.
//
// What bounds it: of many rows the tensor cores and the device's power (4097 x 5120 x
// 27648: 345 us cold under the profiler, the tensor pipe busy 91% of the time at full
// clock; 380 to 425 in a row of calls, where the clock falls under the power limit; 8192
// x 8192 x 8192 335 to 346 us, 3.2 x 10^15 operations a second). Of 64 x 13824 x 5120
// (16.9 us) the weights' way to 120 multiprocessors (11 us at the copy rate), a block's
// start and first copy (1.6 us) and the cluster's sums. Of 333 x 5120 x 7168 (15.1 us)
// copies from L2, 29 KB a step and block, 40 steps in 8 us, then 9.5 MB of results at
// once.
#include <cudaTypedefs.h>
#include <math.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "i8_plan.h"
#include "kernels.h"
#include "paged.h"
#include "tcgen05.cuh"

namespace myos {
namespace {

struct MatArgs {
  void* out;
  int64_t out_stride;
  const int8_t* a;
  int64_t a_stride;
  const int8_t* w;
  int64_t w_stride;
  const float* a_scales;
  const float* w_scales;
  const float* bias;
  int rows, k, channels, steps;
  I8Plan plan;
};

__device__ uint32_t g_wait_failed, g_wait_taken;

// Reads and clears at once: what fails meanwhile is the next answer's.
__global__ void k_take_failed() { g_wait_taken = atomicExch(&g_wait_failed, 0u); }

MYOS_DEV float scaled(int sum, float as, float ws, float bias) {
  return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(sum), as), ws), bias);
}
MYOS_DEV void put(float* p, float v) { *p = v; }
MYOS_DEV void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

MYOS_DEV void put4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
MYOS_DEV void put4(__nv_bfloat16* p, const float* v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                            *reinterpret_cast<const uint32_t*>(&b));
}

// Up to 16 rows of one channel. Whole groups without a branch: the loads, products
// and stores of 16 rows overlap (a row at a time they took 95 cycles each).
template <class OT>
MYOS_DEV void store16(OT* o, int64_t stride, const int* v, const float* as, float ws, float bias,
                      int left, bool ok) {
  if (left >= 16 && ok) {
    float a[16];
#pragma unroll
    for (int j = 0; j < 16; j += 4)
      *reinterpret_cast<float4*>(a + j) = *reinterpret_cast<const float4*>(as + j);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      put(o, scaled(v[j], a[j], ws, bias));
      o += stride;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (j < left) put(o, ok ? scaled(v[j], as[j], ws, bias) : __uint_as_float(0x7fc00000u));
      o += stride;
    }
  }
}

constexpr int kThreads = 192;

// A whole warp's wait, its answer one for all lanes; by the clock from the 64th poll on.
MYOS_DEV bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t code) {
  bool ok = false;
  for (int i = 0; i < 64 && !ok; ++i) ok = mbar_try_wait(bar, parity);
  if (!ok) ok = mbar_wait(bar, parity, &g_wait_failed, code);
  return __all_sync(0xffffffffu, ok);
}

// Tile t: its first channel and row.
MYOS_DEV void tile_at(const I8Plan& p, int64_t t, int& c0, int& r0) {
  const int64_t each = (int64_t)p.group * p.tiles_c;
  const int first = (int)(t / each) * p.group, wide = min(p.group, p.tiles_r - first);
  const int64_t in = t % each;
  c0 = (int)(in / wide) * p.tc;
  r0 = (first + (int)(in % wide)) * p.tn;
}

template <class OT, bool PAIR>
__global__ void __launch_bounds__(kThreads)
    k_matmul_i8(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap amap,
                const MatArgs g) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kI8MaxStages], empty[kI8MaxStages], acc_full[2], acc_empty[2];
  __shared__ __align__(16) float as[2][kI8MaxRows];
  __shared__ uint32_t tmem_s;
  __shared__ int peer_dead;  // a wait of a block of the cluster ran out
  uint8_t* const smem = raw + (-smem_u32(raw) & 1023);
  const I8Plan& p = g.plan;
  // The copying and the issuing warp run as a whole, one lane of them acting: the
  // tensor core's operands are registers of the warp, and a single lane's own values
  // would have to be moved there one by one (390 cycles a step).
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const bool acts = one_lane();
  constexpr int kPair = PAIR ? 2 : 1;
  const int tr = p.tn / kPair;  // rows that a block copies
  // rows of a tile that the tensor core takes: of the last one no more than there are
  auto taken = [&](int r0) { return min(p.tn, (g.rows - r0 + 16 * kPair - 1) / (16 * kPair) * (16 * kPair)); };
  const uint32_t stage_bytes = (kI8Channels + tr) * kI8Step;
  const int split = PAIR ? 1 : p.split;
  const int rank = PAIR || split > 1 ? (int)cluster_rank() : 0;
  const int k0 = PAIR ? 0 : (int)((int64_t)g.steps * rank / split);
  const int k1 = PAIR ? g.steps : (int)((int64_t)g.steps * (rank + 1) / split);
  const int64_t tiles = (int64_t)p.tiles_c * p.tiles_r;
  const int64_t tile0 = blockIdx.x / (kPair * split), tile_step = gridDim.x / (kPair * split);

  if (warp == 0) {
    if (lane < p.stages) {
      mbar_init(&full[lane], 1);
      mbar_init(&empty[lane], 1);
    } else if (lane < p.stages + 2) {
      mbar_init(&acc_full[lane - p.stages], 1);
      mbar_init(&acc_empty[lane - p.stages], 128 * kPair);
    } else if (lane == 31) {
      peer_dead = 0;
      tma_ahead(&wmap);
      tma_ahead(&amap);
    }
    mbar_fence_init();
  }
  __syncwarp();
  if (warp == 1) tmem_alloc<PAIR>(&tmem_s, p.columns);
  tc_fence_before();
  // before a block's shared memory is written from another it has to be there: a
  // pair's at once, the others' before the sums go out
  if (PAIR) {
    cluster_meet();
  } else {
    if (split > 1) cluster_enter();
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  pdl_wait();
  pdl_launch();

  if (warp == 0) {  // ---- copies
    int s = 0, phase = 0, issued = 0;
    bool ok = true;
    for (int64_t t = tile0; ok && t < tiles; t += tile_step) {
      int c0, r0;
      tile_at(p, t, c0, r0);
      const int rank_r0 = PAIR && rank ? r0 + taken(r0) / 2 : r0;
      for (int k = k0; k < k1; ++k) {
        ok = warp_wait(&empty[s], phase ^ 1, kErrWaitEmpty);
        if (!ok) break;
        uint8_t* const at = smem + s * stage_bytes;
        if (acts) {
          if constexpr (PAIR) {
            // both blocks' copies are counted where the products wait for them
            const uint32_t bar = cluster_at(&full[s], 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * stage_bytes);
            tma_load_2d_pair(at, &wmap, k * kI8Step, c0 + rank * kI8Channels, bar);
            tma_load_2d_pair(at + kI8Channels * kI8Step, &amap, k * kI8Step, rank_r0, bar);
          } else {
            mbar_arrive_expect_tx(&full[s], stage_bytes);
            tma_load_2d(at, &wmap, k * kI8Step, c0, &full[s]);
            tma_load_2d(at + kI8Channels * kI8Step, &amap, k * kI8Step, r0, &full[s]);
          }
        }
        __syncwarp();
        ++issued;
        if (++s == p.stages) s = 0, phase ^= 1;
      }
    }
    // The products' arrivals at the last stages come before the block ends (in a pair
    // they are written from the other block).
    for (int n = 0, last = s, turn = phase; ok && n < p.stages; ++n) {
      ok = warp_wait(&empty[last], turn ^ 1, kErrWaitEmpty);
      if (++last == p.stages) last = 0, turn ^= 1;
    }
    if (!ok) {  // the copies in flight are waited for as well
      for (int n = rank == 0 || !PAIR ? min(issued, p.stages) : 0; n > 0; --n) {
        if (--s < 0) s = p.stages - 1, phase ^= 1;
        warp_wait(&full[s], phase, kErrWaitFull);
      }
    }
  } else if (warp == 1) {  // ---- products
    int s = 0, phase = 0, n = 0;
    bool ok = !PAIR || rank == 0;
    for (int64_t t = tile0; ok && t < tiles; t += tile_step, ++n) {
      const int b = n & 1;
      ok = warp_wait(&acc_empty[b], (n >> 1 & 1) ^ 1, kErrWaitEmpty);
      if (!ok) break;
      tc_fence_after();
      int c0, r0;
      tile_at(p, t, c0, r0);
      const uint32_t shape = tc_i8_shape(kPair * kI8Channels, taken(r0));
      const uint32_t d = tmem + b * p.tn;
      for (int k = k0; k < k1; ++k) {
        ok = warp_wait(&full[s], phase, kErrWaitFull);
        if (!ok) break;
        tc_fence_after();
        const uint8_t* const at = smem + s * stage_bytes;
        const uint64_t wd = tc_operand(at), ad = tc_operand(at + kI8Channels * kI8Step);
        if (acts) {
#pragma unroll
          for (int i = 0; i < kI8Step / 32; ++i)
            tc_mma_i8<PAIR>(d, wd + 2 * i, ad + 2 * i, shape, k > k0 || i > 0);
          tc_commit<PAIR>(&empty[s]);
          if (k + 1 == k1) tc_commit<PAIR>(&acc_full[b]);
        }
        __syncwarp();
        if (++s == p.stages) s = 0, phase ^= 1;
      }
    }
  } else if (split == 1) {  // ---- scales and stores
    const int quarter = warp % 4, tid = threadIdx.x - 64;
    bool ok = true;
    int n = 0;
    for (int64_t t = tile0; t < tiles; t += tile_step, ++n) {
      int c0, r0;
      tile_at(p, t, c0, r0);
      const int b = n & 1, left = min(p.tn, g.rows - r0);
      for (int j = tid; j < left; j += 128) as[b][j] = g.a_scales[r0 + j];
      const int c = c0 + (PAIR ? rank * kI8Channels : 0) + quarter * 32 + lane;
      const bool on = c < g.channels;
      const float ws = on ? g.w_scales[c] : 0.0f, bias = on && g.bias ? g.bias[c] : 0.0f;
      named_sync(1, 128);
      if (ok) ok = warp_wait(&acc_full[b], n >> 1 & 1, kErrWaitFull);
      tc_fence_after();
      OT* o = static_cast<OT*>(g.out) + (int64_t)r0 * g.out_stride + c;
      // 16 rows at a time, the next 16 on their way from tensor memory meanwhile
      const uint32_t from = tmem + (quarter * 32 << 16) + b * p.tn;
      int v[2][16];
      tmem_load16(from, v[0]);
      for (int j0 = 0; j0 < left; j0 += 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = j0 + 16 * h;
          if (j >= left) break;
          tmem_load_wait();
          if (j + 16 < left) tmem_load16(from + j + 16, v[h ^ 1]);
          store16(o, g.out_stride, v[h], &as[b][j], ws, bias, on ? left - j : 0, ok);
          o += 16 * g.out_stride;
        }
      }
      tc_fence_before();
      if (t + 2 * tile_step < tiles) {  // the products of a later tile wait for it
        if (PAIR) cluster_arrive(cluster_at(&acc_empty[b], 0));
        else mbar_arrive(&acc_empty[b]);
      }
    }
  }
  if (!PAIR && split > 1) {  // ---- one tile, k shared by the cluster
    // Each block ends up with i8_wide(split) of the channels, of all rows: every block
    // stores its sums of them into its shared memory straight from tensor memory
    // (stores answer nothing, so no load waits for another block). Sums of large
    // tiles go over the stages, once every block is done with its own.
    int c0, r0;
    tile_at(p, tile0, c0, r0);
    const int left = min(p.tn, g.rows - r0), wide = i8_wide(split);
    int* const sums = reinterpret_cast<int*>(smem + (p.apart ? p.stages * stage_bytes : 0));
    const int tid = threadIdx.x - 64, quarter = warp % 4;
    // what a thread adds up: 4 channels of one row in 128 / (wide / 4)
    const int part = tid % (wide / 4) * 4, first = tid / (wide / 4), c = c0 + rank * wide + part;
    const int end = min(g.channels, c0 + kI8Channels);
    float ws[4], bias[4];
    bool ok = true;
    if (warp >= 2) {
      for (int j = tid; j < left; j += 128) as[0][j] = g.a_scales[r0 + j];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ws[i] = c + i < end ? g.w_scales[c + i] : 0.0f;
        bias[i] = g.bias && c + i < end ? g.bias[c + i] : 0.0f;
      }
      ok = warp_wait(&acc_full[0], 0, kErrWaitFull);
      tc_fence_after();
    }
    __syncwarp();
    cluster_leave();  // of the start
    if (!p.apart) cluster_meet();
    if (warp >= 2 && ok) {
      const int ch = quarter * 32 + lane;
      uint32_t at = cluster_at(sums + (rank * p.tn) * wide + ch % wide, ch / wide);
      const uint32_t from = tmem + (quarter * 32 << 16);
      int v[2][16];
      tmem_load16(from, v[0]);
      for (int j0 = 0; j0 < left; j0 += 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int jh = j0 + 16 * h;
          if (jh >= left) break;
          tmem_load_wait();
          if (jh + 16 < left) tmem_load16(from + jh + 16, v[h ^ 1]);
#pragma unroll
          for (int j = 0; j < 16; ++j) cluster_store(at + j * wide * 4, v[h][j]);
          at += 16 * wide * 4;
        }
      }
      tc_fence_before();
    }
    if (warp >= 2 && !ok && lane == 0)
      for (int q = 0; q < split; ++q) cluster_store(cluster_at(&peer_dead, q), 1);
    __syncwarp();
    cluster_meet();
    if (warp >= 2) {
      OT* const o = static_cast<OT*>(g.out) + (int64_t)r0 * g.out_stride + c;
      const int* const mine = sums + part;
      const bool bad = peer_dead, whole = p.vec && c + 4 <= end;
      auto join = [&](auto blocks) {
        constexpr int S = decltype(blocks)::value, kWide = i8_wide(S), kRows = 128 / (kWide / 4);
        if (first >= kRows || c >= end) return;
        for (int j = first; j < left; j += kRows) {
          int4 v[S];
#pragma unroll
          for (int q = 0; q < S; ++q)
            v[q] = *reinterpret_cast<const int4*>(mine + (q * p.tn + j) * kWide);
#pragma unroll
          for (int q = 1; q < S; ++q)
            v[0].x += v[q].x, v[0].y += v[q].y, v[0].z += v[q].z, v[0].w += v[q].w;
          const float x = bad ? __uint_as_float(0x7fc00000u) : as[0][j];
          const float y[4] = {scaled(v[0].x, x, ws[0], bias[0]), scaled(v[0].y, x, ws[1], bias[1]),
                              scaled(v[0].z, x, ws[2], bias[2]), scaled(v[0].w, x, ws[3], bias[3])};
          OT* const to = o + (int64_t)j * g.out_stride;
          if (whole) {
            put4(to, y);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c + i < end) put(to + i, y[i]);
          }
        }
      };
      switch (split) {  // i8_plan's parts
        case 2: join(std::integral_constant<int, 2>()); break;
        case 3: join(std::integral_constant<int, 3>()); break;
        case 4: join(std::integral_constant<int, 4>()); break;
        case 6: join(std::integral_constant<int, 6>()); break;
        default: join(std::integral_constant<int, 8>());
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  // a pair's memory is free when both are done with it; their results need not have
  // arrived (waiting for that took 0.8 us)
  if (PAIR) cluster_end();
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_free<PAIR>(tmem, p.columns);
}

// ---- up to 16 rows: the weights pass once, from memory into registers
//
// mma.sync of 16 rows by 8 channels by 32 bytes of k. The order of k inside the
// sum is free, so a lane takes 16 bytes of a channel at once (4 lanes 64 bytes of
// it side by side) and feeds them to two products, the rows' bytes in the same
// order. The block's warps share k and meet once in shared memory.
MYOS_DEV void mma_i8(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                     uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, "
      "%9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from i on; zeros from k on, where nothing is read.
MYOS_DEV uint4 piece(const int8_t* row, int i, int k) {
  if (i + 16 <= k) return *reinterpret_cast<const uint4*>(row + i);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (i + e < k) v[e / 4] |= (uint32_t)(uint8_t)row[i + e] << (8 * (e % 4));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// NT: groups of 8 channels a block. U: 64-byte pieces of k at once. HI: rows 8 to 15.
template <class OT, int NT, int U, bool HI>
__global__ void __launch_bounds__(512) k_few_i8(const MatArgs g) {
  constexpr int kTok = HI ? 16 : 8, kCh = NT * 8;
  extern __shared__ int parts[];  // [warp][row][channel]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int gr = lane / 4, q = lane % 4;
  const int c0 = (int)blockIdx.x * kCh;
  const int blocks = (g.k + 63) / 64;
  const int b0 = (int)((int64_t)blocks * warp / warps), b1 = (int)((int64_t)blocks * (warp + 1) / warps);
  const int8_t* wp[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    wp[n] = g.w + (int64_t)min(c0 + n * 8 + gr, g.channels - 1) * g.w_stride + q * 16;
  const int8_t* const lo = g.a + (int64_t)min(gr, g.rows - 1) * g.a_stride + q * 16;
  const int8_t* const hi = g.a + (int64_t)min(gr + 8, g.rows - 1) * g.a_stride + q * 16;
  const bool has_lo = gr < g.rows, has_hi = HI && gr + 8 < g.rows;
  int acc[NT][4] = {};
  pdl_wait();
  pdl_launch();
#pragma unroll
  for (int n = 0; n < NT; ++n) after_wait(wp[n]);
  const uint4 z = make_uint4(0, 0, 0, 0);
  auto multiply = [&](const uint4* w, const uint4& x, const uint4& y) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mma_i8(acc[n], x.x, y.x, x.y, y.y, w[n].x, w[n].y);
      mma_i8(acc[n], x.z, y.z, x.w, y.w, w[n].z, w[n].w);
    }
  };
  const int whole = min(b1, g.k / 64);
  for (int b = b0; b < whole; b += U) {
    uint4 w[U][NT], x[U], y[U];
    // (two branches that meet: without them the loads sink to their products, a few at
    // a time, and 1 x 13824 x 5120 takes 21 us for 14)
    if (b + U <= whole) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
          w[u][n] = ld_once(reinterpret_cast<const uint4*>(wp[n] + (b + u) * 64));
        x[u] = has_lo ? *reinterpret_cast<const uint4*>(lo + (b + u) * 64) : z;
        y[u] = has_hi ? *reinterpret_cast<const uint4*>(hi + (b + u) * 64) : z;
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = min(b + u, whole - 1) * 64;  // past the end the last again, times nothing
        const bool in = b + u < whole;
#pragma unroll
        for (int n = 0; n < NT; ++n) w[u][n] = ld_once(reinterpret_cast<const uint4*>(wp[n] + at));
        x[u] = in && has_lo ? *reinterpret_cast<const uint4*>(lo + at) : z;
        y[u] = in && has_hi ? *reinterpret_cast<const uint4*>(hi + at) : z;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) multiply(w[u], x[u], y[u]);
  }
  if (b1 > whole && b1 > b0) {  // the piece that k ends in
    const int at = whole * 64, left = g.k - q * 16;
    uint4 w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) w[n] = piece(wp[n], at, left);
    multiply(w, has_lo ? piece(lo, at, left) : z, has_hi ? piece(hi, at, left) : z);
  }
  int* const mine = parts + warp * kTok * kCh;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    *reinterpret_cast<int2*>(mine + gr * kCh + n * 8 + q * 2) = make_int2(acc[n][0], acc[n][1]);
    if (HI)
      *reinterpret_cast<int2*>(mine + (gr + 8) * kCh + n * 8 + q * 2) = make_int2(acc[n][2], acc[n][3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < g.rows * kCh; i += blockDim.x) {
    const int r = i / kCh, c = c0 + i % kCh;
    int sum = 0;
    for (int p = 0; p < warps; ++p) sum += parts[p * kTok * kCh + i];
    if (c < g.channels)
      put(static_cast<OT*>(g.out) + (int64_t)r * g.out_stride + c,
          scaled(sum, g.a_scales[r], g.w_scales[c], g.bias ? g.bias[c] : 0.0f));
  }
}

template <class OT, int NT, int U>
cudaError_t launch_few_of(const MatArgs& g, int warps, cudaStream_t st) {
  const bool hi = g.rows > 8;
  const size_t smem = (size_t)warps * (hi ? 16 : 8) * NT * 8 * 4;
  const dim3 grid((unsigned)i8_ceil(g.channels, NT * 8));
  return counted(hi ? launch_pdl(k_few_i8<OT, NT, U, true>, grid, warps * 32, smem, st, 1, g)
                    : launch_pdl(k_few_i8<OT, NT, U, false>, grid, warps * 32, smem, st, 1, g));
}
template <class OT>
cudaError_t launch_few(const MatArgs& g, const I8Few& f, cudaStream_t st) {
  if (f.groups == 4) return launch_few_of<OT, 4, 3>(g, f.warps, st);
  if (f.groups == 2) return launch_few_of<OT, 2, 4>(g, f.warps, st);
  return launch_few_of<OT, 1, 6>(g, f.warps, st);
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static std::atomic<void*> known{nullptr};
  void* f = known.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    known.store(f, std::memory_order_release);
  }
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
}

// Rows of k bytes in boxes of `box` rows by 128 bytes; what lies outside reads as 0.
bool map_rows(CUtensorMap* map, const int8_t* p, int64_t k, int64_t rows, int64_t stride, int box) {
  const auto encode = encoder();
  if (!encode) return false;
  const cuuint64_t size[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
  const cuuint32_t boxes[2] = {kI8Step, (cuuint32_t)box}, steps[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), size, strides, boxes,
                steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class OT, bool PAIR>
cudaError_t launch(const MatArgs& g, const CUtensorMap& wmap, const CUtensorMap& amap,
                   const I8Device& d, cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  const cudaError_t e =
      raise_smem_limit((const void*)k_matmul_i8<OT, PAIR>, kI8Smem + 1024, &raised);
  if (e != cudaSuccess) return e;
  const size_t smem = (g.plan.two ? kI8SmemTwo : kI8Smem) + 1024;
  const int64_t tiles = (int64_t)g.plan.tiles_c * g.plan.tiles_r;
  const int blocks_a_tile = PAIR ? 2 : g.plan.split;
  const int64_t most = PAIR ? d.one[2] / 2 : d.sms * (g.plan.two ? 2 : 1);
  const int64_t at_once = g.plan.split > 1 ? tiles : std::min(tiles, most);
  return counted(launch_pdl(k_matmul_i8<OT, PAIR>, dim3((unsigned)(at_once * blocks_a_tile)),
                            kThreads, smem, st, blocks_a_tile, wmap, amap, g));
}
// A kernel of k_matmul_i8's size: for that itself, as for any that takes tensor
// memory, the occupancy calls answer one block a multiprocessor.
__global__ void __launch_bounds__(kThreads) k_room() {}

// The clusters that the current device holds.
I8Device this_device() {
  static std::atomic<uint64_t> known[64][kI8MaxSplit + 1];
  I8Device d = {};
  d.sms = sm_count();
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return d;  // nothing is split
  const void* const kernel = (const void*)k_room;
  i8_room(d, known[dev], [&](int s, bool two, int* blocks) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)s);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (two ? kI8SmemTwo : kI8Smem) + 4096;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    static std::atomic<uint64_t> raised{0};
    int clusters = 0;
    if (raise_smem_limit(kernel, kI8Smem + 4096, &raised) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    *blocks = clusters * s;
    return true;
  });
  return d;
}

template <class OT>
cudaError_t launch_tiles(const MatArgs& g, const CUtensorMap& wmap, const CUtensorMap& amap,
                         const I8Device& d, cudaStream_t st) {
  return g.plan.pair ? launch<OT, true>(g, wmap, amap, d, st)
                     : launch<OT, false>(g, wmap, amap, d, st);
}

}  // namespace
}  // namespace myos

using namespace myos;

extern "C" {

int myos_dev_matmul_i8(void* d_out, int32_t out_dtype, size_t out_stride, const int8_t* d_a,
                       size_t a_stride, const float* d_a_scales, const int8_t* d_w,
                       size_t w_stride, const float* d_w_scales, const float* d_bias, size_t rows,
                       size_t k, size_t channels, void* stream) {
  if (out_dtype != MYOS_F32 && out_dtype != MYOS_BF16) return MYOS_ERR_ARG;
  if (rows == 0 || channels == 0) return MYOS_OK;
  if (!d_out || !d_a || !d_a_scales || !d_w || !d_w_scales) return MYOS_ERR_ARG;
  const size_t most = (size_t)1 << 39;
  if (rows > 0x7fffff00 || channels > 0x7fffff00 || k == 0 || k > MYOS_I8_MAX_K || a_stride < k ||
      w_stride < k || out_stride < channels || a_stride > most || w_stride > most ||
      out_stride > most)
    return MYOS_ERR_SHAPE;
  if (!aligned(d_out, out_dtype == MYOS_F32 ? 4 : 2) || !aligned(d_a, 16) || !aligned(d_w, 16) ||
      a_stride % 16 != 0 || w_stride % 16 != 0 || !aligned(d_a_scales, 4) ||
      !aligned(d_w_scales, 4) || !aligned(d_bias, 4))
    return MYOS_ERR_ARG;
  MatArgs g;
  g.out = d_out;
  g.out_stride = (int64_t)out_stride;
  g.a = d_a;
  g.a_stride = (int64_t)a_stride;
  g.w = d_w;
  g.w_stride = (int64_t)w_stride;
  g.k = (int)k;
  g.a_scales = d_a_scales;
  g.w_scales = d_w_scales;
  g.bias = d_bias;
  g.rows = (int)rows;
  g.channels = (int)channels;
  g.steps = (int)i8_ceil((int64_t)k, kI8Step);
  const I8Few few = i8_few((int64_t)rows, (int64_t)k, (int64_t)channels);
  if (few.use) {
    const cudaError_t e = out_dtype == MYOS_F32
                              ? launch_few<float>(g, few, (cudaStream_t)stream)
                              : launch_few<__nv_bfloat16>(g, few, (cudaStream_t)stream);
    return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
  }
  const size_t size = out_dtype == MYOS_F32 ? 4 : 2;
  const I8Device device = this_device();
  g.plan = i8_plan((int64_t)rows, (int64_t)k, (int64_t)channels, device);
  g.plan.vec = aligned(d_out, 4 * size) && (rows == 1 || out_stride % 4 == 0);
  CUtensorMap wmap, amap;
  if (!map_rows(&wmap, d_w, (int64_t)k, (int64_t)channels, (int64_t)w_stride, kI8Channels) ||
      !map_rows(&amap, d_a, (int64_t)k, (int64_t)rows, (int64_t)a_stride,
                g.plan.tn / (g.plan.pair ? 2 : 1)))
    return MYOS_ERR_CUDA;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = out_dtype == MYOS_F32 ? launch_tiles<float>(g, wmap, amap, device, st)
                                              : launch_tiles<__nv_bfloat16>(g, wmap, amap, device, st);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}

int myos_dev_matmul_i8_status(void) {
  static std::mutex one;  // callers share the answer's place
  const std::lock_guard<std::mutex> hold(one);
  uint32_t failed = 0;
  // a copy from a symbol waits for the default stream, and that for no other that was
  // made non-blocking
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) {
    k_take_failed<<<1, 1>>>();
    e = counted(cudaGetLastError());
  }
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&failed, g_wait_taken, sizeof failed);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return MYOS_ERR_CUDA;
  }
  return failed ? MYOS_ERR_TIMEOUT : MYOS_OK;
}

}  // extern "C"
