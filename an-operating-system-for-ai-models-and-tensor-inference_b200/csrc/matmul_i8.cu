// The product of 8-bit rows and 8-bit channels with a scale each
// (include/myos_cuda.h, "Projections in 8-bit integers"): out[r][c] =
// (sum_i a[r][i] w[c][i]) a_scales[r] w_scales[c] + bias[c].
//
// The sum is exact in 32-bit integers, so it may be split and joined in any order
// and gives the same bits.
//
// A tile is 128 channels (the tensor core's M, the lanes of its memory) by up to
// 256 rows (its N, the columns): a lane holds one channel, so a warp's store of
// one row is 32 channels side by side, and few rows cost nothing but their own
// columns. Six warps: copies (TMA, 128 bytes of k a stage), products (tcgen05,
// 32 bytes of k each), and four that scale and store while the next tile's
// products go into the other half of the tensor memory. Where there are fewer
// tiles than multiprocessors, a cluster shares a tile's k and adds its parts
// through shared memory.
#include <cudaTypedefs.h>
#include <math.h>

#include "i8_plan.h"
#include "kernels.h"
#include "paged.h"
#include "tcgen05.cuh"

namespace myos {
namespace {

struct MatArgs {
  void* out;
  int64_t out_stride;
  const float* a_scales;
  const float* w_scales;
  const float* bias;
  int rows, channels, steps;
  I8Plan plan;
};

__device__ uint32_t g_wait_failed;

MYOS_DEV float scaled(int sum, float as, float ws, float bias) {
  return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(sum), as), ws), bias);
}
MYOS_DEV void put(float* p, float v) { *p = v; }
MYOS_DEV void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

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
constexpr int kGroup = 16;  // row tiles that share a channel tile's weights in L2 before the next

// Tile t: its first channel and row.
MYOS_DEV void tile_at(const I8Plan& p, int64_t t, int& c0, int& r0) {
  const int64_t group = t / ((int64_t)kGroup * p.tiles_c);
  const int first = (int)group * kGroup;
  const int wide = min(kGroup, p.tiles_r - first);
  const int64_t in = t - group * kGroup * p.tiles_c;
  c0 = (int)(in / wide) * kI8Channels;
  r0 = (first + (int)(in % wide)) * p.tn;
}

template <class OT>
__global__ void __launch_bounds__(kThreads, 1)
    k_matmul_i8(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap amap,
                const MatArgs g) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kI8MaxStages], empty[kI8MaxStages], acc_full[2], acc_empty[2];
  __shared__ __align__(16) float as[2][kI8MaxRows];
  __shared__ uint32_t tmem_s;
  __shared__ int dead;  // a wait of this block ran out
  uint8_t* const smem = raw + (-smem_u32(raw) & 1023);
  const I8Plan& p = g.plan;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t stage_bytes = (kI8Channels + p.tn) * kI8Step;
  const int split = p.split, rank = split > 1 ? (int)cluster_rank() : 0;
  const int k0 = (int)((int64_t)g.steps * rank / split);
  const int k1 = (int)((int64_t)g.steps * (rank + 1) / split);
  const int64_t tiles = (int64_t)p.tiles_c * p.tiles_r;
  const int64_t tile0 = blockIdx.x / split, tile_step = gridDim.x / split;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 128);
    }
    dead = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&tmem_s, p.columns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  pdl_wait();
  pdl_launch();

  if (warp == 0) {
    if (lane == 0) {  // ---- copies
      int s = 0, phase = 0, issued = 0;
      bool ok = true;
      for (int64_t t = tile0; ok && t < tiles; t += tile_step) {
        int c0, r0;
        tile_at(p, t, c0, r0);
        for (int k = k0; k < k1; ++k) {
          if (!mbar_wait(&empty[s], phase ^ 1, &g_wait_failed, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          uint8_t* const at = smem + s * stage_bytes;
          mbar_arrive_expect_tx(&full[s], stage_bytes);
          tma_load_2d(at, &wmap, k * kI8Step, c0, &full[s]);
          tma_load_2d(at + kI8Channels * kI8Step, &amap, k * kI8Step, r0, &full[s]);
          ++issued;
          if (++s == p.stages) s = 0, phase ^= 1;
        }
      }
      if (!ok) {  // its copies in flight are waited for before the block ends
        *(volatile int*)&dead = 1;
        for (int n = min(issued, p.stages); n > 0; --n) {
          if (--s < 0) s = p.stages - 1, phase ^= 1;
          mbar_wait(&full[s], phase, &g_wait_failed, kErrWaitFull);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {  // ---- products
      const uint32_t shape = tc_i8_shape(kI8Channels, p.tn);
      int s = 0, phase = 0, n = 0;
      bool ok = true;
      for (int64_t t = tile0; ok && t < tiles; t += tile_step, ++n) {
        const int b = n & 1;
        ok = mbar_wait(&acc_empty[b], (n >> 1 & 1) ^ 1, &g_wait_failed, kErrWaitEmpty);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + b * p.tn;
        for (int k = k0; k < k1; ++k) {
          ok = mbar_wait(&full[s], phase, &g_wait_failed, kErrWaitFull);
          if (!ok) break;
          tc_fence_after();
          const uint8_t* const at = smem + s * stage_bytes;
          const uint64_t wd = tc_operand(at), ad = tc_operand(at + kI8Channels * kI8Step);
#pragma unroll
          for (int i = 0; i < kI8Step / 32; ++i)
            tc_mma_i8(d, wd + 2 * i, ad + 2 * i, shape, k > k0 || i > 0);
          tc_commit(&empty[s]);
          if (++s == p.stages) s = 0, phase ^= 1;
        }
        if (ok) tc_commit(&acc_full[b]);
      }
      if (!ok) *(volatile int*)&dead = 1;
    }
    __syncwarp();
  } else if (split == 1) {  // ---- scales and stores
    const int quarter = warp % 4, tid = threadIdx.x - 64;
    bool ok = true;
    int n = 0;
    for (int64_t t = tile0; t < tiles; t += tile_step, ++n) {
      int c0, r0;
      tile_at(p, t, c0, r0);
      const int b = n & 1, left = min(p.tn, g.rows - r0);
      for (int j = tid; j < left; j += 128) as[b][j] = g.a_scales[r0 + j];
      const int c = c0 + quarter * 32 + lane;
      const bool on = c < g.channels;
      const float ws = on ? g.w_scales[c] : 0.0f, bias = on && g.bias ? g.bias[c] : 0.0f;
      named_sync(1, 128);
      if (ok) ok = mbar_wait(&acc_full[b], n >> 1 & 1, &g_wait_failed, kErrWaitFull);
      if (!ok) *(volatile int*)&dead = 1;
      ok = __all_sync(0xffffffffu, ok);
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
      mbar_arrive(&acc_empty[b]);
    }
  }
  if (split > 1) {  // ---- one tile, k shared by the cluster
    int c0, r0;
    tile_at(p, tile0, c0, r0);
    const int left = min(p.tn, g.rows - r0);
    int* const part = reinterpret_cast<int*>(smem);  // [row][channel], over the stages
    if (warp >= 2) {
      const int quarter = warp % 4;
      bool ok = mbar_wait(&acc_full[0], 0, &g_wait_failed, kErrWaitFull);
      if (!ok) *(volatile int*)&dead = 1;
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (ok) {
        for (int j0 = 0; j0 < left; j0 += 16) {
          int v[16];
          tmem_load16(tmem + (quarter * 32 << 16) + j0, v);
          tmem_load_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(j0 + j) * kI8Channels + quarter * 32 + lane] = v[j];
        }
      }
      tc_fence_before();
    }
    __syncwarp();
    cluster_meet();
    if (warp >= 2) {
      const int ch = threadIdx.x - 64, c = c0 + ch;
      const bool on = c < g.channels;
      const float ws = on ? g.w_scales[c] : 0.0f, bias = on && g.bias ? g.bias[c] : 0.0f;
      int bad = 0;
      for (int q = 0; q < split; ++q) bad |= cluster_load(cluster_at(&dead, q));
      const int j1 = left * (rank + 1) / split;
      for (int j = left * rank / split; j < j1; ++j) {
        int sum = 0;
        for (int q = 0; q < split; ++q)
          sum += cluster_load(cluster_at(part + j * kI8Channels + ch, q));
        if (on)
          put(static_cast<OT*>(g.out) + (int64_t)(r0 + j) * g.out_stride + c,
              bad ? __uint_as_float(0x7fc00000u) : scaled(sum, g.a_scales[r0 + j], ws, bias));
      }
    }
    __syncwarp();
    cluster_meet();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_free(tmem, p.columns);
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

template <class OT>
cudaError_t launch(const MatArgs& g, const CUtensorMap& wmap, const CUtensorMap& amap, int sms,
                   cudaStream_t st) {
  constexpr size_t kSmem = kI8StageBytes + 1024;
  static std::atomic<uint64_t> raised{0};
  const cudaError_t e = raise_smem_limit((const void*)k_matmul_i8<OT>, kSmem, &raised);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)g.plan.tiles_c * g.plan.tiles_r;
  const int64_t blocks = g.plan.split > 1 ? tiles * g.plan.split : tiles < sms ? tiles : sms;
  return counted(launch_pdl(k_matmul_i8<OT>, dim3((unsigned)blocks), kThreads, kSmem, st,
                            g.plan.split, wmap, amap, g));
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
  const int sms = sm_count();
  MatArgs g;
  g.out = d_out;
  g.out_stride = (int64_t)out_stride;
  g.a_scales = d_a_scales;
  g.w_scales = d_w_scales;
  g.bias = d_bias;
  g.rows = (int)rows;
  g.channels = (int)channels;
  g.steps = i8_ceil((int64_t)k, kI8Step);
  g.plan = i8_plan((int64_t)rows, (int64_t)k, (int64_t)channels, sms);
  CUtensorMap wmap, amap;
  if (!map_rows(&wmap, d_w, (int64_t)k, (int64_t)channels, (int64_t)w_stride, kI8Channels) ||
      !map_rows(&amap, d_a, (int64_t)k, (int64_t)rows, (int64_t)a_stride, g.plan.tn))
    return MYOS_ERR_CUDA;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = out_dtype == MYOS_F32 ? launch<float>(g, wmap, amap, sms, st)
                                              : launch<__nv_bfloat16>(g, wmap, amap, sms, st);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}

int myos_dev_matmul_i8_status(void) {
  uint32_t failed = 0, none = 0;
  if (cudaMemcpyFromSymbol(&failed, g_wait_failed, sizeof failed) != cudaSuccess) {
    cudaGetLastError();
    return MYOS_ERR_CUDA;
  }
  if (failed == 0) return MYOS_OK;
  if (cudaMemcpyToSymbol(g_wait_failed, &none, sizeof none) != cudaSuccess) {
    cudaGetLastError();
    return MYOS_ERR_CUDA;
  }
  return MYOS_ERR_TIMEOUT;
}

}  // extern "C"
