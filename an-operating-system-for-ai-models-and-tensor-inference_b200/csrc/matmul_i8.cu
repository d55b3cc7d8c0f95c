// The product of 8-bit rows and 8-bit channels with a scale each
// (include/myos_cuda.h, "Projections in 8-bit integers"): out[r][c] =
// (sum_i a[r][i] w[c][i]) a_scales[r] w_scales[c] + bias[c].
//
// The sum is exact in 32-bit integers, so it may be split and joined in any order
// and gives the same bits.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace myos {
namespace {

struct MatArgs {
  void* out;
  int64_t out_stride;
  const int8_t* a;
  int64_t a_stride;
  const float* a_scales;
  const int8_t* w;
  int64_t w_stride;
  const float* w_scales;
  const float* bias;
  int rows, k, channels;
};

MYOS_DEV float scaled(int sum, float as, float ws, float bias) {
  return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(sum), as), ws), bias);
}
MYOS_DEV void put(float* p, float v) { *p = v; }
MYOS_DEV void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// 16 bytes of a row from i on; zeros behind k.
MYOS_DEV uint4 piece(const int8_t* row, int i, int k) {
  if (i + 16 <= k) return *reinterpret_cast<const uint4*>(row + i);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (i + e < k) v[e / 4] |= (uint32_t)(uint8_t)row[i + e] << (8 * (e % 4));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// 64 x 64 results a block, 4 x 4 a thread, 64 bytes of k at a time.
template <class OT>
__global__ void __launch_bounds__(256) k_matmul_i8(const MatArgs g) {
  __shared__ uint32_t as[16][68], ws[16][68];
  pdl_wait();
  pdl_launch();
  const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  const int lr = threadIdx.x / 4, lp = threadIdx.x % 4;
  int sum[4][4] = {};
  for (int k0 = 0; k0 < g.k; k0 += 64) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    const uint4 x = r0 + lr < g.rows ? piece(g.a + (r0 + lr) * g.a_stride, k0 + lp * 16, g.k) : z;
    const uint4 y =
        c0 + lr < g.channels ? piece(g.w + (c0 + lr) * g.w_stride, k0 + lp * 16, g.k) : z;
    as[lp * 4 + 0][lr] = x.x, as[lp * 4 + 1][lr] = x.y, as[lp * 4 + 2][lr] = x.z, as[lp * 4 + 3][lr] = x.w;
    ws[lp * 4 + 0][lr] = y.x, ws[lp * 4 + 1][lr] = y.y, ws[lp * 4 + 2][lr] = y.z, ws[lp * 4 + 3][lr] = y.w;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          sum[r][c] = __dp4a((int)as[i][tr + 16 * r], (int)ws[i][tc + 16 * c], sum[r][c]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int64_t col = c0 + tc + 16 * c;
    if (col >= g.channels) continue;
    const float scale = g.w_scales[col], bias = g.bias ? g.bias[col] : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = r0 + tr + 16 * r;
      if (row < g.rows)
        put(static_cast<OT*>(g.out) + row * g.out_stride + col,
            scaled(sum[r][c], g.a_scales[row], scale, bias));
    }
  }
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
  g.a_scales = d_a_scales;
  g.w = d_w;
  g.w_stride = (int64_t)w_stride;
  g.w_scales = d_w_scales;
  g.bias = d_bias;
  g.rows = (int)rows;
  g.k = (int)k;
  g.channels = (int)channels;
  const cudaStream_t st = (cudaStream_t)stream;
  for (size_t r = 0; r < rows; r += 65535 * 64) {  // a grid's second side has at most 65535 blocks
    MatArgs p = g;
    const size_t n = rows - r < 65535 * 64 ? rows - r : 65535 * 64;
    p.rows = (int)n;
    p.a += r * a_stride;
    p.a_scales += r;
    p.out = static_cast<char*>(d_out) + r * out_stride * (out_dtype == MYOS_F32 ? 4 : 2);
    const dim3 grid((unsigned)((channels + 63) / 64), (unsigned)((n + 63) / 64));
    const cudaError_t e =
        out_dtype == MYOS_F32
            ? counted(launch_pdl(k_matmul_i8<float>, grid, 256, 0, st, 1, p))
            : counted(launch_pdl(k_matmul_i8<__nv_bfloat16>, grid, 256, 0, st, 1, p));
    if (e != cudaSuccess) return MYOS_ERR_CUDA;
  }
  return MYOS_OK;
}

int myos_dev_matmul_i8_status(void) { return MYOS_OK; }

}  // extern "C"
