// Rows in 8 bits with a scale each: plain rows, silu(gate) * up, and the
// residual's addition with RMSNorm (include/myos_cuda.h, "Projections in 8-bit
// integers").
//
// The mathematics: y of the row, scale = f32(max|y| / 127), q = rint(y / scale).
// A row's largest value and the nearest integer are where a rounding decides:
// with y off by 2^-23 one value in some ten thousand lands one step away, and
// which one depends on the order of the row's sum. So both are decided in 64
// bits, but only where 32 leave them open: y is computed in f32 with a bound on
// its error (kRel below); the values within that bound of the maximum are computed
// again in f64 from the inputs, and those within it of a border between two steps
// (about one in 10^4) are compared with border * scale, which is exact. The sum of
// squares is f64 throughout.
//
// A row is read once into registers (a block per row, or a warp where it has at most
// 1024 values), two meetings of the block, q and scale out. f32 rows are bound by the
// memory (8191 x 5120: 6.25 TB/s for the norm, 5.4 with bf16 x; 6.6 for plain rows), bf16
// rows by instructions (27648 x 5120: 93 us, 4.6 TB/s), SwiGLU too (4099 x 13824 bf16:
// 85 us, 3.3; f32: 106 us, 4.8), a few rows by their latency (norm 1 x 1536: 2.3 us). Of a
// SwiGLU whose up values do not begin at 16 bytes, and of other rows that do not, a block
// takes one value at a time, three times over: 4099 x 13823 bf16 367 us.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace myos {
namespace {

enum { kQuant, kSwiglu, kNorm };

struct RowArgs {
  int8_t* q;
  int64_t q_stride;
  float* scales;
  const void* x;
  int64_t x_stride;
  const float* residual;
  int64_t residual_stride;
  float* total;
  int64_t total_stride;
  const uint16_t* gamma;
  float eps;
  int rows, width;
};

constexpr float kSmallest = 1.17549435e-38f;  // 2^-126
constexpr float kTiny = 7.8886e-31f;          // 2^-100: below it f32 products lose bits, all goes through f64
constexpr uint64_t kPast = 0x47effffff0000000ull;  // f64's 2^128 - 2^103: rounds to no finite f32

MYOS_DEV float get(const float* p) { return *p; }
MYOS_DEV float get(const uint16_t* p) { return bf16_at(p); }

// 8 values at a 16-byte boundary. Plain loads: in place, x or the residual is written.
MYOS_DEV void load8(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
MYOS_DEV void load8(const uint16_t* p, float* v) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  v[0] = bf16_lo(a.x), v[1] = bf16_hi(a.x), v[2] = bf16_lo(a.y), v[3] = bf16_hi(a.y);
  v[4] = bf16_lo(a.z), v[5] = bf16_hi(a.z), v[6] = bf16_lo(a.w), v[7] = bf16_hi(a.w);
}
MYOS_DEV uint4 some8(const uint16_t* p, int n) {
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) v[e / 2] |= (uint32_t)p[e] << (16 * (e % 2));
  return make_uint4(v[0], v[1], v[2], v[3]);
}
template <class T>
MYOS_DEV void load_some(const T* p, float* v, int n) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? get(p + e) : 0.0f;
}

__device__ __noinline__ double silu_up64(float g, float u) {
  return (double)g / (1.0 + exp(-(double)g)) * (double)u;
}

// In f32, exp(-g) by the special function unit. The rounding of its argument
// makes the result relatively off by |g| 2^-23 where g is negative, so values
// below -8 (rare in a gate) go through f64; the rest is off by 1.6 x 2^-20 at
// most: the argument 2^-20, ex2 2^-22, rcp 2^-23, a sum and two products 2^-24
// each. That holds for every y that counts in a row past kTiny, whatever the inputs:
// r * u first, which is below f32's normal numbers only where u is nearly so itself, and
// with such a u y reaches 2^-121 only by a gate above 17, whose r is 1. g * r first lost
// bits of the smallest gates, which a large u brings back.
MYOS_DEV bool silu_fast(float g) { return g >= -8.0f; }
MYOS_DEV float silu_up(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * (r * u);
}

// One row as a thread sees it.
template <int KIND, class XT>
struct Row {
  const XT* x;
  const float* residual;
  float* total;
  const uint16_t* gamma;
  int width;

  // y of one value in 64 bits, from the inputs. scale64: what the norm multiplies by.
  MYOS_DEV double exact(int i, double inv) const {
    if (KIND == kQuant) return (double)get(x + i);
    if (KIND == kSwiglu) return silu_up64(get(x + i), get(x + width + i));
    // in place the inputs are gone: the total was written by this thread
    const float t = total ? total[i] : residual ? __fadd_rn(get(x + i), residual[i]) : get(x + i);
    // each product rounded: drawn into decide's difference, the last one would not be
    return __dmul_rn((double)bf16_at(gamma + i), __dmul_rn((double)t, inv));
  }

  // The f32 values that go with y (of the norm: gamma * total, without its
  // factor), for 8 of the row from i on, n of them in it; adds the squares.
  template <bool FULL>
  MYOS_DEV void values(int i, int n, float* p, double& squares) const {
    float a[8], b[8];
    if (FULL) load8(x + i, a);
    else load_some(x + i, a, n);
    if (KIND == kQuant) {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = a[e];
    } else if (KIND == kSwiglu) {
      if (FULL) load8(x + width + i, b);
      else load_some(x + width + i, b, n);
      float lowest = a[0];  // (a NaN is one in p)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = silu_up(a[e], b[e]);
        lowest = fminf(lowest, a[e]);
      }
      if (!silu_fast(lowest)) {  // one place for the call: eight of them cost registers
#pragma unroll 1
        for (int f = 0; f < n && f < 8; ++f) {
          const float g = get(x + i + f);
          if (silu_fast(g)) continue;
          const float y = (float)silu_up64(g, get(x + width + i + f));
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] = e == f ? y : p[e];
        }
      }
    } else {
      if (residual) {
        if (FULL) load8(residual + i, b);
        else load_some(residual + i, b, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = __fadd_rn(a[e], b[e]);
      }
      if (FULL) load8(gamma + i, b);
      else load_some(gamma + i, b, n);
      if (total) {
        if (FULL) {
          reinterpret_cast<float4*>(total + i)[0] = make_float4(a[0], a[1], a[2], a[3]);
          reinterpret_cast<float4*>(total + i)[1] = make_float4(a[4], a[5], a[6], a[7]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) total[i + e] = a[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        squares += (double)a[e] * (double)a[e];
        p[e] = __fmul_rn(a[e], b[e]);
      }
    }
  }
  // The f32 value of one, its inputs read again.
  MYOS_DEV float value(int i) const {
    if (KIND == kQuant) return get(x + i);
    if (KIND == kSwiglu) {
      const float g = get(x + i), u = get(x + width + i);
      return silu_fast(g) ? silu_up(g, u) : (float)silu_up64(g, u);
    }
    const float t = total ? total[i] : residual ? __fadd_rn(get(x + i), residual[i]) : get(x + i);
    return __fmul_rn(t, bf16_at(gamma + i));
  }
};

// How far an f32 value, or its position among the steps, may be from that in 64 bits,
// relatively: a rounding each of gamma * total and of the factor that makes steps of it
// (2^-24 each; four times that here); silu_up's own error beside them. The values that
// may be the largest are within twice that of it.
template <int KIND>
constexpr float kRel = KIND == kSwiglu ? 1.9073e-6f : 2.3842e-7f;  // 2^-19, 2^-22

// The larger magnitude, NaN above infinity above all others.
MYOS_DEV float larger(float a, float v) {
  float r;
  asm("{\n .reg .f32 t;\n abs.f32 t, %2;\n max.NaN.f32 %0, %1, t;\n}" : "=f"(r) : "f"(a), "f"(v));
  return r;
}
// The same order among integers. The sign is taken off the bits (arithmetic may
// leave a NaN's as it is).
MYOS_DEV uint64_t magnitude(double v) {
  return (uint64_t)__double_as_longlong(v) & 0x7fffffffffffffffull;
}

MYOS_DEV uint64_t warp_most(uint64_t v) {  // the upper halves, then the lower of those
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, v >> 32 == hi ? (uint32_t)v : 0u);
  return (uint64_t)hi << 32 | lo;
}

// x / 127, correctly rounded: a quotient by the rounded reciprocal, its remainder
// exactly, and the correction (Markstein's division).
MYOS_DEV double over127(double x) {
  const double y = 1.0 / 127.0, q = x * y;
  return q < 1e300 ? fma(fma(-127.0, q, x), y, q) : q;
}

// p * per rounded to the nearest integer, in the low byte. The addition rounds: the
// sum's last bit is 1 (rint and its conversion run at a quarter of the rate). edge:
// the largest distance from an integer, with what it may be wrong by; from kEdge on
// a value may lie on the other side of the border between two steps.
constexpr float kEdge = 0.5f;
template <int KIND>
MYOS_DEV uint32_t step(float p, float per, float& edge) {
  const float t = __fmaf_rn(p, per, 12582912.0f), n = __fsub_rn(t, 12582912.0f);
  const float off = __fmaf_rn(p, per, -n);
  // of the silu the bound goes by the step: a bound for all would open four times as many
  edge = KIND == kSwiglu ? larger(edge, __fmaf_rn(fabsf(n), kRel<KIND>, fabsf(off) + kRel<KIND>))
                         : larger(edge, off);
  return __float_as_uint(t);
}
template <int KIND>
MYOS_DEV bool open(float edge) {
  return !(edge < (KIND == kSwiglu ? kEdge : kEdge - 128.0f * kRel<KIND>));
}

// A chunk's 8 values between the passes: bf16 rows as they came, for more rows at once.
template <int KIND, class XT>
struct Held {
  float v[8];
  MYOS_DEV void keep(const float* p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = p[e];
  }
  MYOS_DEV void take(float* p) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = v[e];
  }
};
template <>
struct Held<kQuant, uint16_t> {
  uint4 v;
  MYOS_DEV void take(float* p) const { load8(reinterpret_cast<const uint16_t*>(&v), p); }
};

// SHARED: the values between the passes in shared memory.
template <int KIND, class XT, int C, bool VEC, bool WARP, bool SHARED>
__global__ void __launch_bounds__(WARP ? 128 : SHARED ? 512 : 1024, SHARED ? 3 : 1)
    k_row_quant(const RowArgs a) {
  extern __shared__ float4 shared[];  // SHARED: [chunk][half][thread]
  __shared__ double sums[32];
  __shared__ uint64_t tops64[32];
  __shared__ uint32_t tops[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t row = WARP ? (int64_t)blockIdx.x * warps + warp : blockIdx.x;
  const int tid = WARP ? lane : threadIdx.x, team = WARP ? 32 : blockDim.x;
  pdl_wait();
  pdl_launch();
  if (WARP && row >= a.rows) return;
  Row<KIND, XT> r;
  r.x = static_cast<const XT*>(a.x) + row * a.x_stride;
  r.residual = KIND == kNorm && a.residual ? a.residual + row * a.residual_stride : nullptr;
  r.total = KIND == kNorm && a.total ? a.total + row * a.total_stride : nullptr;
  r.gamma = a.gamma;
  r.width = a.width;
  int8_t* const q = a.q + row * a.q_stride;

  // ---- the row, its largest f32 value and its sum of squares
  constexpr int kHeld = VEC && !SHARED ? C : 1;
  Held<KIND, XT> held[kHeld];
  auto keep = [&](int c, const float* p) {
    if constexpr (SHARED) {
      shared[2 * c * team + tid] = make_float4(p[0], p[1], p[2], p[3]);
      shared[(2 * c + 1) * team + tid] = make_float4(p[4], p[5], p[6], p[7]);
    } else if constexpr (KIND != kQuant || sizeof(XT) == 4) {
      held[c].keep(p);
    }
  };
  auto take = [&](int c, float* p) {
    if constexpr (SHARED) {
      const float4 x = shared[2 * c * team + tid], y = shared[(2 * c + 1) * team + tid];
      p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w, p[4] = y.x, p[5] = y.y, p[6] = y.z, p[7] = y.w;
    } else {
      held[c].take(p);
    }
  };
  double squares = 0.0;
  float largest = 0.0f;
  if constexpr (VEC) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (c * team + tid) * 8;
      float p[8];
      if constexpr (KIND == kQuant && sizeof(XT) == 2) {
        held[c].v = i + 8 <= a.width ? *reinterpret_cast<const uint4*>(r.x + i)
                                     : some8(r.x + i, a.width - i);
        held[c].take(p);
      } else {
        if (i + 8 <= a.width) {
          r.template values<true>(i, 8, p, squares);
        } else {
          r.template values<false>(i, a.width - i, p, squares);
        }
        keep(c, p);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = larger(largest, p[e]);
    }
  } else {
    for (int i = tid; i < a.width; i += team) {
      if (KIND == kNorm) {
        const float t = r.residual ? __fadd_rn(get(r.x + i), r.residual[i]) : get(r.x + i);
        if (r.total) r.total[i] = t;
        squares += (double)t * (double)t;
      }
      largest = larger(largest, r.value(i));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (KIND == kNorm) squares += __shfl_xor_sync(0xffffffffu, squares, o);
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(largest) & 0x7fffffffu);
  if (!WARP) {
    if (lane == 0) {
      sums[warp] = squares;
      tops[warp] = top;
    }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? tops[lane] : 0u);
    if (KIND == kNorm) {
      squares = lane < warps ? sums[lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    }
  }
  const double inv = KIND == kNorm ? rsqrt(squares / a.width + (double)a.eps) : 1.0;
  const float P = __uint_as_float(top);
  // A SwiGLU's f32 value may pass f32's range where y does not, and the other way round.
  const bool finite = KIND == kSwiglu ? top <= 0x7f800000u : top < 0x7f800000u;
  // Nothing but zeros: scale 2^-126. (A product below f32's smallest number is 0
  // as well, and a norm may still make it large.)
  const bool zero = top == 0 && (KIND != kNorm || (squares == 0.0 && inv < 1e300));
  const bool all64 = P < kTiny || (KIND == kSwiglu && P == INFINITY);  // the steps all in f64

  // the place of this thread's value n
  auto place = [&](int n) { return ((n >> 3) * team + tid) * 8 + (n & 7); };

  // ---- the largest value in 64 bits, of those that may be it
  uint64_t most = 0;
  if (KIND != kQuant && finite && !zero) {
    const float least =
        P < kTiny ? 0.0f : fminf(P, 3.40282347e38f) * (1.0f - 2.0f * kRel<KIND>);
    if constexpr (VEC) {
      uint32_t may = 0;  // (most threads have none)
      if (largest >= least) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float p[8];
          take(c, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) may |= fabsf(p[e]) >= least ? 1u << (8 * c + e) : 0u;
        }
      }
      while (may) {
        const int i = place(__ffs(may) - 1);
        may &= may - 1;
        if (i < a.width) most = max(most, magnitude(r.exact(i, inv)));
      }
    } else {
      for (int i = tid; i < a.width; i += team)
        if (fabsf(r.value(i)) >= least) most = max(most, magnitude(r.exact(i, inv)));
    }
    most = warp_most(most);
    if (!WARP) {
      if (lane == 0) tops64[warp] = most;
      __syncthreads();
      most = warp_most(lane < warps ? tops64[lane] : 0);
    }
  }
  float scale = fmaxf(KIND == kQuant ? __fdiv_rn(P, 127.0f)
                                     : (float)over127(__longlong_as_double((long long)most)),
                      kSmallest);
  // fmaxf passes a NaN over
  if (!finite || most >= kPast) scale = __uint_as_float(0x7fc00000u);
  if (tid == 0) a.scales[row] = scale;

  // ---- the steps
  const bool good = scale == scale;
  const float per = KIND == kNorm ? (float)(inv / (double)scale) : __frcp_rn(scale);
  // Value i by its f32 value p: on which side of the nearest border it lies, exactly
  // (a border times the scale has 32 bits; plain rows compare through one fma's sign).
  auto decide = [&](int i, float p) {
    if (all64) return (int)rint(r.exact(i, inv) / (double)scale);
    const float v = p * per, border = floorf(v) + 0.5f;
    float side;
    if (KIND == kQuant) {
      side = __fmaf_rn(-border, scale, p);
    } else {
      const double d = r.exact(i, inv) - (double)border * (double)scale;
      side = d > 0.0 ? 1.0f : d < 0.0 ? -1.0f : 0.0f;
    }
    const int below = (int)floorf(border);
    return side > 0.0f || (side == 0.0f && (below & 1)) ? below + 1 : below;
  };
  if constexpr (VEC) {
    uint32_t unsure = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (c * team + tid) * 8;
      if (i >= a.width) break;
      uint32_t s[8] = {};
      float p[8], edge = 0.0f;
      take(c, p);
      if (good && !zero) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = step<KIND>(p[e], per, edge);
        if (all64) {
          unsure |= 255u << (8 * c);
        } else if (open<KIND>(edge)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float one = 0.0f;
            step<KIND>(p[e], per, one);
            unsure |= open<KIND>(one) ? 1u << (8 * c + e) : 0u;
          }
        }
      }
      if (i + 8 <= a.width) {
        uint2 w;
        w.x = __byte_perm(__byte_perm(s[0], s[1], 0x0040), __byte_perm(s[2], s[3], 0x0040), 0x5410);
        w.y = __byte_perm(__byte_perm(s[4], s[5], 0x0040), __byte_perm(s[6], s[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2*>(q + i) = w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < a.width) q[i + e] = (int8_t)s[e];
      }
    }
    while (unsure) {
      const int i = place(__ffs(unsure) - 1);
      unsure &= unsure - 1;
      if (i < a.width) q[i] = (int8_t)decide(i, r.value(i));
    }
  } else {
    for (int i = tid; i < a.width; i += team) {
      const float p = r.value(i);
      float edge = 0.0f;
      const uint32_t n = step<KIND>(p, per, edge);
      q[i] = (int8_t)(!good || zero ? 0 : open<KIND>(edge) || all64 ? decide(i, p) : (int)n);
    }
  }
}

template <int KIND, class XT, int C, bool VEC, bool WARP, bool SHARED = false>
cudaError_t launch(const RowArgs& a, int threads, cudaStream_t st) {
  const int per = WARP ? threads / 32 : 1;
  const auto kernel = k_row_quant<KIND, XT, C, VEC, WARP, SHARED>;
  const size_t smem = SHARED ? (size_t)threads * C * 32 : 0;
  if (SHARED) {
    static std::atomic<uint64_t> raised{0};
    const cudaError_t e = raise_smem_limit((const void*)kernel, 512 * C * 32, &raised);
    if (e != cudaSuccess) return e;
  }
  return counted(launch_pdl(kernel, dim3((unsigned)((a.rows + (int64_t)per - 1) / per)), threads,
                            smem, st, 1, a));
}

template <int KIND, class XT>
cudaError_t launch_kind(const RowArgs& a, bool vec, cudaStream_t st) {
  if (!vec || a.width > 32768) return launch<KIND, XT, 1, false, false>(a, 512, st);
  if (a.width <= 256) return launch<KIND, XT, 1, true, true>(a, 128, st);
  if (a.width <= 512) return launch<KIND, XT, 2, true, true>(a, 128, st);
  if (a.width <= 1024) return launch<KIND, XT, 4, true, true>(a, 128, st);
  const int chunks = (a.width + 7) / 8;
  // Few rows: as many threads as chunks, for the latency. Many: more chunks a thread,
  // so that more rows are on their way at once (norm of 8191 x 5120 f32 with 1, 2, 4:
  // 104, 92, 87 us; of 8191 x 1536: 33, 29, 34 us; of 512 x 5120: 10.7, 10.6, 10.3 us; of
  // 64 x 5120: 3.8, 3.9, 4.5 us; rows 27648 x 5120 bf16: 168, 111, 93 us).
  const int many = a.rows < 512 ? 1 : chunks <= 256 ? 2 : 4;
  const int each = chunks > 2048 || many == 4 ? 4 : chunks > 1024 || many == 2 ? 2 : 1;
  const int threads = (chunks + 32 * each - 1) / (32 * each) * 32;
  if (each == 1) return launch<KIND, XT, 1, true, false>(a, threads, st);
  if (each == 2) return launch<KIND, XT, 2, true, false>(a, threads, st);
  // SwiGLU's values in shared memory: 40 registers a thread (20 words of it spilled),
  // three rows at once where held in registers there were two (4099 x 13824 bf16: 91, 85
  // us; f32: 110, 106; 512 x 8960 f32: 14.3, 13.4).
  if constexpr (KIND == kSwiglu)
    if (many == 4 && chunks <= 2048) return launch<KIND, XT, 4, true, false, true>(a, threads, st);
  return launch<KIND, XT, 4, true, false>(a, threads, st);
}

// The checks that the three calls share, and the launch.
template <int KIND>
int row_quant(RowArgs a, int32_t x_dtype, size_t q_stride, size_t x_stride, size_t rows,
              size_t width, void* stream) {
  if (x_dtype != MYOS_F32 && x_dtype != MYOS_BF16) return MYOS_ERR_ARG;
  if (rows == 0) return MYOS_OK;
  if (!a.q || !a.scales || !a.x) return MYOS_ERR_ARG;
  const size_t most = (size_t)1 << 40, in = KIND == kSwiglu ? 2 * width : width;
  if (rows > 0x7fffffff || width == 0 || width > MYOS_I8_MAX_K || q_stride < width ||
      x_stride < in || q_stride > most || x_stride > most)
    return MYOS_ERR_SHAPE;
  const size_t size = x_dtype == MYOS_F32 ? 4 : 2;
  if (!aligned(a.x, size) || !aligned(a.scales, 4)) return MYOS_ERR_ARG;
  a.q_stride = (int64_t)q_stride;
  a.x_stride = (int64_t)x_stride;
  a.rows = (int)rows;
  a.width = (int)width;
  // whole vectors: 8 bytes of q, 16 of everything else (one row has no stride)
  bool vec = aligned(a.q, 8) && aligned(a.x, 16) && aligned(a.gamma, 16) &&
             aligned(a.residual, 16) && aligned(a.total, 16);
  if (rows > 1)
    vec &= q_stride % 8 == 0 && x_stride * size % 16 == 0 && a.residual_stride % 4 == 0 &&
           a.total_stride % 4 == 0;
  if (KIND == kSwiglu) vec &= width * size % 16 == 0;  // the up values
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = x_dtype == MYOS_F32 ? launch_kind<KIND, float>(a, vec, st)
                                            : launch_kind<KIND, uint16_t>(a, vec, st);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}

}  // namespace
}  // namespace myos

using namespace myos;

extern "C" {

int myos_dev_add_norm_quant(int8_t* d_q, size_t q_stride, float* d_scales, float* d_total,
                            size_t total_stride, const void* d_x, int32_t x_dtype, size_t x_stride,
                            const float* d_residual, size_t residual_stride, const void* d_gamma,
                            float eps, size_t rows, size_t width, void* stream) {
  if (rows > 0) {
    if (!d_gamma || !(eps >= 0.0f)) return MYOS_ERR_ARG;
    if (!aligned(d_gamma, 2) || !aligned(d_residual, 4) || !aligned(d_total, 4)) return MYOS_ERR_ARG;
    const size_t most = (size_t)1 << 40;
    if ((d_residual && (residual_stride < width || residual_stride > most)) ||
        (d_total && (total_stride < width || total_stride > most)))
      return MYOS_ERR_SHAPE;
    if (d_total && rows > 1 &&
        ((d_total == d_residual && total_stride != residual_stride) ||
         (d_total == d_x && total_stride != x_stride)))
      return MYOS_ERR_ARG;
    if (d_total && d_total == d_x && x_dtype != MYOS_F32) return MYOS_ERR_ARG;
  }
  RowArgs a = {};
  a.q = d_q;
  a.scales = d_scales;
  a.x = d_x;
  a.residual = d_residual;
  a.residual_stride = d_residual ? (int64_t)residual_stride : 0;
  a.total = d_total;
  a.total_stride = d_total ? (int64_t)total_stride : 0;
  a.gamma = static_cast<const uint16_t*>(d_gamma);
  a.eps = eps;
  return row_quant<kNorm>(a, x_dtype, q_stride, x_stride, rows, width, stream);
}

int myos_dev_quant_rows(int8_t* d_q, size_t q_stride, float* d_scales, const void* d_x,
                        int32_t x_dtype, size_t x_stride, size_t rows, size_t width, void* stream) {
  RowArgs a = {};
  a.q = d_q;
  a.scales = d_scales;
  a.x = d_x;
  return row_quant<kQuant>(a, x_dtype, q_stride, x_stride, rows, width, stream);
}

int myos_dev_swiglu_quant(int8_t* d_q, size_t q_stride, float* d_scales, const void* d_x,
                          int32_t x_dtype, size_t x_stride, size_t rows, size_t width,
                          void* stream) {
  RowArgs a = {};
  a.q = d_q;
  a.scales = d_scales;
  a.x = d_x;
  return row_quant<kSwiglu>(a, x_dtype, q_stride, x_stride, rows, width, stream);
}

}  // extern "C"
