// Attention of one new token per sequence over a paged KV cache.
//
// out = softmax(scale q K^T) V in one pass over the keys: a running maximum m,
// sum l and weighted output o per query head, joined across warps, and across
// blocks where a sequence is split, by rescaling to the common maximum.
//
// The work is memory: every key and value is read once for the whole group of
// query heads that share it. All (sequence, KV head) items are cut into tiles
// of keys, and the tiles, in one row, into equal shares, one per block: the
// lengths live on the device, so each block finds its share itself from a scan
// of them, and no split has to be chosen on the host. An item that lies in one
// share is finished there; else each block leaves its part in the work buffer
// and the last to arrive joins them, in the order of the shares (the same bits
// whoever is last). A block has at most two parts, its first and its last
// piece, so the buffer's size does not depend on the batch.
//
// Each warp streams keys of its own through its own stages of shared memory
// (cp.async, three deep, pages looked up one tile ahead), so warps never wait
// for one another inside an item.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace myos {
namespace {

constexpr int kMaxGroup = 8;  // query heads per KV head, as tensor_core::gqa_attn_f32 here
constexpr int kMaxShares = 592;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct PagedAttnArgs {
  float* out;
  float* lse;
  const float* q;
  int64_t out_stride, q_stride;
  int nseq, hq, group;
  const int32_t* table;
  int64_t table_stride, max_keys;
  const int32_t* kv_lens;
  float scale2;  // scale * log2(e): scores are kept in powers of two
  uint32_t window;
  int page_shift;  // log2 of the page size, or -1
  unsigned* arrived;  // [shares], zero between launches
  float* parts;       // [shares][2][8 * DH + 16]
};

MYOS_DEV void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
MYOS_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
MYOS_DEV void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

MYOS_DEV void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
MYOS_DEV void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// c += A B, A 16 x 16 (rows 0-7 in a0, a2, rows 8-15 in a1, a3), B 16 x 8.
MYOS_DEV void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                       uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// x = hi + mid + lo, exactly: three times the leading 8 significand bits, by
// truncation (two values at a time, packed as bf16 pairs).
struct Split3 {
  uint32_t hi, mid, lo;
};
MYOS_DEV float top_bits(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
MYOS_DEV uint32_t pack_top(float x, float y) {
  return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}
MYOS_DEV Split3 split3(float x, float y) {
  Split3 s;
  s.hi = pack_top(x, y);
  x -= top_bits(x);
  y -= top_bits(y);
  s.mid = pack_top(x, y);
  x -= top_bits(x);
  y -= top_bits(y);
  s.lo = pack_top(x, y);
  return s;
}

// Rescaling of a part with maximum m to the common maximum top.
MYOS_DEV float weight_of(float m, float top) { return top == -INFINITY ? 0.f : exp2f(m - top); }

// ---------------------------------------------------------- a warp's state
// bf16 cache: 16 keys a tile through mma. The A operand's 16 rows hold the
// group's (at most 8) heads twice, the hi terms in rows 0-7 and the mid terms
// in rows 8-15, and a second mma adds the lo terms, so the f32 queries and
// weights enter exactly; a lane's c0, c1 and c2, c3 belong to the same head
// (lane / 4). The tensor core truncates its f32 sums, so no long chain runs
// through it: four steps of a score, one tile of an output, the rest are f32
// adds, rounded to nearest.
template <int DH>
struct MmaWarp {
  static constexpr int kKeys = 16, kRegs = DH / 4, kSteps = DH / 16;
  using KT = __nv_bfloat16;
  Split3 q[kSteps][2];
  float o[kRegs];
  float m, l;

  MYOS_DEV void begin(const float* q_row, int G, int d) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = 16 * k + 8 * u + c;
        float2 x = make_float2(0.f, 0.f);
        if (g < G && at < d) x = *reinterpret_cast<const float2*>(q_row + g * d + at);
        q[k][u] = split3(x.x, x.y);
      }
#pragma unroll
    for (int r = 0; r < kRegs; ++r) o[r] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  // Chunks of 16 bytes; row r keeps chunk i at i ^ (r & 7): the eight rows
  // that an ldmatrix reads at one chunk lie in different banks.
  static MYOS_DEV int place(int row, int chunk) { return row * (DH / 8) + (chunk ^ (row & 7)); }

  MYOS_DEV void tile(uint32_t ks, uint32_t vs, uint32_t ok, float scale2) {
    const int lane = threadIdx.x & 31, c = (lane & 3) * 2;
    float s[4];
    {
      float a[2][2][4], lo[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[n][0][i] = a[n][1][i] = lo[n][i] = 0.f;
      const int row = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t b[4];
        ldmatrix4(b, ks + 16 * place(row, 2 * k + half));
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          mma16816(lo[n], q[k][0].lo, 0u, q[k][1].lo, 0u, b[2 * n], b[2 * n + 1]);
          mma16816(a[n][(k >> 2) & 1], q[k][0].hi, q[k][0].mid, q[k][1].hi, q[k][1].mid, b[2 * n],
                   b[2 * n + 1]);
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = (a[n][0][i] + a[n][1][i]) + ((a[n][0][i + 2] + a[n][1][i + 2]) + lo[n][i]);
          s[2 * n + i] = (ok >> (8 * n + c + i)) & 1u ? x * scale2 : -INFINITY;
        }
    }
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = fmaxf(top, m);  // finite: the tile has a key
    const float keep = exp2f(m - top);
    m = top;
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = exp2f(s[i] - top);
    l = fmaf(l, keep, (p[0] + p[1]) + (p[2] + p[3]));
    const Split3 w0 = split3(p[0], p[1]), w1 = split3(p[2], p[3]);
    const int row = lane & 15, half = lane >> 4;
#pragma unroll
    for (int j = 0; j < DH / 16; ++j) {
      uint32_t b[4];
      ldmatrix4t(b, vs + 16 * place(row, 2 * j + half));
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816(t, w0.lo, 0u, w1.lo, 0u, b[2 * n], b[2 * n + 1]);
        mma16816(t, w0.hi, w0.mid, w1.hi, w1.mid, b[2 * n], b[2 * n + 1]);
        float* x = &o[4 * j + 2 * n];
        x[0] = fmaf(x[0], keep, t[0] + t[2]);
        x[1] = fmaf(x[1], keep, t[1] + t[3]);
      }
    }
  }

  // Sums over the lanes of a head, once per piece.
  MYOS_DEV void finish() {
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
  }
  MYOS_DEV void put_ml(float* ms, float* ls) const {
    const int lane = threadIdx.x & 31;
    if ((lane & 3) == 0) {
      ms[lane >> 2] = m;
      ls[lane >> 2] = l;
    }
  }
  // o of a part (regs apart by 32 lanes) into this state; m, l per head.
  MYOS_DEV void join(const float* part, const float* ms, const float* ls) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const float pm = ms[g], top = fmaxf(m, pm);
    const float a = weight_of(m, top), b = weight_of(pm, top);
    m = top;
    l = l * a + ls[g] * b;
#pragma unroll
    for (int r = 0; r < kRegs; r += 4) {
      const float4 x = *reinterpret_cast<const float4*>(part + r * 32 + lane * 4);
      o[r] = o[r] * a + x.x * b;
      o[r + 1] = o[r + 1] * a + x.y * b;
      o[r + 2] = o[r + 2] * a + x.z * b;
      o[r + 3] = o[r + 3] * a + x.w * b;
    }
  }
  MYOS_DEV void write(float* out, float* lse, int G, int d) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = (lane & 3) * 2;
    if (g >= G) return;
    const float inv = l > 0.f ? __fdiv_rn(1.0f, l) : 0.f;
#pragma unroll
    for (int j = 0; j < DH / 8; ++j)
      if (8 * j < d)
        *reinterpret_cast<float2*>(out + g * d + 8 * j + c) =
            make_float2(o[2 * j] * inv, o[2 * j + 1] * inv);
    if (lse && c == 0) lse[g] = l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
  }
};

// f32 cache: 8 keys a tile on the FMA units; a lane holds DH / 32 dims of
// every head. The products of 32 (head, key) pairs are summed over the lanes
// by a halving exchange that leaves one pair in each lane.
template <int DH, int GP>
struct FmaWarp {
  static constexpr int kKeys = 8, kDims = DH / 32, kRegs = GP * kDims;
  static constexpr int kVec = kDims < 4 ? kDims : 4, kJ = 32 / GP;  // kJ keys at a time
  using KT = float;
  float q[GP][kDims];
  float o[kRegs];
  float m[GP], l[GP];

  // dims of a lane: kVec at lane * kVec, then (DH 256) at 128 + lane * kVec
  static MYOS_DEV int dim(int i) { return (i / kVec) * 32 * kVec + (threadIdx.x & 31) * kVec + i % kVec; }

  MYOS_DEV void begin(const float* q_row, int G, int d) {
#pragma unroll
    for (int g = 0; g < GP; ++g) {
#pragma unroll
      for (int i = 0; i < kDims; ++i) {
        q[g][i] = g < G && dim(i) < d ? q_row[g * d + dim(i)] : 0.f;
        o[g * kDims + i] = 0.f;
      }
      m[g] = -INFINITY;
      l[g] = 0.f;
    }
  }
  static MYOS_DEV int place(int row, int chunk) { return row * (DH / 4) + chunk; }

  static MYOS_DEV void row_of(float (&x)[kDims], uint32_t base, int row) {
    const uint32_t at = base + (row * DH + (threadIdx.x & 31) * kVec) * 4;
    if constexpr (kVec == 2) {
      asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(x[0]), "=f"(x[1]) : "r"(at) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < kDims; i += 4)
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                     : "=f"(x[i]), "=f"(x[i + 1]), "=f"(x[i + 2]), "=f"(x[i + 3])
                     : "r"(at + i * 128)
                     : "memory");
    }
  }

  MYOS_DEV void tile(uint32_t ks, uint32_t vs, uint32_t ok, float scale2) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j0 = 0; j0 < kKeys; j0 += kJ) {
      const uint32_t now = (ok >> j0) & ((1u << kJ) - 1u);
      if (now == 0) continue;
      float d[32];  // (head, key) pair g * kJ + j
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        float x[kDims];
        row_of(x, ks, j0 + j);
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < kDims; ++i) s = fmaf(q[g][i], x[i], s);
          d[g * kJ + j] = s;
        }
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) {
        const bool up = (lane & w) != 0;
#pragma unroll
        for (int i = 0; i < w; ++i) {
          const float give = up ? d[i] : d[i + w];
          const float have = up ? d[i + w] : d[i];
          d[i] = have + __shfl_xor_sync(0xffffffffu, give, w);
        }
      }
      // lane g * kJ + j has the score of head g, key j0 + j
      const float s = (now >> (lane % kJ)) & 1u ? d[0] * scale2 : -INFINITY;
      float top = s;
#pragma unroll
      for (int w = 1; w < kJ; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      float keep[GP];
      float mine = -INFINITY;
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float t = fmaxf(m[g], __shfl_sync(0xffffffffu, top, g * kJ));
        keep[g] = exp2f(m[g] - t);
        m[g] = t;
        if (lane / kJ == g) mine = t;
      }
      const float p = exp2f(s - mine);
      float w[GP][kJ];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          w[g][j] = __shfl_sync(0xffffffffu, p, g * kJ + j);
          t += w[g][j];
        }
        l[g] = fmaf(l[g], keep[g], t);
#pragma unroll
        for (int i = 0; i < kDims; ++i) o[g * kDims + i] *= keep[g];
      }
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        float x[kDims];
        row_of(x, vs, j0 + j);
#pragma unroll
        for (int g = 0; g < GP; ++g)
#pragma unroll
          for (int i = 0; i < kDims; ++i) o[g * kDims + i] = fmaf(w[g][j], x[i], o[g * kDims + i]);
      }
    }
  }
  MYOS_DEV void finish() {}
  MYOS_DEV void put_ml(float* ms, float* ls) const {
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        ms[g] = m[g];
        ls[g] = l[g];
      }
  }
  MYOS_DEV void join(const float* part, const float* ms, const float* ls) {
    const int lane = threadIdx.x & 31;
    float a[GP], b[GP];
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      const float pm = ms[g], top = fmaxf(m[g], pm);
      a[g] = weight_of(m[g], top);
      b[g] = weight_of(pm, top);
      m[g] = top;
      l[g] = l[g] * a[g] + ls[g] * b[g];
    }
#pragma unroll
    for (int r = 0; r < kRegs; r += 4) {
      const float4 x = *reinterpret_cast<const float4*>(part + r * 32 + lane * 4);
      const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int g = (r + i) / kDims;
        o[r + i] = o[r + i] * a[g] + y[i] * b[g];
      }
    }
  }
  MYOS_DEV void write(float* out, float* lse, int G, int d) const {
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      if (g >= G) break;
      const float inv = l[g] > 0.f ? __fdiv_rn(1.0f, l[g]) : 0.f;
#pragma unroll
      for (int i = 0; i < kDims; ++i)
        if (dim(i) < d) out[g * d + dim(i)] = o[g * kDims + i] * inv;
      if (lse && (threadIdx.x & 31) == 0)
        lse[g] = l[g] > 0.f ? (m[g] + log2f(l[g])) * kLn2 : -INFINITY;
    }
  }
};

// A tile of the row of all tiles: sequence b, KV head h, tile t of [t0, t1).
struct Cursor {
  int b, h, t, t0, t1, len, start;
};

template <int T>
MYOS_DEV void span_of(const PagedAttnArgs& a, int b, Cursor* c) {
  c->len = (int)min((int64_t)max(a.kv_lens[b], 0), a.max_keys);
  c->start = a.window > 0 && (uint32_t)c->len > a.window ? c->len - (int)a.window : 0;
  c->t0 = c->start / T;
  c->t1 = (c->len + T - 1) / T;
}

template <int T>
MYOS_DEV void advance(const PagedAttnArgs& a, int heads, Cursor* c) {
  if (++c->t < c->t1) return;
  if (++c->h == heads) {
    c->h = 0;
    do {
      if (++c->b >= a.nseq) {
        c->t0 = c->t1 = c->len = c->start = 0;
        break;
      }
      span_of<T>(a, c->b, c);
    } while (c->t0 >= c->t1);
  }
  c->t = c->t0;
}

constexpr int kStages = 3, kWarps = 4;

template <class W, int DH>
constexpr size_t attn_smem() {
  return (size_t)kStages * kWarps * 2 * W::kKeys * DH * sizeof(typename W::KT) +
         (kWarps - 1) * W::kRegs * 32 * 4;
}

template <class W, int DH>
__global__ void __launch_bounds__(kWarps * 32)
    k_paged_attn(const PagedAttnArgs a, const PagedKv<typename W::KT> kv) {
  using KT = typename W::KT;
  constexpr int T = W::kKeys * kWarps, kThreads = kWarps * 32;
  constexpr int kRowBytes = DH * (int)sizeof(KT), kHalf = W::kKeys * kRowBytes;
  constexpr int kPart = kMaxGroup * DH + 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float ms[kWarps][kMaxGroup], ls[kWarps][kMaxGroup];
  __shared__ uint32_t okay[kWarps][kStages];
  __shared__ int64_t sums[33];
  __shared__ Cursor first_s;
  __shared__ int last_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = (int)kv.heads, G = a.group, d = (int)kv.d;
  const int64_t me = blockIdx.x;
  float* swap = reinterpret_cast<float*>(smem + (size_t)kStages * kWarps * 2 * kHalf);

  // this block's share [lo, hi) of the tiles, and where it begins
  const int per = (a.nseq + kThreads - 1) / kThreads;
  const int b0 = min(a.nseq, (int)threadIdx.x * per), b1 = min(a.nseq, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    Cursor c;
    span_of<T>(a, b, &c);
    mine += c.t1 - c.t0;
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += sums[w];
    total += sums[w];
  }
  total *= heads;
  // as many shares as blocks, or as tiles if those are fewer: none is empty
  const int64_t n = max((int64_t)1, min((int64_t)gridDim.x, total));
  const int64_t lo = min(total, me * total / n), hi = min(total, (me + 1) * total / n);
  if (lo < hi && (upto - mine) * heads <= lo && lo < upto * heads) {
    int64_t at = (upto - mine) * heads;
    Cursor c;
    int b = b0;
    for (;; ++b) {
      span_of<T>(a, b, &c);
      const int64_t next = at + (int64_t)(c.t1 - c.t0) * heads;
      if (lo < next) break;
      at = next;
    }
    c.b = b;
    c.h = (int)((lo - at) / (c.t1 - c.t0));
    c.t = c.t0 + (int)((lo - at) % (c.t1 - c.t0));
    first_s = c;
  }
  // sequences without a key have no tile: their outputs are spread over the blocks
  for (int b = (int)me; b < a.nseq; b += (int)gridDim.x) {
    Cursor c;
    span_of<T>(a, b, &c);
    if (c.t0 < c.t1) continue;
    for (int i = threadIdx.x; i < a.hq * d; i += kThreads) a.out[b * a.out_stride + i] = 0.f;
    if (a.lse)
      for (int i = threadIdx.x; i < a.hq; i += kThreads) a.lse[(int64_t)b * a.hq + i] = -INFINITY;
  }
  __syncthreads();
  if (lo >= hi) return;

  Cursor ahead = first_s, c = first_s;
  const uint32_t stage0 = smem_u32(smem) + warp * 2 * kHalf;
  // the page of this lane's key in a tile (lanes past the tile's keys: none)
  auto look = [&](const Cursor& x) -> int {
    const int key = x.t * T + warp * W::kKeys + lane;
    if (lane >= W::kKeys || key < x.start || key >= x.len) return -1;
    const int pg = a.page_shift >= 0 ? key >> a.page_shift : key / (int)kv.page_size;
    return a.table[x.b * a.table_stride + pg];
  };
  auto issue = [&](const Cursor& x, int page, int stage) {
    const int key = x.t * T + warp * W::kKeys + lane;
    const bool on = page >= 0 && (uint32_t)page < kv.num_pages;
    const int in = a.page_shift >= 0 ? key & ((1 << a.page_shift) - 1) : key % (int)kv.page_size;
    const int64_t off =
        on ? page * kv.page_stride + x.h * kv.head_stride + in * kv.slot_stride : -1;
    const uint32_t ok = __ballot_sync(0xffffffffu, on);
    if (lane == 0) okay[warp][stage] = ok;
    constexpr int kChunks = kRowBytes / 16, kEach = 16 / (int)sizeof(KT);
    const uint32_t dst = stage0 + stage * (kWarps * 2 * kHalf);
#pragma unroll
    for (int i = 0; i < W::kKeys * kChunks / 32; ++i) {
      const int row = (i * 32 + lane) / kChunks, ch = (i * 32 + lane) % kChunks;
      const int64_t from = __shfl_sync(0xffffffffu, off, row);
      const bool load = from >= 0 && ch * kEach < d;
      const int64_t at = load ? from + ch * kEach : 0;
      const uint32_t to = dst + 16 * W::place(row, ch);
      cp_async16(to, kv.k + at, load);
      cp_async16(to + kHalf, kv.v + at, load);
    }
  };
  int page = look(ahead);
  int64_t next = lo;  // the tile that is copied next; `page` belongs to it
  auto step = [&]() {
    if (next < hi) {
      const Cursor x = ahead;
      const int pg = page;
      advance<T>(a, heads, &ahead);
      if (next + 1 < hi) page = look(ahead);
      issue(x, pg, (int)((next - lo) % kStages));
    }
    cp_commit();
    ++next;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) step();

  W w;
  for (int64_t i = lo; i < hi; ++i) {
    if (i == lo || c.t == c.t0)
      w.begin(a.q + c.b * a.q_stride + (int64_t)c.h * G * d, G, d);
    cp_wait<kStages - 2>();
    __syncwarp();
    step();
    const int stage = (int)((i - lo) % kStages);
    const uint32_t ok = okay[warp][stage];
    const uint32_t base = stage0 + stage * (kWarps * 2 * kHalf);
    if (ok) w.tile(base, base + kHalf, ok, a.scale2);
    __syncwarp();
    if (c.t + 1 == c.t1 || i + 1 == hi) {
      // the piece's end: the warps' states into warp 0's
      w.finish();
      __syncthreads();  // the swap space of the piece before is free
      w.put_ml(ms[warp], ls[warp]);
      if (warp > 0) {
        float* s = swap + (warp - 1) * W::kRegs * 32;
#pragma unroll
        for (int r = 0; r < W::kRegs; r += 4)
          *reinterpret_cast<float4*>(s + r * 32 + lane * 4) =
              make_float4(w.o[r], w.o[r + 1], w.o[r + 2], w.o[r + 3]);
      }
      __syncthreads();
      const int64_t i0 = i - (c.t - c.t0), i1 = i0 + (c.t1 - c.t0);
      const bool whole = i0 >= lo && i1 <= hi;
      if (warp == 0)
#pragma unroll 1
        for (int u = 1; u < kWarps; ++u) w.join(swap + (u - 1) * W::kRegs * 32, ms[u], ls[u]);
      if (!whole) {
        const int64_t c0 = ((i0 + 1) * n - 1) / total, c1 = (i1 * n - 1) / total;
        if (warp == 0) {
          float* part = a.parts + (me * 2 + (i0 < lo ? 0 : 1)) * kPart;
          w.put_ml(part, part + kMaxGroup);
          part += 16;
#pragma unroll
          for (int r = 0; r < W::kRegs; r += 4)
            *reinterpret_cast<float4*>(part + r * 32 + lane * 4) =
                make_float4(w.o[r], w.o[r + 1], w.o[r + 2], w.o[r + 3]);
          __threadfence();
          __syncwarp();
          if (lane == 0) {
            const unsigned before = atomicAdd(&a.arrived[c0], 1u);
            last_s = before == (unsigned)(c1 - c0);
            if (last_s) a.arrived[c0] = 0;
          }
          __threadfence();
        }
        __syncthreads();
        if (last_s) {
          // the parts in the order of their shares, a run of them for each warp
          __threadfence();
          const int64_t count = c1 - c0 + 1, run = (count + kWarps - 1) / kWarps;
          const int64_t p0 = c0 + min(count, warp * run), p1 = c0 + min(count, (warp + 1) * run);
          w.begin(a.q, 0, 0);
          for (int64_t p = p0; p < p1; ++p) {
            const float* part = a.parts + (p * 2 + (i0 < p * total / n ? 0 : 1)) * kPart;
            w.join(part + 16, part, part + kMaxGroup);
          }
          w.put_ml(ms[warp], ls[warp]);
          if (warp > 0) {
            float* s = swap + (warp - 1) * W::kRegs * 32;
#pragma unroll
            for (int r = 0; r < W::kRegs; r += 4)
              *reinterpret_cast<float4*>(s + r * 32 + lane * 4) =
                  make_float4(w.o[r], w.o[r + 1], w.o[r + 2], w.o[r + 3]);
          }
          __syncthreads();
          if (warp == 0)
#pragma unroll 1
            for (int u = 1; u < kWarps; ++u) w.join(swap + (u - 1) * W::kRegs * 32, ms[u], ls[u]);
        }
      }
      if (warp == 0 && (whole || last_s))
        w.write(a.out + c.b * a.out_stride + (int64_t)c.h * G * d,
                a.lse ? a.lse + (int64_t)c.b * a.hq + c.h * G : nullptr, G, d);
    }
    advance<T>(a, heads, &c);
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <class W, int DH>
cudaError_t launch(PagedAttnArgs a, const myos_paged_kv* kv, void* work, cudaStream_t st) {
  constexpr size_t smem = attn_smem<W, DH>();
  constexpr int T = W::kKeys * kWarps;
  static_assert(256 * 4 * 16 + (size_t)kMaxShares * 2 * (kMaxGroup * DH + 16) * 4 <=
                MYOS_PAGED_WORK_BYTES);
  cudaError_t e = cudaFuncSetAttribute(k_paged_attn<W, DH>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  a.arrived = static_cast<unsigned*>(work);
  a.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + 256 * 4 * 16);
  // a share per resident block, and never more shares than there can be tiles
  int64_t keys = a.max_keys;
  if (a.window > 0 && (int64_t)a.window + T < keys) keys = (int64_t)a.window + T;
  const int64_t most = (int64_t)a.nseq * kv->num_kv_heads * ((keys + T - 1) / T);
  int64_t grid = (int64_t)sm_count() * (smem <= 110 * 1024 ? 2 : 1);
  if (grid > kMaxShares) grid = kMaxShares;
  if (grid > most) grid = most;
  k_paged_attn<W, DH><<<(int)grid, kWarps * 32, smem, st>>>(a, paged_view<typename W::KT>(kv));
  return counted(cudaGetLastError());
}

template <int DH>
cudaError_t launch_d(const PagedAttnArgs& a, const myos_paged_kv* kv, void* work,
                     cudaStream_t st) {
  if (kv->kv_dtype == MYOS_KV_BF16) return launch<MmaWarp<DH>, DH>(a, kv, work, st);
  return a.group <= 4 ? launch<FmaWarp<DH, 4>, DH>(a, kv, work, st)
                      : launch<FmaWarp<DH, 8>, DH>(a, kv, work, st);
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
      max_blocks * kv->page_size > 0x7fffff00 || q_stride < num_q_heads * d ||
      out_stride < num_q_heads * d || q_stride > ((size_t)1 << 30) ||
      out_stride > ((size_t)1 << 30))
    return MYOS_ERR_SHAPE;
  if (!aligned(d_q, 16) || !aligned(d_out, 16) || q_stride % 4 != 0 || out_stride % 4 != 0 ||
      !aligned(d_lse, 4) || !aligned(d_block_table, 4) || !aligned(d_kv_lens, 4) ||
      !aligned(d_work, 16))
    return MYOS_ERR_ARG;
  if (work_bytes < MYOS_PAGED_WORK_BYTES) return MYOS_ERR_SCRATCH_LIMIT;
  PagedAttnArgs a = {};
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
  a.max_keys = (int64_t)(max_blocks * kv->page_size);
  a.kv_lens = d_kv_lens;
  a.scale2 = scale * kLog2e;
  a.window = window;
  a.page_shift = -1;
  if ((kv->page_size & (kv->page_size - 1)) == 0)
    for (a.page_shift = 0; (1u << a.page_shift) < kv->page_size;) ++a.page_shift;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = d <= 64    ? launch_d<64>(a, kv, d_work, st)
                        : d <= 128 ? launch_d<128>(a, kv, d_work, st)
                                   : launch_d<256>(a, kv, d_work, st);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}
