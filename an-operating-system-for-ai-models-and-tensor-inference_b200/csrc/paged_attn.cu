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
// share is finished there. Where there are blocks for two shares of every item,
// the items get equal numbers of shares, and neighbouring ones meet in a pair of
// blocks' shared memory. What is left in parts goes through the work buffer: the
// last block to arrive joins them, in the order of the shares (the same bits
// whoever is last). A block has at most two parts, its first and its last
// piece, so the buffer's size does not depend on the batch.
//
// Each warp streams keys of its own through its own stages of shared memory
// (cp.async, three deep, pages looked up two tiles ahead), so warps never wait
// for one another inside an item. A copy instruction takes 64 bytes of each of
// eight rows: a lane stays with one or two rows of a tile, and all its
// addresses are one base each and constants.
#include "common.cuh"
#include "cp_async.cuh"
#include "kernels.h"
#include "paged.h"

namespace myos {
namespace {

constexpr int kMaxGroup = 8;  // query heads per KV head, as tensor_core::gqa_attn_f32 here
constexpr int kMaxShares = 592;
constexpr int kStages = 3, kWarps = 4;
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
  uint32_t page_mul;  // key / page_size = key * page_mul >> page_shift, keys below 2^31
  int page_shift;
  unsigned* arrived;  // [shares], zero between launches
  float* parts;       // [shares][2][8 * DH + 16]
};

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

MYOS_DEV void mma16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// The same in tf32, A 16 x 8, B 8 x 8.
MYOS_DEV void mma1688(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                      uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
MYOS_DEV void lds4(float4& x, uint32_t addr) {
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(addr)
               : "memory");
}
MYOS_DEV unsigned arrive(unsigned* count) {
  unsigned before;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
  return before;
}
// All threads of the cluster; what was written before is seen after.
MYOS_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// An address of this block's shared memory in block `rank` of the cluster.
MYOS_DEV uint32_t in_block(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
MYOS_DEV float ldc(uint32_t addr) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
MYOS_DEV float4 ldc4(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(addr)
               : "memory");
  return x;
}
// Bits 0, 4, .., 28 next to each other.
MYOS_DEV uint32_t gather_rows(uint32_t x) {
  x &= 0x11111111u;
  x = (x | x >> 3) & 0x03030303u;
  x = (x | x >> 6) & 0x000f000fu;
  return (x | x >> 12) & 0xffu;
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

MYOS_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rescaling of a part with maximum m to the common maximum top.
MYOS_DEV float weight_of(float m, float top) { return top == -INFINITY ? 0.f : ex2(m - top); }

// ---------------------------------------------------------- a warp's state
// The group's (at most 8) heads are rows 0-7 of an mma's A operand, with the
// leading part of the f32 queries (or weights); rows 8-15 take the next part
// of the same heads, so a lane's c0, c1 and c2, c3 belong to one head
// (lane / 4) and are added up. The tensor core truncates its f32 sums, so no
// long chain runs through it: four steps of a score, one tile of an output;
// the rest are f32 adds, rounded to nearest. (The products with a side's last
// term, at most 2^-11 of the others, go through in one chain of all steps, 32 at
// most: what that cuts off is below 1/64 of a step of the scores' terms.)
//
// o[2 t + i] is value i of column tile t (8 of the head's dims).
template <int DH>
struct WarpState {
  static constexpr int kRegs = DH / 4;
  float o[kRegs];
  float m, l;

  MYOS_DEV void clear() {
#pragma unroll
    for (int r = 0; r < kRegs; ++r) o[r] = 0.f;
    m = -INFINITY;
    l = 0.f;
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
  // The meeting of a block's warps: warp u < kOwners ends with values
  // [u kOwn, (u + 1) kOwn) of o, summed over the warps in their order (m and l
  // in every warp). A warp first leaves the others' shares in `swap`,
  // kOwners * (kWarps - 1) blocks of kOwn * 32 floats.
  static constexpr int kOwners = kRegs / 8 < kWarps ? kRegs / 8 : kWarps, kOwn = kRegs / kOwners;
  MYOS_DEV void leave(float* ms, float* ls, float* swap) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    put_ml(ms + warp * kMaxGroup, ls + warp * kMaxGroup);
#pragma unroll
    for (int u = 0; u < kOwners; ++u) {
      if (u == warp) continue;
      float* to = swap + (u * (kWarps - 1) + (warp < u ? warp : warp - 1)) * kOwn * 32 + lane * 4;
#pragma unroll
      for (int r = 0; r < kOwn; r += 4)
        *reinterpret_cast<float4*>(to + r * 32) = make_float4(
            o[u * kOwn + r], o[u * kOwn + r + 1], o[u * kOwn + r + 2], o[u * kOwn + r + 3]);
    }
  }
  MYOS_DEV void meet(const float* ms, const float* ls, const float* swap, float (&own)[kOwn]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
    float top = -INFINITY, f[kWarps];
#pragma unroll
    for (int v = 0; v < kWarps; ++v) top = fmaxf(top, f[v] = ms[v * kMaxGroup + g]);
    l = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      f[v] = weight_of(f[v], top);
      l = fmaf(ls[v * kMaxGroup + g], f[v], l);
    }
    m = top;
    float mine[kOwn];
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      mine[r] = o[r];
#pragma unroll
      for (int u = 1; u < kOwners; ++u) mine[r] = warp == u ? o[u * kOwn + r] : mine[r];
      own[r] = 0.f;
    }
    const float* from = swap + warp * (kWarps - 1) * kOwn * 32 + lane * 4;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      if (v == warp) {
#pragma unroll
        for (int r = 0; r < kOwn; ++r) own[r] = fmaf(mine[r], f[v], own[r]);
        continue;
      }
#pragma unroll
      for (int r = 0; r < kOwn; r += 4) {
        const float4 x = *reinterpret_cast<const float4*>(from + r * 32);
        own[r] = fmaf(x.x, f[v], own[r]);
        own[r + 1] = fmaf(x.y, f[v], own[r + 1]);
        own[r + 2] = fmaf(x.z, f[v], own[r + 2]);
        own[r + 3] = fmaf(x.w, f[v], own[r + 3]);
      }
      from += kOwn * 32;
    }
  }
  // Maximum and weights of a tile's scores s (in powers of two, -inf: no key;
  // the tile has one); the factor for what came before.
  template <int N>
  MYOS_DEV float weigh(float (&s)[N]) {
    float top = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, s[i]);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = fmaxf(top, m);
    const float keep = ex2(m - top);
    m = top;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) t += s[i] = ex2(s[i] - top);
    l = fmaf(l, keep, t);
    return keep;
  }
  // 1 / l, or 0 without a key. l is at least 1 (the largest weight), at most the
  // number of keys: an approximate reciprocal and one Newton step, no special cases.
  // A NaN query's l is NaN, and so are its out and lse.
  MYOS_DEV float inverse() const {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(l));
    return l == 0.f ? 0.f : fmaf(r, fmaf(-l, r, 1.0f), r);
  }
  MYOS_DEV void put_lse(float* lse, int G) const {
    const int lane = threadIdx.x & 31;
    if (lse && (lane & 3) == 0 && (lane >> 2) < G)
      lse[lane >> 2] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
};

// bf16 cache, 16 keys a tile: queries and weights enter as three bf16 terms
// that sum to them exactly, hi and mid in the A operand's two halves, lo in a
// second mma. 64 mma of 2048 products a tile at head_dim 128: a third of the
// tile's share of the memory's time.
template <int DH>
struct Bf16Warp : WarpState<DH> {
  using KT = __nv_bfloat16;
  using WarpState<DH>::o;
  static constexpr int kKeys = 16, kSteps = DH / 16;
  // The queries' terms: in registers, or (kShared, longer heads) for all warps in
  // the swap space, which is free while the tiles go by (16 x 8192 keys of 16/4
  // heads of 256: 110 us, f32 210; split again for each tile 9 and 30 us more).
  static constexpr bool kShared = DH > 128;
  static constexpr int kRoom = kShared ? kSteps * 32 * 24 : 0;
  Split3 q[kShared ? 1 : kSteps][2];
  const uint32_t* room;

  MYOS_DEV void begin(const float* q_row, int G, int d, float* swap) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = (lane & 3) * 2;
    auto load = [&](int at) -> Split3 {
      float2 x = make_float2(0.f, 0.f);
      if (g < G && at < d) x = *reinterpret_cast<const float2*>(q_row + g * d + at);
      return split3(x.x, x.y);
    };
    if constexpr (kShared) {
      uint32_t* to = reinterpret_cast<uint32_t*>(swap);
      room = to;
      __syncthreads();  // the states of the piece before have been read
#pragma unroll
      for (int k = threadIdx.x >> 5; k < kSteps; k += kWarps) {
        const Split3 q0 = load(16 * k + c), q1 = load(16 * k + 8 + c);
        reinterpret_cast<uint4*>(to)[k * 32 + lane] = make_uint4(q0.hi, q0.mid, q1.hi, q1.mid);
        reinterpret_cast<uint2*>(to + kSteps * 128)[k * 32 + lane] = make_uint2(q0.lo, q1.lo);
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u) q[k][u] = load(16 * k + 8 * u + c);
    }
    this->clear();
  }

  // Row r keeps 16-byte chunk i at i ^ (r & 7), so the eight rows that an
  // ldmatrix reads at one chunk lie in different banks.
  static MYOS_DEV uint32_t flip_k(int row) { return row & 7; }
  static MYOS_DEV uint32_t flip_v(int row) { return row & 7; }

  MYOS_DEV void tile(uint32_t ks, uint32_t vs, uint32_t ok, float scale2) {
    const int lane = threadIdx.x & 31, c = (lane & 3) * 2;
    float s[4];
    {
      constexpr int kSums = DH > 128 ? 4 : 2;  // of four steps each
      float a[2][kSums][4], lo[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[n][i] = 0.f;
#pragma unroll
          for (int u = 0; u < kSums; ++u) a[n][u][i] = 0.f;
        }
      const int row = (lane & 7) + ((lane >> 4) << 3);
      const uint32_t base = ks + row * (DH * 2) + ((((lane >> 3) & 1) ^ (row & 7)) << 4);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t b[4];
        ldmatrix4(b, (base ^ ((2 * k & 6) << 4)) + (k >> 2) * 128);
        Split3 q0, q1;
        if constexpr (kShared) {
          const uint4 h = reinterpret_cast<const uint4*>(room)[k * 32 + lane];
          const uint2 l = reinterpret_cast<const uint2*>(room + kSteps * 128)[k * 32 + lane];
          q0 = Split3{h.x, h.y, l.x};
          q1 = Split3{h.z, h.w, l.y};
        } else {
          q0 = q[k][0];
          q1 = q[k][1];
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          mma16816(lo[n], q0.lo, 0u, q1.lo, 0u, b[2 * n], b[2 * n + 1]);
          mma16816(a[n][(k >> 2) & (kSums - 1)], q0.hi, q0.mid, q1.hi, q1.mid, b[2 * n], b[2 * n + 1]);
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (kSums == 4) {
#pragma unroll
            for (int u = i; u < 4; u += 2) {
              a[n][0][u] += a[n][2][u];
              a[n][1][u] += a[n][3][u];
            }
          }
          const float x = (a[n][0][i] + a[n][1][i]) + ((a[n][0][i + 2] + a[n][1][i + 2]) + lo[n][i]);
          s[2 * n + i] = (ok >> (8 * n + c + i)) & 1u ? x * scale2 : -INFINITY;
        }
    }
    const float keep = this->weigh(s);
    const Split3 w0 = split3(s[0], s[1]), w1 = split3(s[2], s[3]);
    const int row = lane & 15;
    const uint32_t base = vs + row * (DH * 2) + (((lane >> 4) ^ (row & 7)) << 4);
#pragma unroll
    for (int j = 0; j < DH / 16; ++j) {
      uint32_t b[4];
      ldmatrix4t(b, (base ^ ((2 * j & 6) << 4)) + (j >> 2) * 128);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float t[4];
        mma16816_zero(t, w0.lo, 0u, w1.lo, 0u, b[2 * n], b[2 * n + 1]);
        mma16816(t, w0.hi, w0.mid, w1.hi, w1.mid, b[2 * n], b[2 * n + 1]);
        float* x = &o[4 * j + 2 * n];
        x[0] = fmaf(x[0], keep, t[0] + t[2]);
        x[1] = fmaf(x[1], keep, t[1] + t[3]);
      }
    }
  }

  static constexpr int kOwn = WarpState<DH>::kOwn;
  MYOS_DEV void write(const float (&own)[kOwn], float* out, int G, int d) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = (lane & 3) * 2;
    if (g >= G) return;
    const float inv = this->inverse();
    const int at = (threadIdx.x >> 5) * kOwn * 4;
#pragma unroll
    for (int j = 0; j < kOwn / 2; ++j)
      if (at + 8 * j < d)
        *reinterpret_cast<float2*>(out + g * d + at + 8 * j + c) =
            make_float2(own[2 * j] * inv, own[2 * j + 1] * inv);
  }
};

// x = hi + lo for a tf32 mma: hi the nearest value of 11 significand bits, lo
// the rest cut to 11 bits, off by at most one step (2^-23) of x.
MYOS_DEV void split2(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
// x without its last bits.
MYOS_DEV float cut(float x, int bits) {
  return __uint_as_float(__float_as_uint(x) & (0xffffffffu << bits));
}

// f32 cache, 8 keys a tile. Keys and queries enter as two tf32 terms, all four
// products (hi and lo of the queries in the A operand's two halves, hi and lo of
// the keys in two mma): a step of a factor can be lost, which is less than the
// scores' own f32 sums round. Values enter exactly, so that a key that takes all
// the weight gives its value: 11 bits in tf32 by both terms of the weights, the
// other 13 as two bf16 terms (8 and 5 bits), side by side along the summed index
// of one mma, by 16 bits of the weights (off by 2^-26 of a product). As two tf32
// terms the values lost their last bit and the kernel took 2 to 6 % less (64
// sequences of 512 to 640 keys of 12/2 heads of 128: 21.3 us, exact 22.2; 16 x
// 8192 of 40/8: 175.5 and 178.8, of 8/8 of 64: 94 and 99, of 16/4 of 256: 210 and
// 217). A third tf32 product takes 5 to 11 % more than two, three bf16 terms of
// keys and values alike 3 to 18.
// On the FMA units a tile cost 1700 instructions, and the 64 sequences took 37 us.
//
// The order in which an mma takes its summed index is free, as long as both
// operands agree: step s of a score sums dims 16 (s / 2) + 4 c + 2 (s % 2) and
// the next (c: lane % 4), so a lane reads its keys 16 bytes at a time; an
// output's step sums key 2 c, which the lane's score is for, and 2 c + 1, and
// column n of tile t is dim 32 (t / 4) + 4 n + t % 4.
template <int DH>
struct F32Warp : WarpState<DH> {
  using KT = float;
  using WarpState<DH>::o;
  static constexpr int kKeys = 8, kChunks = DH / 16;
  static constexpr bool kShared = DH > 128;  // as above
  static constexpr int kRoom = kShared ? kChunks * 32 * 32 : 0;
  uint32_t q[kShared ? 1 : kChunks][8];
  const uint32_t* room;

  static MYOS_DEV void split_q(const float4& x, uint32_t (&y)[8]) {
    split2(x.x, y[0], y[1]);
    split2(x.y, y[2], y[3]);
    split2(x.z, y[4], y[5]);
    split2(x.w, y[6], y[7]);
  }
  MYOS_DEV void begin(const float* q_row, int G, int d, float* swap) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    auto load = [&](int at, uint32_t (&y)[8]) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (g < G && at < d) x = *reinterpret_cast<const float4*>(q_row + g * d + at);
      split_q(x, y);
    };
    if constexpr (kShared) {
      uint4* to = reinterpret_cast<uint4*>(swap);
      room = reinterpret_cast<const uint32_t*>(swap);
      __syncthreads();  // the states of the piece before have been read
#pragma unroll
      for (int k = threadIdx.x >> 5; k < kChunks; k += kWarps) {
        uint32_t y[8];
        load(16 * k + 4 * c, y);
        to[k * 64 + lane] = make_uint4(y[0], y[1], y[2], y[3]);
        to[k * 64 + 32 + lane] = make_uint4(y[4], y[5], y[6], y[7]);
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < kChunks; ++k) load(16 * k + 4 * c, q[k]);
    }
    this->clear();
  }

  // Chunks of a row are exchanged so that the 8 lanes of a 16-byte read phase
  // (two keys x four chunks of K, four even or odd keys x two chunks of V)
  // lie in different banks.
  static MYOS_DEV uint32_t flip_k(int row) { return (row & 1) << 2; }
  static MYOS_DEV uint32_t flip_v(int row) { return (row & 6); }

  MYOS_DEV void tile(uint32_t ks, uint32_t vs, uint32_t ok, float scale2) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    float s[2];
    {
      constexpr int kChains = DH / 32;  // of four steps each
      float a[kChains][4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = 0.f;
#pragma unroll
        for (int n = 0; n < kChains; ++n) a[n][i] = 0.f;
      }
      const uint32_t base = ks + g * (DH * 4) + ((c ^ flip_k(g)) << 4);
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        float4 x;
        lds4(x, (base ^ ((4 * k & 4) << 4)) + (k >> 1) * 128);
        uint32_t y[8], qs[8];
        split_q(x, y);
        if constexpr (kShared) {
          const uint4 l = reinterpret_cast<const uint4*>(room)[k * 64 + lane];
          const uint4 h = reinterpret_cast<const uint4*>(room)[k * 64 + 32 + lane];
          qs[0] = l.x, qs[1] = l.y, qs[2] = l.z, qs[3] = l.w;
          qs[4] = h.x, qs[5] = h.y, qs[6] = h.z, qs[7] = h.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) qs[i] = q[k][i];
        }
        float(&m4)[4] = a[k * kChains / kChunks];
        mma1688(lo, qs[0], qs[1], qs[2], qs[3], y[1], y[3]);
        mma1688(m4, qs[0], qs[1], qs[2], qs[3], y[0], y[2]);
        mma1688(lo, qs[4], qs[5], qs[6], qs[7], y[5], y[7]);
        mma1688(m4, qs[4], qs[5], qs[6], qs[7], y[4], y[6]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (kChains == 8) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            a[n][i] += a[n + 4][i];
            a[n][i + 2] += a[n + 4][i + 2];
          }
        }
        float x = a[0][i], y = a[0][i + 2];
#pragma unroll
        for (int n = 1; n < (kChains < 4 ? kChains : 4); ++n) {
          x += a[n][i];
          y += a[n][i + 2];
        }
        x += y + (lo[i] + lo[i + 2]);
        s[i] = (ok >> (2 * c + i)) & 1u ? x * scale2 : -INFINITY;
      }
    }
    const float keep = this->weigh(s);
    uint32_t w[4];
    split2(s[0], w[0], w[1]);
    split2(s[1], w[2], w[3]);
    const uint32_t w_hi = pack_top(s[0], s[1]);
    const uint32_t w_mid = pack_top(s[0] - top_bits(s[0]), s[1] - top_bits(s[1]));
    // rows 2 c and 2 c + 1 have the same exchange
    const uint32_t base = vs + 2 * c * (DH * 4) + ((g ^ flip_v(2 * c)) << 4);
    // Column tiles whose two mma, one upon the other, go in turn: four (64 x 640
    // above 22.1 us, one by one 23.3), where the registers hold them (128 x 300
    // keys of 32/8 heads of 64: 25.4 us, one by one 24.1).
    constexpr int kTurn = DH > 64 ? 4 : 1;
#pragma unroll
    for (int j = 0; j < DH / 32; ++j) {
      float4 x4, y4;
      lds4(x4, base + j * 128);
      lds4(y4, base + j * 128 + DH * 4);
      const float x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
      for (int e0 = 0; e0 < 4; e0 += kTurn) {
        float t[kTurn][4], x0[kTurn], y0[kTurn];
#pragma unroll
        for (int n = 0; n < kTurn; ++n) {
          const float xe = x[e0 + n], ye = y[e0 + n], x1 = cut(xe, 5), y1 = cut(ye, 5);
          x0[n] = cut(xe, 13);
          y0[n] = cut(ye, 13);
          mma16816_zero(t[n], w_hi, w_mid, w_hi, w_mid, pack_top(x1 - x0[n], y1 - y0[n]),
                        pack_top(xe - x1, ye - y1));
        }
#pragma unroll
        for (int n = 0; n < kTurn; ++n)
          mma1688(t[n], w[0], w[1], w[2], w[3], __float_as_uint(x0[n]), __float_as_uint(y0[n]));
#pragma unroll
        for (int n = 0; n < kTurn; ++n) {
          float* r = &o[8 * j + 2 * (e0 + n)];
          r[0] = fmaf(r[0], keep, t[n][0] + t[n][2]);
          r[1] = fmaf(r[1], keep, t[n][1] + t[n][3]);
        }
      }
    }
  }

  static constexpr int kOwn = WarpState<DH>::kOwn;
  MYOS_DEV void write(const float (&own)[kOwn], float* out, int G, int d) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (g >= G) return;
    const float inv = this->inverse();
#pragma unroll
    for (int j = 0; j < kOwn / 8; ++j) {
      const float* r = &own[8 * j];
      const int at = (threadIdx.x >> 5) * kOwn * 4 + 32 * j + 8 * c;
      if (at >= d) continue;
      float* to = out + g * d + at;
      *reinterpret_cast<float4*>(to) = make_float4(r[0] * inv, r[2] * inv, r[4] * inv, r[6] * inv);
      *reinterpret_cast<float4*>(to + 4) =
          make_float4(r[1] * inv, r[3] * inv, r[5] * inv, r[7] * inv);
    }
  }
};

// n shares of a row of `total` tiles, the first `more` of them one tile longer
// than `each`.
struct Shares {
  uint32_t each, more;
  MYOS_DEV void cut(uint32_t total, uint32_t n) {
    each = total / n;
    more = total - each * n;
  }
  MYOS_DEV uint32_t begin(uint32_t i) const { return i * each + min(i, more); }
  MYOS_DEV uint32_t of(uint32_t tile) const {
    const uint32_t longer = more * (each + 1);
    const bool in = tile < longer;
    const uint32_t at = (in ? tile : tile - longer) / (in ? each + 1 : each);
    return in ? at : at + more;
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
#pragma unroll 1
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

// The meeting of several blocks costs about as much as kJoinTiles tiles (2 us),
// and each of its parts (0.06 us) about a sixth of one: an item of L tiles is
// soonest done in sqrt(kPartsPerTile * L) shares. A second piece in a share
// costs kPieceTiles.
constexpr int kJoinTiles = 5, kPartsPerTile = 6, kPieceTiles = 4;

// The parts of one split item: shares first .. last. All but the first share
// begin inside the item, so their part is their first piece (slot 0); the
// first share's is its last piece (slot 1).
struct Split {
  int first, last;
  int b, h;
  bool second;  // whether the first share's part is in slot 1
};

template <int DH, class P>
MYOS_DEV P* part_of(P* parts, const Split& ps, int share) {
  const int slot = share == ps.first && ps.second ? 1 : 0;
  return parts + (size_t)(share * 2 + slot) * (kMaxGroup * DH + 16);
}

// By the last block of a split item: its parts through the stages, as many at
// a time as fit (their copies all in flight at once), then warp u adds up
// values [u kOwn, (u + 1) kOwn) of them in the order of their shares. Out of
// line: its registers are not the main loop's.
template <class W, int DH>
__device__ __noinline__ void join_parts(const float* parts, const Split ps, float* room,
                                        float* out, float* lse, int G, int d) {
  constexpr int kOwn = W::kOwn, kPart = kMaxGroup * DH + 16, kChunks = kPart / 4;
  constexpr int kFit = kStages * kWarps * 2 * W::kKeys * DH * (int)sizeof(typename W::KT) / (kPart * 4);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
  const int count = ps.last - ps.first + 1;
  W w;
  w.m = -INFINITY;
  w.l = 0.f;
  float own[kOwn];
#pragma unroll
  for (int r = 0; r < kOwn; ++r) own[r] = 0.f;
#pragma unroll 1
  for (int p0 = 0; p0 < count; p0 += kFit) {
    const int now = min(kFit, count - p0);
    __syncthreads();  // the stages are free
#pragma unroll 4
    for (int i = threadIdx.x; i < now * kChunks; i += kWarps * 32) {
      const int p = i / kChunks;
      cp_async16(smem_u32(room) + i * 16,
                 part_of<DH>(parts, ps, ps.first + p0 + p) + (i - p * kChunks) * 4, true);
    }
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    if (warp >= W::kOwners) continue;
    float top = w.m;
#pragma unroll 4
    for (int p = 0; p < now; ++p) top = fmaxf(top, room[p * kPart + g]);
    const float keep = weight_of(w.m, top);
    w.m = top;
    w.l *= keep;
#pragma unroll
    for (int r = 0; r < kOwn; ++r) own[r] *= keep;
#pragma unroll 2
    for (int p = 0; p < now; ++p) {
      const float* part = room + p * kPart;
      const float f = weight_of(part[g], top);
      w.l = fmaf(part[kMaxGroup + g], f, w.l);
      part += 16 + warp * kOwn * 32 + lane * 4;
#pragma unroll
      for (int r = 0; r < kOwn; r += 4) {
        const float4 x = *reinterpret_cast<const float4*>(part + r * 32);
        own[r] = fmaf(x.x, f, own[r]);
        own[r + 1] = fmaf(x.y, f, own[r + 1]);
        own[r + 2] = fmaf(x.z, f, own[r + 2]);
        own[r + 3] = fmaf(x.w, f, own[r + 3]);
      }
    }
  }
  if (warp < W::kOwners) w.write(own, out, G, d);
  if (warp == 0) w.put_lse(lse, G);
}

template <class W, int DH>
constexpr size_t attn_smem() {
  static_assert(W::kRoom <= (kWarps - 1) * W::kRegs * 32 * 4);  // in the swap space
  return (size_t)kStages * kWarps * 2 * W::kKeys * DH * sizeof(typename W::KT) +
         (kWarps - 1) * W::kRegs * 32 * 4;
}

// Blocks resident on a multiprocessor, by shared memory (55, 108 or 216 KB each),
// and blocks of a cluster, in launches of at least so many for each item: two
// shares of one meet through the pair's shared memory, not the work buffer. That
// gains where many items are split (64 x 640 of 12/2 heads of 128, 22.2 us instead
// of 23.7 in f32 and 14.1 instead of 15.3 in bf16; 1 x 32768 of 40/8 31.4 instead
// of 33.2; 16 x 8192 f32 of 16/4 of 256 216 instead of 223) and loses up to 9 % of
// a few short ones, whose launch by cluster takes longer (1 x 128 5.7 instead of
// 5.6, 8 x 1024 10.9 instead of 10.0, 1 x 4097 11.3 instead of 10.7, 2 x 500 f32 of
// 40/8 10.5 instead of 9.7): the lengths that tell them apart are the device's.
// Clusters of 4 are not all placed at once: 32 ragged sequences took 380 us
// instead of 281.
template <int DH>
constexpr int kResident = DH == 64 ? 4 : DH == 128 ? 2 : 1;
constexpr int kCluster = 2;

// kFull: head_dim is DH itself (else the chunks behind it are zero-filled).
template <class W, int DH, bool kFull>
__global__ void __launch_bounds__(kWarps * 32, kResident<DH>)
    k_paged_attn(const PagedAttnArgs a, const PagedKv<typename W::KT> kv) {
  using KT = typename W::KT;
  constexpr int T = W::kKeys * kWarps, kThreads = kWarps * 32;
  constexpr int kRowBytes = DH * (int)sizeof(KT), kHalf = W::kKeys * kRowBytes;
  constexpr int kStageBytes = kWarps * 2 * kHalf;
  constexpr int kRowsEach = W::kKeys / 8, kSegs = kRowBytes / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float ms[kWarps][kMaxGroup], ls[kWarps][kMaxGroup];
  __shared__ uint32_t sums[kWarps];
  __shared__ int longs[kWarps];
  __shared__ Cursor first_s;
  __shared__ Split splits[2];  // split items that this block was the last to arrive at
  __shared__ int ready[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = (int)kv.heads, G = a.group, d = kFull ? DH : (int)kv.d;
  const uint32_t me = blockIdx.x;
  float* swap = reinterpret_cast<float*>(smem + kStages * kStageBytes);
  if (threadIdx.x < 2) ready[threadIdx.x] = 0;
  pdl_launch();
  pdl_wait();

  // this block's share [lo, hi) of the tiles (fewer than 2^31 in all), and
  // where it begins
  const int per = (a.nseq + kThreads - 1) / kThreads;
  const int b0 = min(a.nseq, (int)threadIdx.x * per), b1 = min(a.nseq, b0 + per);
  uint32_t mine = 0;
  int longest = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    Cursor c;
    span_of<T>(a, b, &c);
    mine += c.t1 - c.t0;
    longest = max(longest, c.t1 - c.t0);
  }
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) {
    sums[warp] = upto;
    longs[warp] = longest;
  }
  // sequences without a key have no tile: their outputs are spread over the blocks
#pragma unroll 1
  for (int b = (int)me; b < a.nseq; b += (int)gridDim.x) {
    Cursor c;
    span_of<T>(a, b, &c);
    if (c.t0 < c.t1) continue;
#pragma unroll 1
    for (int i = threadIdx.x; i < a.hq * d; i += kThreads) {
      a.out[b * a.out_stride + i] = 0.f;
      if (a.lse && i < a.hq) a.lse[(int64_t)b * a.hq + i] = -INFINITY;
    }
  }
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += sums[w];
    total += sums[w];
    longest = max(longest, longs[w]);
  }
  total *= heads;
  // n equal shares, none of them empty; or each item in k of its own, where its
  // longest is not much longer than an equal share
  const uint32_t items = (uint32_t)a.nseq * heads;
  const uint32_t best = items * sqrtf(kPartsPerTile * ((float)total / items));
  const uint32_t n = max(1u, min(min(gridDim.x, total), best));
  Shares shares;
  shares.cut(total, n);
  const bool alone = (uint32_t)longest <= shares.each + kJoinTiles;
  uint32_t k = alone ? 1u : max(1u, n / items);
  if (k > 1) k -= k % kCluster;  // n / items > 1 only in launches by cluster
  const bool by_item = items <= gridDim.x &&
                       (alone || ((uint32_t)longest + k - 1) / k <= shares.each + kPieceTiles);
  // By item, `group` neighbouring shares of one lie in a cluster and meet there;
  // the first of them goes on with the group's part, if the item has more than one.
  const uint32_t group = by_item && k > 1 ? kCluster : 1u;
  uint32_t lo = 0, hi = 0, member = 0, members = 1, first = 0, last = 0;
  Cursor ahead;
  if (by_item) {
    const uint32_t item = me / k, at = me - item * k;
    if (item < items) {
      ahead.b = item / heads;
      ahead.h = item - ahead.b * heads;
      span_of<T>(a, ahead.b, &ahead);
      const uint32_t tiles = ahead.t1 - ahead.t0, cuts = min(k, tiles);
      if (at < cuts) {
        Shares own;  // at * tiles may pass 32 bits
        own.cut(tiles, cuts);
        lo = own.begin(at);
        hi = own.begin(at + 1);
        ahead.t = ahead.t0 + lo;
        member = at % group;
        members = min(group, cuts - (at - member));
        first = item * k / group;
        last = first + (cuts - 1) / group;
      }
    }
  } else {
    if (me < n) {
      lo = shares.begin(me);
      hi = shares.begin(me + 1);
    }
    if (lo < hi && (upto - mine) * heads <= lo && lo < upto * heads) {
      uint32_t at = lo - (upto - mine) * heads;  // tiles between b0's first and the share
      Cursor c;
      int b = b0;
#pragma unroll 1
      for (;; ++b) {
        span_of<T>(a, b, &c);
        const uint32_t all = (uint32_t)(c.t1 - c.t0) * heads;
        if (at < all) break;
        at -= all;
      }
      c.b = b;
      c.h = at / (uint32_t)(c.t1 - c.t0);
      c.t = c.t0 + at - c.h * (c.t1 - c.t0);
      first_s = c;
    }
    __syncthreads();
    ahead = first_s;
  }
  if (lo >= hi) {
    if (group > 1) {  // the cluster's barriers are for all its blocks
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  Cursor c = ahead;
  const uint32_t stages = smem_u32(smem) + warp * 2 * kHalf;
  // this lane's copies: rows lane / 4 (+ 8), 16-byte chunks 4 j + lane % 4
  const int row = lane >> 2, seg = lane & 3;
  uint32_t to_k[2], to_v[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    to_k[u] = row * kRowBytes + (((4 * u + seg) ^ W::flip_k(row)) << 4);
    to_v[u] = kHalf + row * kRowBytes + (((4 * u + seg) ^ W::flip_v(row)) << 4);
  }
  // where this lane's rows of a tile lie, up to the page, which is on its way
  struct Rows {
    int page[kRowsEach];
    int64_t in[kRowsEach];
  };
  int left = (int)(hi - lo);  // tiles not looked up yet
  auto look = [&](Rows& x) {
#pragma unroll
    for (int r = 0; r < kRowsEach; ++r) {
      const int key = ahead.t * T + warp * W::kKeys + row + 8 * r;
      const int pg = (int)((uint64_t)(uint32_t)key * a.page_mul >> a.page_shift);
      x.in[r] = ahead.h * kv.head_stride + (key - pg * (int)kv.page_size) * kv.slot_stride +
                seg * (16 / (int)sizeof(KT));
      x.page[r] = left > 0 && key >= ahead.start && key < ahead.len
                      ? a.table[ahead.b * a.table_stride + pg]
                      : -1;
    }
    if (left > 1) advance<T>(a, heads, &ahead);
    if (left > 0) --left;
  };
  Rows soon, later;
#pragma unroll
  for (int r = 0; r < kRowsEach; ++r) soon.page[r] = later.page[r] = -1;
  int put_at = 1;     // the stage of the tile that is copied next: 0 for the first
  uint64_t okay = 0;  // 16 bits of keys for each tile in flight, the newest on top
  static_assert(kStages == 3, "key bits of three tiles in one word");
  // copies the tile that was looked up two calls before, looks the next one up
  auto pump = [&]() {
    uint32_t ok = 0;
    const uint32_t dst = stages + put_at * kStageBytes;
    const KT *src_k[kRowsEach], *src_v[kRowsEach];
    bool on[kRowsEach];
#pragma unroll
    for (int r = 0; r < kRowsEach; ++r) {
      on[r] = (uint32_t)soon.page[r] < kv.num_pages;
      const int64_t at = on[r] ? soon.page[r] * kv.page_stride + soon.in[r] : 0;
      src_k[r] = kv.k + at;
      src_v[r] = kv.v + at;
      ok |= gather_rows(__ballot_sync(0xffffffffu, on[r])) << (8 * r);  // bit 4 i: row i
    }
    if (ok) {
#pragma unroll
      for (int r = 0; r < kRowsEach; ++r)
#pragma unroll
        for (int j = 0; j < kSegs; ++j) {
          const bool load = on[r] && (kFull || (4 * j + seg) * (16 / (int)sizeof(KT)) < d);
          const uint32_t off = dst + r * 8 * kRowBytes + (j >> 1) * 128;
          const int from = j * (64 / (int)sizeof(KT));
          cp_async16(off + to_k[j & 1], kFull || load ? src_k[r] + from : kv.k, load);
          cp_async16(off + to_v[j & 1], kFull || load ? src_v[r] + from : kv.v, load);
        }
    }
    cp_commit();
    put_at = put_at == kStages - 1 ? 0 : put_at + 1;
    okay = okay >> 16 | (uint64_t)ok << 32;
    soon = later;
    look(later);
  };
#pragma unroll 1
  for (int s = 0; s < 4; ++s) pump();  // two calls copy nothing yet

  int take_at = 0;
#pragma unroll 1
  for (uint32_t i = lo; i < hi;) {
    // one piece: the tiles of item (c.b, c.h) from c.t on in this share
    const uint32_t i0 = i - (c.t - c.t0), i1 = i0 + (c.t1 - c.t0);
    W w;
    w.begin(a.q + c.b * a.q_stride + (int64_t)c.h * G * d, G, d, swap);
#pragma unroll 1
    for (const uint32_t end = min(hi, i1); i < end; ++i) {
      cp_wait<kStages - 2>();
      __syncwarp();
      pump();
      const uint32_t base = stages + take_at * kStageBytes, ok = (uint32_t)okay & 0xffffu;
      take_at = take_at == kStages - 1 ? 0 : take_at + 1;
      if (ok) w.tile(base, base + kHalf, ok, a.scale2);
      __syncwarp();
    }
    w.finish();
    __syncthreads();  // the swap space is free
    w.leave(&ms[0][0], &ls[0][0], swap);
    __syncthreads();
    const bool whole = by_item ? first == last : i0 >= lo && i1 <= hi;
    float own[W::kOwn];
    if (warp < W::kOwners) w.meet(&ms[0][0], &ls[0][0], swap, own);
    if (group > 1) {
      // the other members' states, left in their stages, into the first's
      float* give = reinterpret_cast<float*>(smem) + 16;
      cp_wait<0>();
      if (member > 0 && warp < W::kOwners) {
        if (warp == 0) w.put_ml(give - 16, give - 8);
#pragma unroll
        for (int r = 0; r < W::kOwn; r += 4)
          *reinterpret_cast<float4*>(give + (warp * W::kOwn + r) * 32 + lane * 4) =
              make_float4(own[r], own[r + 1], own[r + 2], own[r + 3]);
      }
      cluster_sync();
      if (member == 0 && warp < W::kOwners) {
        const int g = lane >> 2;
#pragma unroll 1
        for (uint32_t u = 1; u < members; ++u) {
          const uint32_t from = in_block(smem_u32(give), me % kCluster + u);
          const float pm = ldc(from - 64 + g * 4), pl = ldc(from - 32 + g * 4);
          const float top = fmaxf(w.m, pm);
          const float fa = weight_of(w.m, top), fb = weight_of(pm, top);
          w.m = top;
          w.l = w.l * fa + pl * fb;
#pragma unroll
          for (int r = 0; r < W::kOwn; r += 4) {
            const float4 x = ldc4(from + ((warp * W::kOwn + r) * 32 + lane * 4) * 4);
            own[r] = own[r] * fa + x.x * fb;
            own[r + 1] = own[r + 1] * fa + x.y * fb;
            own[r + 2] = own[r + 2] * fa + x.z * fb;
            own[r + 3] = own[r + 3] * fa + x.w * fb;
          }
        }
      }
      cluster_sync();  // the members' memory has been read
      if (member > 0) return;
    }
    if (warp < W::kOwners) {
      const int64_t head = (int64_t)c.h * G;
      if (whole) {
        w.write(own, a.out + c.b * a.out_stride + head * d, G, d);
        if (warp == 0) w.put_lse(a.lse ? a.lse + (int64_t)c.b * a.hq + head : nullptr, G);
      } else {
        Split sp;
        sp.first = (int)(by_item ? first : shares.of(i0));
        sp.last = (int)(by_item ? last : shares.of(i1 - 1));
        sp.second = !by_item && i0 >= shares.begin(sp.first);
        sp.b = c.b;
        sp.h = c.h;
        float* part = part_of<DH>(a.parts, sp, (int)(by_item ? me / group : me));
        if (warp == 0) w.put_ml(part, part + kMaxGroup);
        part += 16 + warp * W::kOwn * 32 + lane * 4;
#pragma unroll
        for (int r = 0; r < W::kOwn; r += 4)
          *reinterpret_cast<float4*>(part + r * 32) =
              make_float4(own[r], own[r + 1], own[r + 2], own[r + 3]);
        __syncwarp();
        if (lane == 0) {
          // the warp's stores before its arrival, the others' parts after it
          const unsigned all = (unsigned)(sp.last - sp.first + 1) * W::kOwners;
          if (arrive(&a.arrived[sp.first]) == all - 1) {
            a.arrived[sp.first] = 0;
            splits[i0 < lo ? 0 : 1] = sp;
            ready[i0 < lo ? 0 : 1] = 1;
          }
        }
      }
    }
    c.t = c.t1 - 1;
    advance<T>(a, heads, &c);
  }
  // the joins that fell to this block, once its own tiles are done
  cp_wait<0>();
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    if (!ready[k]) continue;
    const Split sp = splits[k];
    const int64_t head = (int64_t)sp.h * G;
    join_parts<W, DH>(a.parts, sp, reinterpret_cast<float*>(smem), a.out + sp.b * a.out_stride + head * d,
                      a.lse ? a.lse + (int64_t)sp.b * a.hq + head : nullptr, G, d);
  }
}

template <class W, int DH, bool kFull>
cudaError_t launch(PagedAttnArgs a, const myos_paged_kv* kv, void* work, cudaStream_t st) {
  constexpr size_t smem = attn_smem<W, DH>(), kCounters = 16 * 1024;
  constexpr int T = W::kKeys * kWarps;
  static_assert(kCounters + (size_t)kMaxShares * 2 * (kMaxGroup * DH + 16) * 4 <=
                MYOS_PAGED_WORK_BYTES);
  static std::atomic<uint64_t> raised{0};
  const cudaError_t e = raise_smem_limit((const void*)k_paged_attn<W, DH, kFull>, smem, &raised);
  if (e != cudaSuccess) return e;
  a.arrived = static_cast<unsigned*>(work);
  a.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + kCounters);
  // a share per resident block, and never more than there can be tiles
  int64_t keys = a.max_keys;
  if (a.window > 0 && (int64_t)a.window + T < keys) keys = (int64_t)a.window + T;
  const int64_t most = (int64_t)a.nseq * kv->num_kv_heads * ((keys + T - 1) / T);
  static_assert((smem + 1536) * kResident<DH> <= 228 * 1024);
  int64_t grid = (int64_t)sm_count() * kResident<DH>;
  if (grid > kMaxShares) grid = kMaxShares;
  if (grid > most) grid = most;
  const int64_t items = (int64_t)a.nseq * kv->num_kv_heads;
  const int cluster = items * kCluster <= grid ? kCluster : 1;
  grid = (grid + cluster - 1) / cluster * cluster;
  return counted(launch_pdl(k_paged_attn<W, DH, kFull>, dim3((unsigned)grid), kWarps * 32, smem, st,
                            cluster, a, paged_view<typename W::KT>(kv)));
}

template <int DH>
cudaError_t launch_d(const PagedAttnArgs& a, const myos_paged_kv* kv, void* work,
                     cudaStream_t st) {
  if (kv->kv_dtype == MYOS_KV_BF16)
    return kv->head_dim == DH ? launch<Bf16Warp<DH>, DH, true>(a, kv, work, st)
                              : launch<Bf16Warp<DH>, DH, false>(a, kv, work, st);
  return kv->head_dim == DH ? launch<F32Warp<DH>, DH, true>(a, kv, work, st)
                            : launch<F32Warp<DH>, DH, false>(a, kv, work, st);
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
      max_blocks * kv->page_size > 0x7fffff00 ||
      (max_blocks * kv->page_size / 32 + 1) * nseq * kv->num_kv_heads > 0x7fffffff || q_stride < num_q_heads * d ||
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
  // ceil(2^s / P) with s = 31 + ceil(log2 P): its error times any key is below 2^s
  int log2 = 0;
  while ((1u << log2) < kv->page_size) ++log2;
  a.page_shift = 31 + log2;
  a.page_mul =
      (uint32_t)((((uint64_t)1 << a.page_shift) + kv->page_size - 1) / kv->page_size);
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = d <= 64    ? launch_d<64>(a, kv, d_work, st)
                        : d <= 128 ? launch_d<128>(a, kv, d_work, st)
                                   : launch_d<256>(a, kv, d_work, st);
  return e == cudaSuccess ? MYOS_OK : MYOS_ERR_CUDA;
}
