// How a product of 8-bit rows and channels is cut (host arithmetic only).
//
// Times below are of a B200, in microseconds a call.
#pragma once
#include <stdint.h>

namespace myos {

constexpr int kI8Channels = 128;        // channels of a block's tile: the tensor core's M
constexpr int kI8Step = 128;            // bytes of k of a stage: one swizzled row
constexpr int kI8MaxRows = 256;         // rows of a tile at most: its N
constexpr int kI8MaxStages = 12;
constexpr int kI8Smem = 200 * 1024;     // a block's stages,
constexpr int kI8SmemTwo = 109 * 1024;  // where two blocks share a multiprocessor
constexpr int kI8MaxSplit = 8;          // blocks that share a tile's k: a portable cluster
constexpr int kI8FewRows = 16;

inline int64_t i8_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Channels that each of `split` blocks adds up: whole groups of 4.
constexpr int i8_wide(int split) { return (kI8Channels / 4 + split - 1) / split * 4; }

// ---- up to 16 rows: how many 8-channel groups a block of how many warps takes
struct I8Few {
  int use, groups, warps;
};

// 9 to 16 rows read as many bytes of rows as of weights, so they take wide blocks,
// and tiles from 64 MB of weights on (16 x 1536 x 151936: 48.7 here, 41.5 in tiles;
// 16 x 5120 x 7168: 10.4, 11.3). Up to 8 rows the blocks are as small as still gives
// each warp a few pieces of k, with some 1700 warps at least where the channels allow
// it: 1 x 1536 x 17920 with 2, 4, 8 warps of 16 channels 6.4, 7.8, 10.3; 1 x 13824 x
// 5120 with 4 warps of 8, 16, 32 channels 14.0, 18.1, 22.9; 1 x 8960 x 1536 with 4, 8
// warps of 8 channels 7.9, 5.7; 1 x 5120 x 27648 with 2, 4 warps of 16 channels 27.1,
// 24.3.
inline I8Few i8_few(int64_t rows, int64_t k, int64_t channels) {
  I8Few f = {rows <= 8 || (rows <= kI8FewRows && k * channels < ((int64_t)64 << 20)), 2, 2};
  const int64_t pieces = i8_ceil(k, 64);
  if (rows > 8) {
    f.groups = 4;
    while (f.warps < 8 && i8_ceil(channels, 32) * f.warps < 1100) f.warps *= 2;
    if (i8_ceil(channels, 32) * f.warps < 1100) f.groups = 2;
  } else {
    f.warps = pieces > 40 ? 4 : 2;
    if (i8_ceil(channels, 16) * 4 < 1700) {
      f.groups = 1;
      f.warps = i8_ceil(channels, 8) * 4 < 1200 && pieces > 48 ? 8 : 4;
    }
  }
  return f;
}

// ---- tiles on tcgen05
struct I8Plan {
  int pair;     // a tile is two blocks', on neighbouring multiprocessors
  int tc;       // channels of a tile: 128, of a pair 256
  int tn;       // rows of a tile, a multiple of 16 (of a pair: of 32)
  int split;    // blocks (a cluster) that share a tile's k
  int two;      // two blocks a multiprocessor
  int apart;    // the cluster's sums have their own place behind the stages
  int stages;
  int group;    // row tiles that follow one another under one channel tile
  int vec;      // four results are stored at once (the caller's to say)
  int columns;  // of tensor memory: two accumulators, a power of two
  int tiles_c, tiles_r;
};

// What a device holds at once: multiprocessors, and blocks in clusters of s with one
// or two blocks a multiprocessor.
struct I8Device {
  int sms;
  int one[kI8MaxSplit + 1], two[kI8MaxSplit + 1];
};

inline I8Plan i8_plan(int64_t rows, int64_t k, int64_t channels, const I8Device& d) {
  I8Plan p = {};
  const int64_t steps = i8_ceil(k, kI8Step);
  // Pairs read a third less from L2 for the same products. They pay where they fill
  // the device (4096 x 5120 x 27648: 490 -> 452; 512 x 5120 x 7168, 56 of 74 pairs:
  // 22.8, 22.4; 1024 x 8960 x 1536, 24 pairs: 30.7, and 21.9 in split tiles).
  const int64_t least_r = i8_ceil(rows, kI8MaxRows), pairs_c = i8_ceil(channels, 2 * kI8Channels);
  p.pair = rows > kI8MaxRows && least_r * pairs_c >= d.sms / 2;
  p.tc = p.pair ? 2 * kI8Channels : kI8Channels;
  p.tiles_c = (int)i8_ceil(channels, p.tc);
  const int unit = p.pair ? 32 : 16;
  // Rows of a tile: the fewest tiles, or a few more that fill the last round better. A
  // step costs its products (2 cycles a row) or its copies (59 bytes a cycle).
  const int64_t places = p.pair ? d.sms / 2 : d.sms;
  int64_t best = 0;
  for (int64_t r = least_r; r < least_r + 4 && (r == least_r || p.pair); ++r) {
    const int64_t tn = i8_ceil(i8_ceil(rows, r), unit) * unit, n = i8_ceil(rows, tn);
    const int64_t copies = (kI8Channels + tn / (p.pair ? 2 : 1)) * kI8Step / 59;
    const int64_t cost = i8_ceil(n * p.tiles_c, places) * (copies > 2 * tn ? copies : 2 * tn);
    if (best == 0 || cost < best) {
      best = cost;
      p.tn = (int)tn;
      p.tiles_r = (int)n;
    }
  }
  const int64_t tiles = (int64_t)p.tiles_c * p.tiles_r;
  p.two = !p.pair && p.tn <= 64;
  // A multiprocessor takes weights from memory at some 49 GB/s, however many of its
  // copies are on their way, so few tiles are split until every one has a part, if the
  // shorter way (0.34 a step) saves what a cluster costs (0.5, and 0.012 a row).
  // 64 x 13824 x 5120 in 1, 2, 4, 6 parts: 39.8, 26.9, 18.8, 18.4; 128 x 13824 x 5120 in
  // 1, 2, 3: 40.8, 25.7, 21.0; 64 x 5120 x 27648 in 1, 2: 27.7, 34.3; 64 x 1536 x 2048
  // in 1, 4, 8: 7.3, 5.0, 6.0.
  p.split = 1;
  const int parts[] = {2, 3, 4, 6, 8};
  int64_t least = steps * 340;
  for (int s : parts) {
    const int64_t most = p.two ? (d.two[s] < 5 * d.sms / 3 ? d.two[s] : 5 * d.sms / 3) : d.one[s];
    const int64_t time = i8_ceil(steps, s) * 340 + 500 + 12 * p.tn;
    if (p.pair || tiles * s > most || steps < 3 * s || time >= least) continue;
    least = time;
    p.split = s;
  }
  const int stage = (kI8Channels + p.tn / (p.pair ? 2 : 1)) * kI8Step;
  const int sums = p.split * p.tn * i8_wide(p.split) * 4;
  p.apart = p.split > 1 && p.tn <= 64;
  p.stages = ((p.two ? kI8SmemTwo : kI8Smem) - (p.apart ? sums : 0)) / stage;
  if (p.stages > kI8MaxStages) p.stages = kI8MaxStages;
  p.columns = 32;
  while (p.columns < 2 * p.tn) p.columns *= 2;
  // Rows that stay in L2 (32 MB of them) while the weights pass once, in equal groups.
  int64_t group = ((int64_t)32 << 20) / (p.tn * k);
  if (group < 1) group = 1;
  if (group > p.tiles_r) group = p.tiles_r;
  p.group = (int)i8_ceil(p.tiles_r, i8_ceil(p.tiles_r, group));
  return p;
}

}  // namespace myos
