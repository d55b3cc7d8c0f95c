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
constexpr int kI8Parts[] = {1, 2, 3, 4, 6, 8};
constexpr int kI8FewRows = 16;

inline int64_t i8_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Channels that each of `split` blocks adds up: whole groups of 4.
constexpr int i8_wide(int split) { return (kI8Channels / 4 + split - 1) / split * 4; }

// ---- up to 16 rows: how many 8-channel groups a block of how many warps takes
struct I8Few {
  int use, groups, warps;
};

// 9 to 16 rows read as many bytes of rows as of weights, so they take wide blocks,
// and tiles from 64 MB of weights on (16 x 1536 x 151936: 47.7 here, 39.5 in tiles;
// 16 x 5120 x 7168: 10.3, 10.2). Up to 8 rows the blocks are as small as still gives
// each warp a few pieces of k, with some 1700 warps at least where the channels allow
// it: 1 x 1536 x 17920 with 2, 4, 8 warps of 16 channels 6.5, 8.0, 9.8; 1 x 13824 x
// 5120 with 4 warps of 8, 16, 32 channels 14.0, 17.5, 21.6; 1 x 8960 x 1536 with 4, 8
// warps of 8 channels 7.5, 5.3; 1 x 5120 x 27648 with 2, 4 warps of 16 channels 28.9,
// 25.3.
inline I8Few i8_few(int64_t rows, int64_t k, int64_t channels) {
  I8Few f = {rows <= 8 || (rows <= kI8FewRows && k * channels < ((int64_t)64 << 20)), 2, 2};
  const int64_t pieces = i8_ceil(k, 64);
  if (rows > 8) {
    f.groups = 4;
    while (f.warps < 8 && i8_ceil(channels, 32) * f.warps < 1100) f.warps *= 2;
    if (i8_ceil(channels, 32) * f.warps < 1100) f.groups = 2;
  } else {
    f.warps = pieces > 40 ? 4 : 2;
    // short rows: fewer blocks, which take 3 ns each (2 x 128 x 73276: 7.7, 5.9)
    if (pieces <= 16 && channels >= 27200) f.groups = 4;
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

// Fills in what the device holds in clusters. known: a word for each size (std::atomic, 0
// at first). ask(s, two, &blocks): whether it could be asked; an answer that could not be
// had counts as no room in this call, and is asked for again in the next.
template <class Word, class Ask>
inline void i8_room(I8Device& d, Word* known, const Ask& ask) {
  for (int s : kI8Parts) {
    if (s == 1) continue;
    uint64_t v = known[s].load();
    if (v == 0) {
      int one = 0, two = 0;
      const bool first = ask(s, false, &one), second = ask(s, true, &two);
      v = (uint64_t)1 << 63 | (uint64_t)(first ? one : 0) << 31 | (uint64_t)(second ? two : 0);
      if (first && second) known[s].store(v);
    }
    d.one[s] = (int)(v >> 31 & 0x7fffffff);
    d.two[s] = (int)(v & 0x7fffffff);
  }
}

// A step's time in a block that waits for its copies alone, in ns, and where pairs fill
// the device and its power (8192 x 8192 x 8192).
inline int64_t i8_step(bool pair, int64_t tn, bool filled) {
  const int64_t copies = pair ? 175 + tn * 9 / 100 : 200 + tn * 3 / 4, products = 20 + tn * 8 / 5;
  return filled && products > copies ? products : copies;
}

// Tiles of `unit` rows and their multiples: the fewest, or a few more that fill the last
// round better (17 row tiles of 256 for 4097 rows, or 19 of 224).
inline int64_t i8_rows(I8Plan& p, int64_t rows, int64_t places, int unit) {
  const int64_t least_r = i8_ceil(rows, kI8MaxRows);
  int64_t best = 0;
  for (int64_t r = least_r; r < least_r + 4; ++r) {
    const int64_t tn = i8_ceil(i8_ceil(rows, r), unit) * unit, n = i8_ceil(rows, tn);
    const int64_t rounds = i8_ceil(n * p.tiles_c, places);
    const int64_t cost = rounds * i8_step(p.pair, tn, n * p.tiles_c >= places);
    if (best != 0 && cost >= best) continue;
    best = cost;
    p.tn = (int)tn;
    p.tiles_r = (int)n;
  }
  return best;
}

inline I8Plan i8_plan(int64_t rows, int64_t k, int64_t channels, const I8Device& d) {
  I8Plan p = {}, q = {};
  const int64_t steps = i8_ceil(k, kI8Step);
  // Pairs copy less for the same products: each block half of the rows. From 65 rows on
  // they are the rule (256 x 5120 x 7168: 13.8 for 18.4; 128 x 1536 x 2048: 5.1 for 6.5).
  q.pair = 1;
  q.tc = 2 * kI8Channels;
  q.tiles_c = (int)i8_ceil(channels, q.tc);
  const int64_t pairs = d.one[2] / 2, paired = pairs ? steps * i8_rows(q, rows, pairs, 32) : 0;
  // Where tiles are few they are split along k, if the shorter way saves what a cluster
  // costs (1.2 us, and 14 ns a row): 64 x 13824 x 5120 in 1, 2, 3 parts 33.1, 18.4, 17.4;
  // 64 x 5120 x 27648 in 1, 2: 27.0, 32.9; 64 x 1536 x 2048 in 1, 4, 8: 5.7, 4.8, 5.5; 128
  // x 13824 x 5120 in 1, 2, 3 and in pairs: 30.7, 21.5, 19.5, 23.3. Two blocks a
  // multiprocessor only where there are more than multiprocessors: they have half the
  // stages (64 x 5120 x 7168 in 2 parts: 13.0 for 11.3). Many rows of few channels are cut
  // into smaller tiles as well (4041 x 2775 x 83: 15.4 in pairs of 256 rows, 9.0).
  p.tc = kI8Channels;
  p.tiles_c = (int)i8_ceil(channels, p.tc);
  int64_t least = 0;
  for (int64_t r = i8_ceil(rows, kI8MaxRows); r == i8_ceil(rows, kI8MaxRows) || rows > 64; ++r) {
    const int64_t tn = i8_ceil(i8_ceil(rows, r), 16) * 16, n_r = i8_ceil(rows, tn);
    if (n_r < r && r > i8_ceil(rows, kI8MaxRows)) continue;  // the tiles of a smaller r
    if ((tn < 64 || r > 2 * d.sms) && least != 0) break;
    const int64_t tiles = p.tiles_c * n_r, step = i8_step(false, tn, false);
    for (int s : kI8Parts) {
      const int64_t n = tiles * s;
      const bool two = s == 1 ? tn <= 64 && n > d.sms : n > d.one[s];
      if (s > 1 && (steps < 3 * s || (two && (tn > 64 || n > d.two[s] || n > 5 * d.sms / 3)))) continue;
      // of one part the tiles follow one another on a multiprocessor, of more they are all
      // there at once; and all that is copied comes through L2, 12000 bytes a ns
      int64_t time = i8_ceil(steps, s) * step * (s == 1 ? i8_ceil(n, d.sms) : two ? 2 : 1);
      const int64_t l2 = tiles * steps * (kI8Channels + tn) * kI8Step / 12000;
      if (time < l2) time = l2;
      time += s == 1 ? 6 * tn : 1200 + 14 * tn;
      if (least != 0 && time >= least) continue;
      least = time;
      p.tn = (int)tn;
      p.tiles_r = (int)n_r;
      p.split = s;
      p.two = two;
    }
  }
  if (rows > 64 && pairs > 0 && paired + 6 * q.tn <= least) p = q, p.split = 1;
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
