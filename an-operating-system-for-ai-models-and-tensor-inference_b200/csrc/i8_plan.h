// How a product of 8-bit rows and channels is cut into tiles (host arithmetic).
#pragma once
#include <stdint.h>
#include <stdlib.h>

namespace myos {

constexpr int kI8Channels = 128;      // channels of a tile: the tensor core's M
constexpr int kI8Step = 128;          // bytes of k of a stage: one swizzled row
constexpr int kI8MaxRows = 256;       // rows of a tile at most: its N
constexpr int kI8MaxStages = 12;
constexpr int kI8Smem = 200 * 1024;     // a block's shared memory,
constexpr int kI8SmemTwo = 109 * 1024;  // where two share a multiprocessor
constexpr int kI8MaxSplit = 8;        // blocks that share a tile's k: a portable cluster

struct I8Plan {
  int pair;             // a tile is two blocks': 256 channels
  int tc;               // channels of a tile
  int tn;               // rows of a tile, a multiple of 16 (of a pair: of 32)
  int split;            // blocks (a cluster) along k
  int stages;
  int two;              // two blocks a multiprocessor
  int apart;            // the cluster's sums have their own place behind the stages
  int vec;              // four results are stored at once (the caller's to say)
  int tiles_c, tiles_r;
  int columns;          // of tensor memory: two accumulators, a power of two
};

inline int i8_ceil(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

inline I8Plan i8_plan(int64_t rows, int64_t k, int64_t channels, int sms) {
  I8Plan p;
  const int steps = i8_ceil(k, kI8Step);
  p.pair = getenv("I8_PAIR") ? atoi(getenv("I8_PAIR")) && rows > 16 : rows > 256;
  p.tc = p.pair ? 2 * kI8Channels : kI8Channels;
  p.tiles_c = i8_ceil(channels, p.tc);
  p.tiles_r = i8_ceil(rows, kI8MaxRows);
  const int unit = p.pair ? 32 : 16;
  p.tn = i8_ceil(i8_ceil(rows, p.tiles_r), unit) * unit;
  p.tiles_r = i8_ceil(rows, p.tn);
  const int64_t tiles = (int64_t)p.tiles_c * p.tiles_r;
  p.two = !p.pair && p.tn <= 64;
  p.split = 1;
  while (p.split < kI8MaxSplit && p.split * 2 <= steps && tiles * p.split * 2 <= sms) p.split *= 2;
  if (const char* e = getenv("I8_S")) p.split = atoi(e);
  if (const char* e = getenv("I8_TWO")) p.two = atoi(e) && p.tn <= 64 && !p.pair;
  if (p.split > steps) p.split = steps;
  if (p.pair) p.split = 1;
  const int sums = p.tn * kI8Channels * 4;
  p.apart = p.split > 1 && p.tn <= 64;
  const int stage = (kI8Channels + p.tn / (p.pair ? 2 : 1)) * kI8Step;
  p.stages = ((p.two ? kI8SmemTwo : kI8Smem) - (p.apart ? sums : 0)) / stage;
  if (p.stages > kI8MaxStages) p.stages = kI8MaxStages;
  p.columns = 32;
  while (p.columns < 2 * p.tn) p.columns *= 2;
  return p;
}

}  // namespace myos
