// How a launch of the logit controls cuts its rows into blocks, passes and
// tables: arithmetic on sizes, for the host (and its tests) and the kernel.
#pragma once
#include <stddef.h>

#ifdef __CUDACC__
#define MYOS_PLAN __host__ __device__ __forceinline__
#else
#define MYOS_PLAN inline
#endif

namespace myos {

constexpr int kMaxCluster = 8;
constexpr int kMaxChunk = 65536, kRun = 128, kRunWords = kRun / 32 + 1;
static_assert(kRunWords <= 8, "eight threads copy a run's mask words");
constexpr size_t kLeastRoom = 512, kMostRoom = 5120;  // multiples of 16
static_assert(kLeastRoom * 5 / 4 >= kRun && kMostRoom * 5 / 4 <= 65536, "a run to a step, slots in 16 bits");

// As many blocks a row as are resident at once, with 2048 ids at least.
inline int logit_cluster(size_t rows, int vocab, int threads, int sms) {
  int cluster = kMaxCluster;
  while (cluster > 1 && (rows * cluster > (size_t)sms * 1024 / threads || vocab / cluster < 2048))
    cluster /= 2;
  return cluster;
}

// Dynamic shared memory of a block.
inline size_t logit_smem(size_t chunk, size_t room, bool mask, int threads, int depth) {
  return (room ? chunk / 8 : 0) + (mask ? 4 * (chunk / kRun * kRunWords + 2) : 0) +
         14 * (room + room / 4) + 8 * room + 16 * (size_t)depth * threads;
}

struct LogitPlan {
  int chunk, slots, room;  // ids of a pass (a multiple of kRun), table slots (of 4), list entries
  size_t smem;
};

// width: of the history (0: no penalties); num_bias: entries of all rows, where
// there are biases; depth: slots of the ring.
inline LogitPlan logit_plan(int threads, int depth, int cluster, int vocab, size_t rows,
                            size_t width, bool biases, size_t num_bias, bool mask) {
  LogitPlan p;
  const int most = ((vocab + 3 + kRun - 1) / kRun + cluster - 1) / cluster * kRun;
  const int passes = (most + kMaxChunk - 1) / kMaxChunk;
  p.chunk = ((most / kRun + passes - 1) / passes) * kRun;
  // a list for three times (beside a ring, so that two blocks fit a multiprocessor,
  // twice) a block's share of the longest history and of the mean number of biases,
  // and five slots of the table for four of its entries; never none where there may
  // be an entry, however few blocks' shares a short history has
  size_t share = width;
  if (biases) share += num_bias / rows + 32;
  size_t room = 0;
  if (share > 0) {
    room = (depth > 0 ? 2 : 3) * share / cluster;
    room = room < kLeastRoom ? kLeastRoom : room > kMostRoom ? kMostRoom : (room + 15) & ~(size_t)15;
  }
  p.room = (int)room;
  p.slots = (int)(room + room / 4);
  p.smem = logit_smem(p.chunk, room, mask, threads, depth);
  return p;
}

// Ids that go at once: the whole chunk where the list holds the block's tokens
// and biases (hashed), else as many as the table has slots.
MYOS_PLAN int logit_step(bool hashed, int chunk, int slots) {
  const int fit = slots & ~(kRun - 1);
  return hashed || chunk < fit ? chunk : fit;
}

}  // namespace myos
