"""How a product of 8-bit rows and channels is cut: the kernel's own host arithmetic,
compiled here, over rows, k and channels, for a whole device and smaller ones."""
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "an-operating-system-for-ai-models-and-tensor-inference_b200", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include "i8_plan.h"
using namespace myos;
int main() {
  const int64_t rows[] = {1, 2, 8, 9, 15, 16, 17, 32, 33, 63, 64, 65, 96, 127, 128, 129, 200, 255, 256, 257, 333, 511, 512,
                          513, 1000, 2048, 4097, 8191, 65536, 1000003, 0x7fffff00};
  const int64_t ks[] = {1, 15, 16, 31, 32, 33, 64, 127, 128, 129, 383, 384, 385, 1024, 1536, 5120, 8960, 13824, 32768, 131071};
  const int64_t channels[] = {1, 7, 8, 15, 16, 17, 127, 128, 129, 255, 256, 257, 512, 1000, 1536, 2048, 5120, 7168, 17920, 27648,
                              151936, 1000003, 0x7fffff00};
  // a B200; one without room for clusters of more than 2; one that could not be asked; few multiprocessors
  const I8Device devices[] = {
      {148, {0, 0, 148, 135, 132, 130, 132, 105, 120}, {0, 0, 296, 279, 284, 280, 270, 259, 264}},
      {148, {0, 0, 148, 0, 0, 0, 0, 0, 0}, {0, 0, 148, 0, 0, 0, 0, 0, 0}},
      {148, {0}, {0}},
      {16, {0, 0, 16, 15, 16, 15, 12, 14, 16}, {0, 0, 32, 30, 32, 30, 30, 28, 32}},
      {1, {0}, {0}}};
  long cases = 0, bad = 0;
  for (const I8Device& d : devices)
    for (int64_t r : rows)
      for (int64_t k : ks)
        for (int64_t c : channels) {
          const I8Few f = i8_few(r, k, c);
          bool ok = !f.use || r <= kI8FewRows;
          ok = ok && (f.groups == 1 || f.groups == 2 || f.groups == 4) && f.warps >= 2 && f.warps <= 8;
          ok = ok && f.warps * 16 * f.groups * 8 * 4 <= 48 * 1024;  // its shared memory, without raising the limit
          const I8Plan p = i8_plan(r, k, c, d);
          const int64_t steps = i8_ceil(k, kI8Step), tiles = (int64_t)p.tiles_c * p.tiles_r;
          const int blocks = p.pair ? 2 : p.split;
          // tiles cover everything, none is empty, and the tensor core takes their shape
          ok = ok && p.tc == (p.pair ? 256 : 128) && p.tn % (p.pair ? 32 : 16) == 0 && p.tn >= 16 && p.tn <= 256;
          ok = ok && (int64_t)p.tiles_c * p.tc >= c && (int64_t)(p.tiles_c - 1) * p.tc < c;
          ok = ok && (int64_t)p.tiles_r * p.tn >= r && (int64_t)(p.tiles_r - 1) * p.tn < r;
          // every block of a cluster has k, and the whole cluster is resident at once
          ok = ok && p.split >= 1 && p.split <= kI8MaxSplit && p.split != 5 && p.split != 7 && p.split <= steps && !(p.pair && p.split > 1);
          if (p.split > 1) ok = ok && tiles * p.split <= (p.two ? d.two[p.split] : d.one[p.split]);
          ok = ok && !(p.two && (p.tn > 64 || p.pair)) && !(p.apart && p.split == 1);
          // shared memory: stages, and the sums behind or over them
          const int stage = (kI8Channels + p.tn / (p.pair ? 2 : 1)) * kI8Step;
          const int sums = p.split > 1 ? p.split * p.tn * i8_wide(p.split) * 4 : 0;
          ok = ok && p.stages >= 3 && p.stages <= kI8MaxStages && p.stages + 2 < 31 && stage % 1024 == 0;
          ok = ok && p.stages * stage + (p.apart ? sums : 0) <= (p.two ? kI8SmemTwo : kI8Smem);
          ok = ok && (p.split == 1 || p.apart || sums <= p.stages * stage);
          ok = ok && i8_wide(p.split) * p.split >= kI8Channels && i8_wide(p.split) % 4 == 0;
          // tensor memory: two accumulators, of all blocks of a multiprocessor
          ok = ok && p.columns >= 2 * p.tn && p.columns * (p.two ? 2 : 1) <= 512 && (p.columns & (p.columns - 1)) == 0;
          ok = ok && p.group >= 1 && p.group <= p.tiles_r;
          // the last row that a copy or a store names fits 32 bits
          ok = ok && (int64_t)p.tiles_r * p.tn + 256 < ((int64_t)1 << 31) + 256 && blocks <= 8;
          ++cases;
          if (!ok && bad++ < 10)
            printf("rows %ld k %ld channels %ld on %d: pair %d tn %d split %d two %d stages %d columns %d group %d tiles %d x %d\n",
                   (long)r, (long)k, (long)c, d.sms, p.pair, p.tn, p.split, p.two, p.stages, p.columns, p.group, p.tiles_c, p.tiles_r);
        }
  printf("%ld cases, %ld bad\n", cases, bad);
  return bad != 0;
}
"""


def test_every_cut_covers_its_product_and_fits(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
