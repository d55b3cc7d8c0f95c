"""How a launch of the logit controls cuts its work: the kernel's own host
arithmetic, compiled here, over rows, vocabularies, history widths and biases."""
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "an-operating-system-for-ai-models-and-tensor-inference_b200", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include "logits_plan.h"
using namespace myos;
int main() {
  const size_t rows[] = {1, 2, 12, 16, 18, 19, 36, 37, 40, 64, 74, 75, 148, 149, 296, 333, 5000};
  const int vocabs[] = {1, 33, 500, 2048, 4095, 16384, 16385, 32003, 65536, 98304, 100003, 151936, 152064, 262147, 1 << 30};
  const size_t widths[] = {0, 1, 2, 3, 4, 5, 8, 100, 170, 171, 256, 1366, 4096, 13654, 32768, 1 << 30};
  const size_t biases[] = {0, 1, 7, 300, 100000, 1 << 30};
  const struct { int threads, depth; } kinds[] = {{1024, 0}, {512, 0}, {512, 4}};
  long cases = 0, bad = 0;
  for (auto kind : kinds)
    for (size_t r : rows)
      for (int v : vocabs)
        for (int cluster = 1; cluster <= kMaxCluster; cluster *= 2)
          for (size_t w : widths)
            for (int b = -1; b < 6; ++b)
              for (int mask = 0; mask < 2; ++mask) {
                const LogitPlan p = logit_plan(kind.threads, kind.depth, cluster, v, r, w, b >= 0,
                                               b >= 0 ? biases[b] : 0, mask);
                const bool some = w > 0 || b >= 0;
                bool ok = p.chunk > 0 && p.chunk % kRun == 0 && p.chunk <= kMaxChunk;
                if (some)  // a list, a table with room to spare, and ids in every step
                  ok = ok && p.room >= (int)kLeastRoom && p.room <= (int)kMostRoom && p.slots > p.room &&
                       p.slots % 4 == 0 && p.slots <= 65536 && logit_step(false, p.chunk, p.slots) >= kRun;
                else
                  ok = ok && p.room == 0 && p.slots == 0;
                ok = ok && logit_step(false, p.chunk, p.slots) <= p.slots;
                ok = ok && logit_step(true, p.chunk, p.slots) == p.chunk;
                ok = ok && p.smem <= logit_smem(kMaxChunk, kMostRoom, true, kind.threads, kind.depth) &&
                     p.smem <= 227 * 1024 - 1024;
                ++cases;
                if (!ok && bad++ < 10)
                  printf("threads %d depth %d cluster %d rows %zu vocab %d width %zu biases %d mask %d: chunk %d room %d slots %d step %d\n",
                         kind.threads, kind.depth, cluster, r, v, w, b, mask, p.chunk, p.room, p.slots,
                         logit_step(false, p.chunk, p.slots));
              }
  for (size_t r : rows)
    for (int v : vocabs)
      for (int threads = 512; threads <= 1024; threads *= 2) {
        const int c = logit_cluster(r, v, threads, 148);
        if (c < 1 || c > kMaxCluster || (c & (c - 1)) || (c > 1 && (v / c < 2048 || r * c > 148u * 1024 / threads))) ++bad;
      }
  printf("%ld cases, %ld bad\n", cases, bad);
  return bad != 0;
}
"""


def test_every_plan_has_room_for_its_tokens(tmp_path):
    """Whatever is listed has a list and a table, and every step has ids: a step
    of none would never end."""
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
