"""Every form that the 8-bit product takes on a B200 is among the shapes that are run
here: on the CPU the kernel's own host arithmetic, compiled, says which form a shape
has; on the GPU each is compared bit for bit."""
import os
import shutil
import subprocess

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "an-operating-system-for-ai-models-and-tensor-inference_b200", "csrc")

# rows, k, channels
SHAPES = [
    # straight from memory: 8, 16, 32 channels a block, 2 to 8 warps, up to 8 and up to 16 rows
    (1, 1536, 2048), (8, 8960, 1536), (1, 5120, 7168), (5, 1536, 17920), (3, 500, 40000), (7, 5120, 27648),
    (9, 1536, 2048), (16, 5120, 2048), (9, 1000, 9000), (16, 1536, 17920), (12, 200, 40000), (16, 5120, 12000), (13, 700, 6001),
    # tiles of one block, one and two a multiprocessor
    (19, 64, 64), (64, 5120, 27648), (33, 130, 30000), (6250, 65, 132), (17, 640, 25001),
    # of 16 rows, one and two a multiprocessor
    (10, 5404, 12419), (16, 5120, 15001), (12, 1536, 151936), (10, 3208, 20921), (9, 1000, 70003),
    # k in 2, 3, 4, 6, 8 parts, the sums behind the stages
    (64, 5120, 7168), (33, 3700, 6001), (64, 13824, 5120), (17, 1287, 64), (17, 1410, 64), (64, 1536, 2048), (18, 2204, 64),
    (64, 2944, 2048), (17, 2998, 65), (64, 8960, 1537),
    # the sums over the stages
    (66, 5302, 6840), (130, 2324, 132), (2547, 2324, 132), (128, 13824, 5120), (1496, 1412, 143), (519, 1956, 390), (250, 2500, 700),
    (66, 2200, 66), (200, 3300, 301), (67, 2954, 66), (255, 8960, 130),
    # two blocks a multiprocessor; 16 rows
    (20, 2570, 9484), (64, 2700, 9501), (16, 13824, 5120), (11, 7620, 8807), (11, 14309, 4691), (13, 6578, 10208), (15, 16247, 4139),
    # pairs
    (66, 64, 68), (128, 1536, 2048), (333, 5120, 7168), (1024, 1536, 4001),
]

PROGRAM = r"""
#include <math.h>
#include <stdio.h>
#include <random>
#include <set>
#include <tuple>
#include "i8_plan.h"
using namespace myos;
typedef std::tuple<int, int, int, int, int> Form;
static Form form(int64_t r, int64_t k, int64_t c) {
  const I8Few f = i8_few(r, k, c);
  if (f.use) return Form(2, f.groups, f.warps, r > 8, 0);
  const I8Device d = {148, {0, 0, 148, 135, 132, 130, 132, 105, 120}, {0, 0, 296, 279, 284, 280, 270, 259, 264}};
  const I8Plan p = i8_plan(r, k, c, d);
  return Form(p.pair, p.split, p.two, p.apart, p.tn == 16);
}
int main() {
  std::set<Form> run;
  long r, k, c;
  while (scanf("%ld %ld %ld", &r, &k, &c) == 3) run.insert(form(r, k, c));
  std::mt19937_64 g(1);
  auto some = [&](double lo, double hi) { return (int64_t)(lo * exp((double)(g() >> 11) / 9007199254740992.0 * log(hi / lo))); };
  std::set<Form> missing;
  for (int i = 0; i < 2000000; ++i) {
    const int64_t r = some(1, 8193), k = some(16, 16385), c = some(1, 160000);
    if (k * c > ((int64_t)1 << 31)) continue;
    const Form f = form(r, k, c);
    if (!run.count(f) && missing.insert(f).second)
      printf("(%d %d %d %d %d): %ld x %ld x %ld\n", std::get<0>(f), std::get<1>(f), std::get<2>(f), std::get<3>(f),
             std::get<4>(f), (long)r, (long)k, (long)c);
  }
  printf("%zu forms run, %zu missing\n", run.size(), missing.size());
  return !missing.empty();
}
"""


def test_no_form_is_missing(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    src, exe = tmp_path / "forms.cpp", tmp_path / "forms"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    shapes = "\n".join("%d %d %d" % s for s in SHAPES)
    r = subprocess.run([str(exe)], input=shapes, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,channels", SHAPES)
def test_product(rows, k, channels):
    """f32 whole, bf16 in rows that are no multiple of four apart."""
    import torch
    from myos import dev
    from test_gpu_i8 import check_product

    rng = np.random.default_rng(rows + k)
    check_product(dev, rng, rows, k, channels)
    check_product(dev, rng, rows, k, channels, bias=False, dtype=torch.bfloat16, out_pad=4 - channels % 4 + 1)
    if channels % 4 == 0:
        check_product(dev, rng, rows, k, channels, dtype=torch.bfloat16)
