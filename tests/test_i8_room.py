"""What a device holds in clusters, as the 8-bit product keeps it: the kernel's own host
code, compiled here with a device that cannot always be asked."""
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "an-operating-system-for-ai-models-and-tensor-inference_b200", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include <atomic>
#include <string>
#include "i8_plan.h"
using namespace myos;
static std::string asked;
static int no_one, no_two;  // the size that cannot be asked about
static I8Device call(std::atomic<uint64_t>* known) {
  I8Device d = {};
  asked.clear();
  i8_room(d, known, [](int s, bool two, int* blocks) {
    asked += std::to_string(s) + (two ? "t " : " ");
    if (s == (two ? no_two : no_one)) return false;
    *blocks = two ? 290 - s : s == 8 ? 0 : 148 - s;  // (no room is an answer too)
    return true;
  });
  return d;
}
static int bad;
static void want(bool ok, const char* what) {
  if (!ok) printf("%s (asked %s)\n", what, asked.c_str()), bad = 1;
}
int main() {
  static std::atomic<uint64_t> known[kI8MaxSplit + 1];
  no_one = 3, no_two = 6;
  I8Device d = call(known);
  want(asked == "2 2t 3 3t 4 4t 6 6t 8 8t ", "the sizes that tiles are cut into, each once");
  want(d.one[2] == 146 && d.two[2] == 288 && d.one[8] == 0 && d.two[8] == 282, "answers");
  want(d.one[3] == 0 && d.two[3] == 287 && d.one[6] == 142 && d.two[6] == 0, "no room where it could not be asked");
  want(d.one[5] == 0 && d.one[7] == 0 && d.one[1] == 0, "other sizes");
  no_one = 0;
  d = call(known);
  want(asked == "3 3t 6 6t ", "what could not be had is asked again, and nothing else");
  want(d.one[3] == 145 && d.two[3] == 287 && d.one[6] == 142 && d.two[6] == 0, "answers of the second call");
  no_two = 0;
  d = call(known);
  want(asked == "6 6t " && d.two[6] == 284, "the third call");
  d = call(known);
  want(asked == "" && d.one[2] == 146 && d.two[3] == 287 && d.two[6] == 284 && d.one[8] == 0, "all known");
  return bad;
}
"""


def test_an_answer_that_could_not_be_had_is_asked_for_again(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("g++ not available")
    src, exe = tmp_path / "room.cpp", tmp_path / "room"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
