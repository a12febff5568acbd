"""The count of clusters that a device holds is kept for each device, and only where the device gave it (no GPU)."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oxidized_gpt_oss_b200", "csrc")
PROGRAM = """
#include "cluster_count.h"
#include <cstdio>
int main() {
  static oxg::ClusterCount known;
  int asked = 0, answer = 0;
  auto ask = [&] { ++asked; return answer; };
  auto is = [&](int device, int want, int want_asked) {
    const int got = known.get(device, 74, ask);
    if (got != want || asked != want_asked) std::printf("device %d: %d after %d questions\\n", device, got, asked);
    return got == want && asked == want_asked;
  };
  bool ok = true;
  answer = 0;
  ok &= is(0, 74, 1);   // a failed question: this call goes by the estimate
  answer = -1;
  ok &= is(0, 74, 2);
  answer = 70;
  ok &= is(0, 70, 3);   // and the next one asks again
  answer = 66;
  ok &= is(0, 70, 3);   // an answer is kept
  ok &= is(1, 66, 4);   // for its device
  ok &= is(0, 70, 4) && is(1, 66, 4);
  ok &= is(64, 66, 5) && is(64, 66, 6) && is(-1, 66, 7);  // devices beyond the table are asked every time
  return ok ? 0 : 1;
}
"""


def test_counts_are_kept_by_device_and_failures_are_not(tmp_path):
    src, exe = tmp_path / "count.cc", tmp_path / "count"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
