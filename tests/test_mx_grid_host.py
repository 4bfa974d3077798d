"""The grids of the microscaled byte movers: fewer than 2^32 threads along x at every count of workgroups."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <stdio.h>
#include "qik_host.h"
static int bad = 0;
static void check(int64_t n, int threads) {
  unsigned x = 0, y = 0;
  if (!qik_host::split_grid(n, threads, &x, &y) || (uint64_t)x * threads >> 32 != 0 || y > 65535 ||
      (int64_t)x * y < n || (int64_t)x * y - n >= y) {
    printf("%lld workgroups of %d: %u x %u\n", (long long)n, threads, x, y);
    ++bad;
  }
}
int main() {
  const int sizes[] = {64, 256, 512, 1024};
  for (int threads : sizes) {
    const int64_t full = ((int64_t)1 << 32) / threads;  // workgroups of 2^32 threads
    for (int64_t k = 1; k <= 40; ++k)
      for (int64_t j = -50; j <= 50; ++j)
        if (k * full + j > 0) check(k * full + j, threads);
    for (int64_t n = 1; n < 65000 * full; n = n * 3 / 2 + 1) check(n, threads);
    for (int64_t n = 1; n <= 100; ++n) check(n, threads);
    unsigned x, y;
    bad += qik_host::split_grid(0, threads, &x, &y) || qik_host::split_grid(65535 * full, threads, &x, &y);
  }
  return bad != 0;
}
"""


def test_grids_stay_below_2_to_32_threads_in_x(tmp_path):
    src, exe = tmp_path / "grid.cpp", tmp_path / "grid"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{os.path.join(ROOT, 'include')}",
                    f"-I{os.path.join(ROOT, 'qwen-image-kernel_amd', 'csrc')}", str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout[-2000:]
