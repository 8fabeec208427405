"""Sizes past one grid's 2^32 - 1 work-items: csrc/a8_launch.h, and the refusals of what no run can cover."""
import os
import shutil
import subprocess

import pytest

from adafactor8bit import _native as nat

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adafactor-8bit_amd", "csrc")
MAIN = """
#include <cstdio>
#include "a8_launch.h"
int main() {
  const int threads[] = {64, 256, 512, 1024};
  for (int t : threads) printf("%lld\\n", (long long)a8::most_groups(t));
  const long long totals[] = {0, 1, 6, 7, 8, 21, 22};
  for (long long total : totals) {
    int e = a8::in_runs(total, 7, [](int64_t first, int64_t n) { return printf("%lld+%lld ", (long long)first, (long long)n), 0; });
    printf("%d\\n", e);
  }
  int calls = 0;
  const int e = a8::in_runs(21, 7, [&](int64_t, int64_t) { return ++calls == 2 ? 9 : 0; });
  printf("%d %d\\n", e, calls);
}
"""


def test_runs_cover_everything_once(tmp_path):
    cc = shutil.which("g++") or shutil.which("c++")
    if cc is None:
        pytest.skip("no host C++ compiler")
    (tmp_path / "runs.cpp").write_text(MAIN)
    exe = tmp_path / "runs"
    subprocess.run([cc, "-std=c++17", "-I", CSRC, str(tmp_path / "runs.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    for threads, n in zip((64, 256, 512, 1024), map(int, out)):
        assert n * threads < 2 ** 32 <= (n + 1) * threads
    assert out[4:] == ["0", "0+1 0", "0+6 0", "0+7 0", "0+7 7+1 0", "0+7 7+7 14+7 0", "0+7 7+7 14+7 21+1 0", "9 2"]


def test_sizes_that_no_launch_covers_are_refused():
    """Refused by the size check, before anything is launched."""
    L, one, size = nat.lib(), 16, -4   # a non-null, aligned address that no refused call reads
    # 128 x 128 tiles down and across: 2^24 workgroups of 256
    assert L.a8_mx_quantize(1, 0, 0, 0, one, 1 << 30, 1, 1, None, None, one, one, 0, None) == size
    assert L.a8_mx_quantize(1, 0, 0, 0, one, 1 << 30, 1, 1, one, one, one, one, 0, None) == size
    # one row of a, 32 rows of b a workgroup
    assert L.a8_mx_matmul(0, 0, 1, one, one, one, one, one, 1, 1 << 30, 256, None) == size
    assert L.a8_mx_matmul(0, 1, 1, one, one, one, one, one, 4, (1 << 31) - 1, 256, None) == size
    # 128 x 128 and 256 x 256 tiles
    assert L.a8_mx_matmul(0, 0, 1, one, one, one, one, one, 1 << 22, 1 << 22, 256, None) == size
    # dw: 32 columns a workgroup of 1024
    assert L.a8_rms_norm_backward(1, 1, 1, one, None, one, None, one, one, one, None, one, one, 1, 1 << 27, None) == size
