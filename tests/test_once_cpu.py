"""csrc/a8_once.h: a kernel's LDS limit is set for every device that it runs on, and again after a failure."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adafactor-8bit_amd", "csrc")
MAIN = """
#include <cstdio>
#include <initializer_list>
#include "a8_once.h"
int main() {
  static a8::OncePerDevice once, other;
  int calls = 0;
  auto set = [&](int result) { return [&calls, result] { ++calls; return result; }; };
  auto show = [&](int r) { printf("%d %d\\n", r, calls); };
  for (int device : {0, 0, 1, 1, 0, 7, 63, 63}) show(once(device, set(0)));
  show(once(3, set(5)));
  show(once(3, set(0)));
  show(once(3, set(5)));
  show(other(0, set(0)));
  show(once(64, set(0)));
  show(once(64, set(0)));
  show(once(-1, set(0)));
}
"""


def test_every_device_is_set_once(tmp_path):
    cc = shutil.which("g++") or shutil.which("c++")
    if cc is None:
        pytest.skip("no host C++ compiler")
    (tmp_path / "once.cpp").write_text(MAIN)
    exe = tmp_path / "once"
    subprocess.run([cc, "-std=c++17", "-I", CSRC, str(tmp_path / "once.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    want = [(0, 1), (0, 1), (0, 2), (0, 2), (0, 2), (0, 3), (0, 4), (0, 4),   # first calls on 0, 1, 7 and 63
            (5, 5), (0, 6), (0, 6),                                            # a failure is tried again
            (0, 7),                                                            # another kernel's
            (0, 8), (0, 9), (0, 10)]                                           # not remembered: set each time
    assert [tuple(map(int, line.split())) for line in out] == want
