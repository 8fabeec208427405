"""The end of a product's tile in LDS (csrc/a8_mx_lds.h): between the barrier behind the other groups' sums
and the end of the kernel a wave reads its sums and writes its staged outputs with nothing to keep it behind
the other waves, so no wave's staging may lie on sums that another has yet to read."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adafactor-8bit_amd", "csrc")


def test_staging_and_sums_lie_apart(tmp_path):
    cc = shutil.which("g++") or shutil.which("c++")
    if cc is None:
        pytest.skip("no host C++ compiler")
    kinds = [(ni, kg, b) for ni, kg in ((1, 1), (2, 1), (4, 1), (1, 4)) for b in (2, 4)]
    lines = ["#include <cstdio>", '#include "a8_mx_lds.h"', "int main() {"]
    for ni, kg, b in kinds:
        e = f"a8::MxEnd<{ni}, {kg}, {b}>"
        lines.append(f'  for (int w = 0; w < 4; ++w) printf("{ni} {kg} {b} 0 %d %d\\n", {e}::staged(w), {e}::kPart);')
        lines.append(f"  for (int g = 1; g < {kg}; ++g) for (int w = 0; w < 4; ++w)")
        lines.append(f'    printf("{ni} {kg} {b} 1 %d %d\\n", {e}::sums(g, w), {e}::kWaveSums);')
        lines.append(f'  printf("{ni} {kg} {b} 2 0 %d\\n", {e}::kBytes);')
    src = tmp_path / "lds.cpp"
    src.write_text("\n".join(lines + ["}"]) + "\n")
    exe = tmp_path / "lds"
    subprocess.run([cc, "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        ni, kg, b, what, at, size = map(int, line.split())
        out.setdefault((ni, kg, b), []).append((what, at, size))
    assert sorted(out) == sorted(kinds)
    for kind, parts in out.items():
        ni, kg, b = kind
        end = [size for what, _, size in parts if what == 2][0]
        parts = sorted((at, at + size) for what, at, size in parts if what != 2)
        assert len(parts) == 4 * kg and parts[0][0] == 0 and parts[-1][1] <= end, kind
        assert all(at % 16 == 0 for at, _ in parts), kind
        assert all(a[1] <= n[0] for a, n in zip(parts, parts[1:])), (kind, parts)
        assert all(stop - at >= 32 * 32 * ni * b for at, stop in parts[:4]), kind
