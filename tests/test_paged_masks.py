"""Which values of a tile a row sees, by the attention kernel's own functions compiled for the host (no GPU): boxes that end inside, boxes without any token."""
import os
import re
import shutil
import subprocess

import pytest

from yasakani_b200 import build

PROGRAM = r"""
#include "paged_common.cuh"
#include <cstdio>
namespace kv4 { void set_error(const char*, ...) {} }
using namespace kv4::paged;
int main() {
  long long checked = 0;
  for (int vis : {1, 2, 7, 16, 47, 53, 64, 100, 4096, 1 << 30, 0x7fffffff - 1024})
    for (int at : {0, 16, 48, 64, 4096 - 16, (1 << 30) - 16, 0x7fffffff - 1024 - 64, NO_TOKEN})
      for (int r16 = 0; r16 < 64; r16 += 16)
        for (int j = 0; j < 4; ++j) {
          const int n = vis - box_base(at, vis) - r16 - 2 * j;
          const uint32_t m[2] = {keep_pair(n), keep_pair(n - 8)};
          for (int i = 0; i < 2; ++i)
            for (int e = 0; e < 2; ++e) {
              const bool sees = at != NO_TOKEN && (long long)at + r16 + 2 * j + 8 * i + e < vis, got = m[i] >> (16 * e) & 1;
              if (sees != got || (m[i] >> (16 * e) & 0xffff) != (got ? 0xffffu : 0u)) { std::printf("vis %d at %d r16 %d j %d i %d e %d: %x\n", vis, at, r16, j, i, e, m[i]); return 1; }
              if ((box_base(at, vis) + r16 + 2 * j + 8 * i + e < vis) != sees) { std::printf("score: vis %d at %d\n", vis, at); return 1; }
              ++checked;
            }
        }
  std::printf("%lld\n", checked);
}
"""


def test_masks_of_boxes(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "masks.cu", tmp_path / "masks"
    src.write_text(PROGRAM)
    r = subprocess.run([nvcc, "-std=c++17", "-O0", "-gencode", "arch=compute_100a,code=sm_100a", "-Xcompiler", "-ftrapv", "-I", build.CSRC, "-o", str(exe), str(src)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and int(out.stdout) > 1000, out.stdout + out.stderr


def test_the_kernel_uses_them():
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(build.CSRC, "paged_attn.cu")).read(), flags=re.S)
    assert "box_base(" in code and "keep_pair(" in code and "0x7fffffff" not in code and "0xffff0000" not in code
