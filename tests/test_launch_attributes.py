"""Kernels with much shared memory have an attribute set before their first launch on a device.  Host calls run without the interpreter lock, so two threads may
come at once: none may pass before the attribute is there, and a failed attempt is made again (the source's own function, compiled for the host; no GPU)."""
import os
import shutil
import subprocess

import pytest

from yasakani_b200 import build

PROGRAM = r"""
#include "kv4_common.cuh"
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
namespace kv4 { void set_error(const char*, ...) {} }
int main() {
  std::atomic<unsigned long long> flags{0};
  std::atomic<int> there{0}, early{0}, calls{0};
  auto use = [&] {
    const int rc = kv4::once_for_bit(flags, 1ull << 3, [&] { ++calls; std::this_thread::sleep_for(std::chrono::milliseconds(200)); there = 1; return 0; });
    if (rc || !there) ++early;
  };
  std::thread a(use);
  while (!calls) std::this_thread::yield();
  std::thread b(use);
  a.join(); b.join();
  use();
  const int after = calls;
  std::atomic<unsigned long long> other{0};
  int tries = 0;
  const int first = kv4::once_for_bit(other, 1, [&] { ++tries; return 7; }), second = kv4::once_for_bit(other, 1, [&] { ++tries; return 0; }),
            third = kv4::once_for_bit(other, 1, [&] { ++tries; return 9; }), device = kv4::once_for_bit(other, 2, [&] { ++tries; return 0; });
  std::printf("early %d calls %d; %d %d %d %d tries %d\n", (int)early, after, first, second, third, device, tries);
}
"""


def test_nobody_launches_before_the_attribute_is_set(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "once.cu", tmp_path / "once"
    src.write_text(PROGRAM)
    r = subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", build.CSRC, "-o", str(exe), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.stdout.strip() == "early 0 calls 2; 7 0 0 0 tries 3", out.stdout + out.stderr


def test_every_launcher_goes_through_it():
    import re
    for path in build.sources():
        code = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)
        for m in re.finditer(r"cudaFuncSetAttribute", code):
            before = code[:m.start()]
            assert before.rfind("once_per_device(") > before.rfind("\n}"), path                # inside a function, behind the call that guards it
