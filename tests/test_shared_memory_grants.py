"""How much dynamic shared memory a kernel was allowed, per kernel and device: the bookkeeping, compiled for the host."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <stdexcept>
#include "shared_memory.h"
int main() {
  q38::SharedMemoryGrants grants;
  int a, b;
  auto ask = [&](const void* kernel, int device, int bytes) { grants.ensure(kernel, device, bytes, [&] { std::printf("%s %d %d\n", kernel == &a ? "a" : "b", device, bytes); }); };
  ask(&a, 0, 100000);
  ask(&a, 0, 100000);
  ask(&a, 0, 50000);      // less than allowed
  ask(&a, 1, 50000);      // a device of its own
  ask(&b, 0, 50000);      // a kernel of its own
  ask(&a, 0, 200000);     // more than allowed
  ask(&a, 0, 200000);
  try { grants.ensure(&b, 1, 300000, [] { throw std::runtime_error("refused"); }); } catch (const std::runtime_error&) { std::printf("refused\n"); }
  ask(&b, 1, 300000);     // what was refused is asked for again
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_a_larger_request_is_passed_on(tmp_path):
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main"), "-pthread"], check=True)
    lines = subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert lines == ["a 0 100000", "a 1 50000", "b 0 50000", "a 0 200000", "refused", "b 1 300000"]


def test_every_permission_goes_through_it():
    """The remembered amount is what the driver was told only if nothing else lowers it for the same kernels."""
    for name in ("layernorm.cu", "vocab_loss.cu", "rotary.cu", "clip.cu"):
        assert "cudaFuncSetAttribute" not in (CSRC / name).read_text(), name
