"""Sizes of the mixture operators' launches (mixture_rules.h), evaluated by a host program."""
import os
import subprocess
import tempfile

from test_mixture_rules import CSRC, evaluate  # noqa: F401


def test_launches_have_fewer_than_2_to_the_32_threads(evaluate):
    """The runtime would take more with their number wrapped round, and leave most of the work undone."""
    assert evaluate(["launchable((1u << 24) - 1, 256)", "launchable(1u << 24, 256)", "launchable((1ull << 32) + 1, 64)",
                     "launchable((1u << 22) - 1, 1024)"]) == [1, 0, 0, 1]
    # copies of operands: a stack of 1024 experts of 9000 x 4095 is 75 GB
    assert evaluate(["pad_blocks(9000, 1024, 4095)", "3 * (uint64_t)pad_blocks(9000, 1024, 4095) * 256 < 1ull << 32", "pad_blocks(3, 2, 9)",
                     "loop_blocks((1u << 24) + 2)", "loop_blocks(1025)"]) == [1 << 20, 1, 1, 1 << 20, 1025]


def test_what_is_made_for_a_kernel_is_made_for_each():
    """Kernels of one type each get their limit on LDS, and each once."""
    program = """
#include "mixture_rules.h"
#include <stdio.h>
void a(int) {}
void b(int) {}
int main() {
  int made = 0;
  auto make = [&] { return ++made; };
  for (int i = 0; i < 3; ++i) {
    if (th::once_for<a>(make) == th::once_for<b>(make)) return 1;
  }
  return made == 2 ? 0 : 2;
}
"""
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "once.cpp"), os.path.join(d, "once")
        with open(src, "w") as f:
            f.write(program)
        subprocess.run(["g++", "-std=c++20", "-Wall", "-Werror", "-I", CSRC, src, "-o", exe], check=True)
        assert subprocess.run([exe]).returncode == 0
