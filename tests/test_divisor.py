"""swd::Divisor (sparsewavecomp_amd/csrc/sw_divisor.h), by which the kernels divide
positions and indexes, compiled for the host with g++ and compared with the
quotient: every divisor that a page size, a number of heads or of pieces can be,
numbers on both sides of its multiples and up to 2^31 - 1."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include "sw_divisor.h"
#include <cstdio>
int main() {
  unsigned d, n;
  while (std::scanf("%u %u", &d, &n) == 2)
    std::printf("%u\n", swd::Divisor(d).quotient(n));
  return swd::Divisor().quotient(7) != 7;
}
'''


@pytest.fixture(scope="module")
def divide(tmp_path_factory):
    gxx = shutil.which("g++")
    hip = "/opt/rocm/include/hip/hip_runtime.h"
    if gxx is None or not os.path.exists(hip):
        pytest.skip("g++ and the HIP headers are needed")
    d = tmp_path_factory.mktemp("divisor")
    src, exe = d / "divisor.cpp", d / "divisor"
    src.write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include",
                    "-I" + os.path.join(ROOT, "sparsewavecomp_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True)

    def run(cases):
        inp = "".join(f"{d} {n}\n" for d, n in cases)
        out = subprocess.run([str(exe)], input=inp, capture_output=True,
                             text=True, check=True).stdout.split()
        return [int(q) for q in out]
    return run


def test_quotients(divide):
    rng = random.Random(3)
    divisors = [*range(1, 260), 1000, 1023, 1024, 1025, 65535, 65536, 131072,
                2 ** 20, 2 ** 20 + 1, 3 * 2 ** 28, 2 ** 30 - 1, 2 ** 30]
    divisors += [rng.randrange(2, 1 << rng.randrange(2, 31))
                 for _ in range(2000)]
    cases = []
    for d in divisors:
        last = (2 ** 31 - 1) // d * d
        cases += [(d, n) for n in (
            0, 1, d - 1, d, d + 1, last - 1, last, 2 ** 31 - 1,
            rng.randrange(2 ** 31), rng.randrange(2 ** 31) // d * d)
            if 0 <= n < 2 ** 31]
    assert divide(cases) == [n // d for d, n in cases]
