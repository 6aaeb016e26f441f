"""CPU (nvcc alone): how many tries the bounded waits of the tensor-core kernels take, counted on the host with the function that the kernels
call after every try."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")

SOURCE = """
#include <stdio.h>
#include "tcgen05.cuh"
using namespace f2c::t5;
// tries of a wait whose phase completes with number `when` (0: never)
static unsigned long long wait(uint32_t& left, unsigned long long when) {
  unsigned long long n = 0;
  uint32_t spent = 0;
  do ++n; while (n < (1ull << 25) && tries_again(n == when, spent, left));
  return n;
}
int main() {
%s
}
"""


def counts(tmp_path, body):
    (tmp_path / "count.cu").write_text(SOURCE % body)
    subprocess.run([NVCC, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a", "-I",
                    os.path.join(ROOT, "f2cgt_b200", "csrc"), "-o", "count", "count.cu"], cwd=tmp_path, check=True, capture_output=True, text=True)
    out = subprocess.run(["./count"], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
    return [int(v) for v in out.split()]


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no CUDA compiler")
def test_a_role_that_has_given_up_tries_once(tmp_path):
    """Waits that find nothing after one that ran out, and waits whose phase is complete: one try each, and no tries come back."""
    limit, first, then, last = counts(tmp_path, """
  uint32_t left = kWaitLimit;
  const unsigned long long first = wait(left, 0);
  unsigned long long then = 0;
  for (int i = 0; i < 5; ++i) then += wait(left, 0);
  then += wait(left, 1);
  printf("%u %llu %llu %u", kWaitLimit, first, then, left);
""")
    assert first == limit and then == 6 and last == 0


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no CUDA compiler")
def test_waits_that_end_leave_later_ones_their_tries(tmp_path):
    """A hundred waits, each of which ends at its last try, and one that never does."""
    limit, before, after, last = counts(tmp_path, """
  uint32_t left = kWaitLimit;
  for (int i = 0; i < 100; ++i) wait(left, kWaitLimit);
  const uint32_t before = left;
  const unsigned long long after = wait(left, 0);
  printf("%u %u %llu %u", kWaitLimit, before, after, left);
""")
    assert before == limit and after == limit and last == 0
