"""CPU: the parts of cut sequences, up to the most tokens that a call takes.  csrc/linear.cuh is compiled as it is, for the host."""
import os
import shutil
import subprocess

import pytest

from tests.test_barrier_order import CSRC

MOST = 2147418111
SIZES = [(n, seg) for seg in (64, 128, 14509696, 7379456, 65536, 1 << 30, 2147483520) for n in (0, 1, 63, 64, 65, 128, 129, seg - 1, seg, seg + 1, 2132973952, 2132973953, 2140104192, MOST - 1, MOST) if 0 <= n <= MOST]
PROGRAM = """
#include <cstdio>
#include "linear.cuh"
int main() {
    int n, seg;
    while (scanf("%d %d", &n, &seg) == 2) printf("%d\\n", mkda::part_count(n, seg));
}
"""


def test_parts_of_long_sequences(tmp_path):
    nvcc = shutil.which("nvcc")
    if not nvcc:
        pytest.skip("needs nvcc")
    (tmp_path / "parts.cu").write_text(PROGRAM)
    exe = str(tmp_path / "parts")
    subprocess.run([nvcc, "-std=c++17", "-Wno-deprecated-gpu-targets", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, str(tmp_path / "parts.cu"), "-o", exe], check=True)
    out = subprocess.run([exe], input="\n".join("%d %d" % s for s in SIZES), capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == [max(1, -(-n // seg)) for n, seg in SIZES]


def test_no_kernel_counts_parts_by_itself():
    for name in ("linear.cu", "linear.cuh", "linear_tc.cu", "scan.cu"):
        assert "seg - 1) /" not in open(os.path.join(CSRC, name)).read(), name
