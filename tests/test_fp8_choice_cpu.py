"""Which kernel an FP8 product takes (csrc/qkm_fp8_choice.h), asked on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "qkm_fp8_choice.h"
#include <cstdio>
#include <cstdlib>
int main(int, char** v) {
    std::printf("%d\n", qkm::fp8_pairs_as_lanes(atoi(v[1]), atoi(v[2]), atoi(v[3])) ? 1 : 0);
    return 0;
}
"""


@pytest.fixture(scope="module")
def as_lanes(tmp_path_factory):
    d = tmp_path_factory.mktemp("choice")
    (d / "choice.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "qwen-kernel_b200", "csrc"), str(d / "choice.cpp"), "-o", str(d / "choice")], check=True)
    return lambda *args: subprocess.run([str(d / "choice"), *[str(a) for a in args]], check=True, capture_output=True, text=True).stdout.strip() == "1"


def test_experts_from_44_pairs_on(as_lanes):
    """The mean is not rounded, and 44 itself counts."""
    assert as_lanes(1408, 8, 256) and not as_lanes(1407, 8, 256)
    assert as_lanes(88, 1, 2) and not as_lanes(87, 1, 2)
    assert not as_lanes(1, 16, 16) and as_lanes((1 << 27) - 1, 16, 16)


def test_a_shard_goes_by_the_whole_table():
    """Its list has its own experts' pairs alone: 192 tokens of top 8 are 6 pairs an expert of 256, whatever part of them is resident."""
    source = open(os.path.join(ROOT, "qwen-kernel_b200", "csrc", "qkm_api.cu")).read()
    assert "a.n_table = c->cfg.dims.n_expert;" in source
    source = open(os.path.join(ROOT, "qwen-kernel_b200", "csrc", "qkm_fp8_gemm.cu")).read()
    assert "fp8_pairs_as_lanes(a.n, a.n_used, a.n_table)" in source
