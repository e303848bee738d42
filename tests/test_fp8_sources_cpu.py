"""What the FP8 kernels' source must hold and no run can show: a warp's lanes leave the poll of a barrier in different turns, and the loads from
tensor memory, its return and a cluster's barrier are for whole warps (.aligned), so a __syncwarp() lies between the two."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-kernel_b200", "csrc")
TOKEN = re.compile(r"\bwait_bar\(|\b__syncwarp\(\)|\btmem_(?:load|ld32|ld|ld16|dealloc)\(|\btmem_give_back<CG>\(|\bcluster_sync\(\)")


def _kernels():
    text = open(os.path.join(CSRC, "qkm_fp8_gemm.cu")).read()
    text = re.sub(r"//[^\n]*", "", text)
    parts = re.split(r"\n(fp8_\w+_kernel)\(", text)
    return dict(zip(parts[1::2], parts[2::2]))


@pytest.mark.parametrize("name", ["fp8_wide_kernel", "fp8_group_kernel", "fp8_pairs_kernel", "fp8_down_kernel"])
def test_a_warp_meets_before_what_all_of_it_does(name):
    body = _kernels()[name].split("\n__global__")[0]
    waiting, loads = False, 0
    for token in TOKEN.findall(body):
        if token.startswith("wait_bar"):
            waiting = True
        elif token.startswith("__syncwarp"):
            waiting = False
        else:
            loads += 1
            assert not waiting, f"{name}: {token} right behind a poll"
    assert loads
