"""Which kernel an FP8 product takes (csrc/qkm_fp8_choice.h), asked on the host."""
import os

import pytest

import fp8_choice as choice


def test_experts_by_their_mean():
    """The mean is not rounded, and the bound itself counts."""
    assert choice.pairs_as_lanes(False, 1184, 8, 256) and not choice.pairs_as_lanes(False, 1183, 8, 256)
    assert choice.pairs_as_lanes(True, 1856, 8, 256) and not choice.pairs_as_lanes(True, 1855, 8, 256)
    assert not choice.pairs_as_lanes(False, 1, 16, 16) and choice.pairs_as_lanes(True, (1 << 27) - 1, 16, 16)


def test_a_shard_goes_by_the_whole_table():
    """Its list has its own experts' pairs alone: 192 tokens of top 8 are 6 pairs an expert of 256, whatever part of them is resident."""
    assert "a.n_table = c->cfg.dims.n_expert;" in open(os.path.join(choice.CSRC, "qkm_api.cu")).read()
    assert "fp8_pairs_as_lanes(MODE == kFp8Down, a.n, a.n_used, a.n_table)" in open(os.path.join(choice.CSRC, "qkm_fp8_gemm.cu")).read()


# (hidden, inner) -> measured us of rows: few rows, lanes; of gate/up and of down
MEASURED = {(1024, 256): ({64: (4.0, 10.3), 256: (4.2, 11.0), 512: (7.1, 11.1)}, {64: (3.0, 10.2), 256: (7.5, 13.2), 400: (10.7, 13.2)}),
            (2048, 512): ({64: (6.1, 15.1), 200: (9.6, 15.9), 320: (13.9, 16.0), 512: (19.0, 16.2)}, {64: (4.8, 13.1), 200: (11.5, 15.4), 320: (16.9, 15.5), 512: (25.9, 15.6)}),
            (2048, 1024): ({64: (6.3, 15.3), 150: (13.3, 16.1), 256: (19.1, 16.2), 512: (33.9, 16.6)}, {64: (5.7, 10.5), 150: (11.2, 12.5), 256: (16.7, 12.5)}),
            (4096, 1536): ({32: (10.1, 24.7), 64: (16.4, 25.1), 150: (29.9, 26.3), 512: (82.1, 26.7)}, {32: (6.7, 12.4), 64: (11.8, 13.0), 100: (17.6, 14.2), 256: (38.2, 14.8)}),
            (5120, 2560): ({32: (20.4, 29.5), 100: (39.5, 30.7), 256: (88.1, 31.7)}, {32: (14.8, 17.1), 64: (26.8, 17.8), 200: (78.6, 19.7)})}


@pytest.mark.parametrize("D,F", MEASURED)
def test_shared_expert_takes_the_kernel_that_was_faster(D, F):
    gateup, down = MEASURED[D, F]
    for n, (few, lanes) in gateup.items():
        assert choice.shared_few_rows(False, n, F, D) == (few < lanes), n
    for n, (few, lanes) in down.items():
        assert choice.shared_few_rows(True, n, D, F) == (few < lanes), n
