"""Registers of the training operators' kernels in the built library (no GPU): none keeps vector registers in scratch memory."""
import os

import pytest

from boa_amd import build
from test_kernel_resources import _kernels


@pytest.mark.parametrize("name", ["10k_norm_fwdI", "10k_norm_bwdI", "10k_loss_fwdI", "10k_loss_bwdI", "10k_conv_fwdI", "10k_conv_bwdI",
                                  "11k_conv_stepI", "10k_scan_fwdI", "16k_scan_bwd_localI", "10k_scan_bwdI", "11k_scan_sumsI",
                                  "11k_scan_stepI"])
def test_operators_do_not_spill(name):
    assert os.path.exists(build.OUT), "build first"
    found = {k: v for k, v in _kernels().items() if name in k}
    assert found, name
    bad = {k: (v[".vgpr_spill_count"], v[".private_segment_fixed_size"]) for k, v in found.items()
           if v[".vgpr_spill_count"] or v[".private_segment_fixed_size"]}
    assert not bad, bad


def test_the_scans_backward_kernel_leaves_room_for_four_workgroups():
    """128 vector registers per lane: four wavefronts on each SIMD."""
    found = [v[".vgpr_count"] for k, v in _kernels().items() if "10k_scan_bwdI" in k]
    assert len(found) == 6 and max(found) <= 128


def test_the_kernel_that_joins_the_scans_chunks_does_not_spill():
    """It holds the ends of 32 chunks and their sums of steps, 64 values per lane."""
    found = {k: v for k, v in _kernels().items() if "11k_scan_joinI" in k}
    assert len(found) == 2
    assert not any(v[".vgpr_spill_count"] or v[".private_segment_fixed_size"] for v in found.values())


def test_no_kernel_of_the_operators_is_left_out():
    """All that norm_op, loss_op, conv_op and scan_op launch are looked at here (k_loss_sum and k_sum_parts are no templates)."""
    import re

    names = set()
    for f in ("norm_op", "loss_op", "conv_op", "scan_op"):
        src = open(os.path.join(build.CSRC, f + ".hip")).read()
        names |= set(re.findall(r"__global__ void (?:__launch_bounds__\((?:[^()]|\([^()]*\))*\) )?(k_\w+)\(", src))
    assert {"k_scan_join", "k_scan_fwd", "k_conv_step", "k_loss_sum", "k_sum_parts", "k_norm_bwd"} <= names
    for name in names:
        found = {k: v for k, v in _kernels().items() if f"{len(name)}{name}" in k}
        assert found, name
        assert not any(v[".vgpr_spill_count"] or v[".private_segment_fixed_size"] for v in found.values()), name
