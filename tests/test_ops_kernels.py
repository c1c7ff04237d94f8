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
