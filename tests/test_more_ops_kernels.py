"""Registers of the kernels of linear attention, gradient clipping and sampling in the built library (no GPU): none keeps any in scratch
memory, and those of up to 64 keys leave room for a second workgroup on each CU."""
import os
import re

import pytest

from boa_amd import build
from test_kernel_resources import _kernels


def _launched(name):
    src = open(os.path.join(build.CSRC, name + ".hip")).read()
    return set(re.findall(r"__global__ void (?:__launch_bounds__\((?:[^()]|\([^()]*\))*\) )?(k_\w+)\(", src))


@pytest.mark.parametrize("source,some", [("attn_op", {"k_attn_fwd", "k_attn_bwd", "k_attn_states", "k_attn_join", "k_attn_step"}),
                                         ("grad_op", {"k_grad_part", "k_grad_scale", "k_grad_norm"}), ("sample_op", {"k_sample"})])
def test_no_kernel_spills(source, some):
    names = _launched(source)
    assert some <= names
    for name in names:
        found = {k: v for k, v in _kernels().items() if f"{len(name)}{name}" in k}
        assert found, name
        bad = {k: (v[".vgpr_spill_count"], v[".private_segment_fixed_size"]) for k, v in found.items()
               if v[".vgpr_spill_count"] or v[".private_segment_fixed_size"]}
        assert not bad, bad


def test_two_workgroups_of_attention_share_a_cu():
    """256 vector registers per lane, accumulation registers among them: two wavefronts on each SIMD."""
    found = {k: v[".vgpr_count"] for k, v in _kernels().items() if re.search(r"k_attn_(fwd|bwd|states)ILi\dELi64E", k)}
    assert len(found) == 3 * (2 + 4 + 4) and max(found.values()) <= 256, found
