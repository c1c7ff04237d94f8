"""Scalar registers that a kernel keeps in vector lanes, which cost a vector instruction for each use (no GPU): none in the kernels of
linear attention that walk or join states or advance them by a token, in clipping's, and in sampling's of up to 256 symbols."""
import pytest

from test_kernel_resources import _kernels


@pytest.mark.parametrize("kernel", ["k_attn_states", "k_attn_join", "k_attn_step", "k_attn_sum", "k_grad_part", "k_grad_scale", "k_grad_norm",
                                    "k_sampleILi0ELi4ELi1ELi1E", "k_sampleILi1ELi4ELi1ELi1E", "k_sampleILi2ELi4ELi1ELi1E"])
def test_no_scalars_in_lanes(kernel):
    found = {k: v[".sgpr_spill_count"] for k, v in _kernels().items() if kernel in k}
    assert found and not any(found.values()), found
