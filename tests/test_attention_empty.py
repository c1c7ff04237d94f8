"""Calls of linear attention that have no position: a decay for each position is an empty tensor then, whose address is null."""
import ctypes

import pytest
import torch

from boa_amd import _native, ops
from test_more_ops_args import _packed


@pytest.mark.parametrize("n,length", [(0, 5), (0, 0), (2, 0)])
def test_c_calls_need_no_pointers(n, length):
    """Those that launch nothing, and so run without a GPU."""
    lib = _native.load_cdll()
    null = _packed(n=n, length=length, p=0, decay=0, ddecay=0, marks=0)
    assert lib.boa_linear_attention_bwd(null, None, 0, None) == _native.BOA_OK
    if n == 0:
        assert lib.boa_linear_attention_fwd(null, None, 0, None) == _native.BOA_OK
    # the gradient of a head's decay is written all the same
    per_head = bytearray(null)
    per_head[20:24] = ctypes.c_int32(1)
    assert lib.boa_linear_attention_bwd(bytes(per_head), None, 0, None) == _native.BOA_ERR_ARG
    for bad in (_packed(decay=0), _packed(ddecay=0)):
        assert lib.boa_linear_attention_bwd(bad, ctypes.c_void_p(16), 1 << 62, None) == _native.BOA_ERR_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("n,length", [(2, 0), (0, 5), (0, 0)])
def test_forward_state_and_gradient(gpu, n, length, per_head, dtype):
    def x(*shape, dtype=dtype):
        return torch.randn(shape, device="cuda").to(dtype).requires_grad_()

    leaves = [x(n, length, 1, 5), x(n, length, 1, 5), x(n, length, 3, 6), x(*((3,) if per_head else (n, length, 3)), dtype=torch.float32)]
    s = torch.randn(n, 3, 5, 6, device="cuda")
    for state in (s, None):
        for lens in (None, torch.zeros(n, dtype=torch.int32, device="cuda")):
            y, last = ops.linear_attention(*leaves, state=state, lens=lens, return_state=True)
            assert y.shape == (n, length, 3, 6) and y.dtype == dtype
            assert torch.equal(last, torch.zeros_like(s) if state is None else s) and (n == 0 or last.data_ptr() != s.data_ptr())
            grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
            assert [g.shape for g in grads] == [t.shape for t in leaves] and not any(g.any() for g in grads)
