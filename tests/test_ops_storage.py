"""Tensors that the training operators cannot read by their address (no GPU: the kernels' launch is stood in for)."""
import types

import pytest
import torch

from boa_amd import ops
from test_ops_tracers import CALLS, C, L, N


class Wrapper(torch.Tensor):
    """Stands for another tensor, as sharded and quantised ones do; has no memory."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device, strides=t.stride())

    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        raise NotImplementedError


@pytest.fixture
def launched(monkeypatch):
    calls = []
    lib = types.SimpleNamespace(**{f"boa_{k}": k for k in ("layer_norm_fwd", "causal_conv_fwd", "causal_conv_step", "selective_scan_fwd",
                                                           "selective_scan_step")}, boa_selective_scan_work_bytes=lambda *a: 0)
    monkeypatch.setattr(ops, "_gpu", lambda *a: None)
    monkeypatch.setattr(ops._nat, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_call", lambda *a: calls.append(a))
    return calls


@pytest.mark.parametrize("call,name", [
    ("layer_norm", "weight"), ("layer_norm", "bias"), ("causal_conv", "bias"), ("causal_conv", "state"), ("causal_conv_step", "bias"),
    ("selective_scan", "D"), ("selective_scan", "z"), ("selective_scan", "delta_bias"), ("selective_scan", "state"),
    ("selective_scan_step", "D"), ("selective_scan_step", "z"), ("selective_scan_step", "delta_bias"),
    ("causal_conv", "lens"), ("selective_scan", "lens")])
def test_an_optional_input_without_memory_is_not_taken_for_none(launched, call, name):
    f, shapes, rest = CALLS[call]
    args = {k: torch.zeros(s) for k, s in shapes.items()}
    with torch.no_grad():
        f(**args, **rest)
    assert len(launched) == 1
    args[name] = Wrapper(torch.full((N,), L, dtype=torch.int32) if name == "lens" else args[name])
    with torch.no_grad(), pytest.raises(ValueError, match="Wrapper of shape .* without memory"):
        f(**args, **rest)
    assert len(launched) == 1


def test_empty_tensors_have_no_address_and_pass(launched):
    assert ops._ptr(torch.empty(0, C)) == 0
    ops.causal_conv(torch.zeros(0, L, C), torch.zeros(C, 4), state=torch.zeros(0, 3, C), lens=torch.zeros(0, dtype=torch.int32))
    assert len(launched) == 1


def test_upstream_gradients_that_are_not_in_memory():
    """Zeros that autograd hands on without memory (of sgn), and a negation that is left to the reader (of a conjugate's imaginary part,
    with one channel, so that nothing copies it)."""
    got = []

    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, dy):
            before = dy
            dy = ops._once("op", dy)
            got.append((before.data_ptr(), before.is_neg(), dy))
            return dy.clone()

    x = torch.randn(N, L, 1, requires_grad=True)
    torch.sgn(Op.apply(x)).sum().backward()
    address, _, dy = got.pop()
    assert not address and dy.data_ptr() and not dy._is_zerotensor() and not dy.any() and dy.shape == x.shape
    up = torch._neg_view(torch.ones(N, L, 1))
    Op.apply(x).backward(up)
    _, neg, dy = got.pop()
    assert neg and not dy.is_neg() and torch.equal(dy, -torch.ones(N, L, 1))
