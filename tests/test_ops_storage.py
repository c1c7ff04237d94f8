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
