"""Upstream gradients that autograd hands to the training operators without memory of their own, or negated for the reader."""
import pytest
import torch

from test_gpu_ops import _gen, _randn, _scan_inputs

pytestmark = pytest.mark.gpu


def test_zeros_without_memory_and_negations(gpu):
    from boa_amd import ops

    g = _gen(1)
    s = {k: v.detach().requires_grad_() for k, v in _scan_inputs(g, 2, 30, 1, torch.float32).items()}
    x, w, b = (_randn(g, *shape).requires_grad_() for shape in ((2, 30, 1), (1, 4), (1,)))
    logits = _randn(g, 6, 9).requires_grad_()
    t = torch.tensor([0, 8, 3, 3, 1, 2], device="cuda")
    for call, leaves in ((lambda: ops.layer_norm(x, None, b), (x, b)), (lambda: ops.causal_conv(x, w, b), (x, w, b)),
                         (lambda: ops.selective_scan(**s), tuple(s.values())),
                         (lambda: ops.cross_entropy(logits, t, reduction="none"), (logits,))):
        y = call()
        zeros = torch.autograd.grad(torch.sgn(y).sum(), leaves)  # sgn's gradient is zero
        assert all(v.shape == leaf.shape and not v.any() for v, leaf in zip(zeros, leaves))
        up = torch.randn(y.shape, device="cuda", generator=g)
        want = torch.autograd.grad(call(), leaves, -up)
        got = torch.autograd.grad(call(), leaves, torch._neg_view(up))
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and any(v.any() for v in want)
