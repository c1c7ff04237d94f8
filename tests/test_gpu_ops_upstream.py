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


def test_one_channel_of_conjugates(gpu):
    """Imaginary parts of conjugates are negated where they are read; with one channel their rows count as contiguous."""
    from boa_amd import ops

    g = _gen(2)

    def imag(*shape):
        v = torch.complex(_randn(g, *shape), _randn(g, *shape)).conj().imag
        assert v.is_neg()
        return v

    x, w, b = imag(2, 30)[..., None], _randn(g, 1, 4), imag(1)
    state, up = _randn(g, 2, 3, 1), _randn(g, 2, 30, 1)
    s = {**_scan_inputs(g, 2, 30, 1, torch.float32), "u": x, "delta": imag(2, 30)[..., None], "z": imag(2, 30)[..., None], "D": b,
         "delta_bias": imag(1)}
    assert x.is_neg() and ops._rows(x) is x
    written = lambda t: t.resolve_neg().clone()  # noqa: E731

    def passes(f):
        x1, b1, s1 = f(x).requires_grad_(), f(b).requires_grad_(), {k: f(v).requires_grad_() for k, v in s.items()}
        y = ops.causal_conv(x1, w, b1)
        z = ops.selective_scan(**s1)
        n = ops.layer_norm(x1, None, b1)
        out = [y, z, n, *torch.autograd.grad(y, (x1, b1), up), *torch.autograd.grad(z, tuple(s1.values()), up),
               *torch.autograd.grad(n, (b1,), up)]
        with torch.no_grad():
            st, h = state.clone(), torch.zeros(2, 16, 1, device="cuda")
            at = {k: v[:, 0] if k in ("u", "delta", "B", "C", "z") else v for k, v in s1.items()}
            out += [ops.causal_conv_step(x1[:, 0], st, w, b1), st, ops.selective_scan_step(**at, state=h), h]
        return out

    assert all(torch.equal(p, q) for p, q in zip(passes(lambda t: t.detach()), passes(lambda t: written(t.detach()))))
