"""What the training operators refuse because a kernel behind a pointer would drop it without a word: tangents of forward-mode
differentiation and the recording of a call by a tracer.  No GPU: the refusal comes before any look at the device."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from boa_amd import ops

# every call, its floating inputs by name
N, L, C = 2, 5, 6
SCAN = dict(u=(N, L, C), delta=(N, L, C), A=(C, 16), B=(N, L, 16), C=(N, L, 16), D=(C,), z=(N, L, C), delta_bias=(C,))
STEP = {k: (s[0], s[2]) if len(s) == 3 else s for k, s in SCAN.items()}
CALLS = {
    "layer_norm": (ops.layer_norm, dict(x=(N, C), weight=(C,), bias=(C,)), {}),
    "cross_entropy": (ops.cross_entropy, dict(logits=(N, C)), dict(targets=torch.zeros(N, dtype=torch.int64))),
    "causal_conv": (ops.causal_conv, dict(x=(N, L, C), weight=(C, 1, 4), bias=(C,), state=(N, 3, C)), {}),
    "causal_conv_step": (ops.causal_conv_step, dict(x=(N, C), weight=(C, 1, 4), bias=(C,), state=(N, 3, C)), {}),
    "selective_scan": (ops.selective_scan, dict(SCAN, state=(N, 16, C)), {}),
    "selective_scan_step": (ops.selective_scan_step, dict(STEP, state=(N, 16, C)), {}),
}
INPUTS = [(call, name) for call, (_, shapes, _) in CALLS.items() for name in shapes]


def _args(call):
    f, shapes, rest = CALLS[call]
    return f, {k: torch.zeros(s) for k, s in shapes.items()}, rest


@pytest.mark.parametrize("call,name", INPUTS)
@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused(call, name, no_grad):
    f, args, rest = _args(call)
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(**args, **rest)
        with torch.inference_mode(), pytest.raises(ValueError, match="on the GPU"):  # where torch drops tangents itself
            f(**args, **rest)


@pytest.mark.parametrize("call", CALLS)
def test_inputs_without_tangents_pass_in_a_dual_level(call):
    f, args, rest = _args(call)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="on the GPU"):
        f(**args, **rest)


@pytest.mark.parametrize("call", CALLS)
def test_tracers_are_refused(call):
    f, args, rest = _args(call)
    names = list(args)
    g = lambda *ts: f(**dict(zip(names, ts)), **rest)  # noqa: E731
    for trace in (lambda: torch.jit.trace(g, tuple(args.values())), lambda: make_fx(g)(*args.values())):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            trace()
    with pytest.raises(ValueError, match="on the GPU"):
        g(*args.values())


@pytest.mark.parametrize("cls,args", [
    (ops._LayerNorm, lambda x: (x, None, None, 1e-5)), (ops._CrossEntropy, lambda x: (x, None, -100, "mean", True)),
    (ops._CausalConv, lambda x: (x, x, None, True, None, None, False)), (ops._SelectiveScan, lambda x: (x,) * 8 + (None, None, False))])
def test_a_tangent_of_the_upstream_gradient_is_refused(monkeypatch, cls, args):
    """Forward over reverse: the gradient's own derivative would be lost.  The forward kernels are left out here."""
    x = torch.zeros(N, L, C, requires_grad=True)
    y = torch.zeros(N, L, C)
    scalar = cls is ops._CrossEntropy

    def forward(ctx, *a):
        return y.sum() if scalar else y.clone()

    monkeypatch.setattr(cls, "forward", staticmethod(forward))
    if cls in (ops._CausalConv, ops._SelectiveScan):
        monkeypatch.setattr(cls, "forward", staticmethod(lambda ctx, *a: (y.clone(), None)))
    out = cls.apply(*args(x))
    out = out[0] if isinstance(out, tuple) else out
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, x, dy)
