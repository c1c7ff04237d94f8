"""The training operators and the model's loss called from a function that torch.compile has taken (its graphs run as they are, backend
"eager"): a kernel behind a pointer cannot be part of such a graph, so the call has to break it and run, with the eager bits."""
import pytest
import torch

from test_gpu_ops import _gen, _randn, _scan_inputs
from test_gpu_train import _model

pytestmark = pytest.mark.gpu


def _cases(g):
    from boa_amd import ops

    n, length, c = 2, 40, 70
    s = _scan_inputs(g, n, length, c, torch.float32)
    t = torch.randint(0, 64, (6,), generator=g, device="cuda")
    yield lambda x, w, b: ops.layer_norm(x * 2, w, b) + 1, (_randn(g, 6, 64), _randn(g, 64), _randn(g, 64))
    yield lambda x: ops.cross_entropy(x * 2, t) * 3, (_randn(g, 6, 64),)
    yield lambda x, w, b: ops.causal_conv(x * 2, w, b) + 1, (_randn(g, n, length, c), _randn(g, c, 4), _randn(g, c))
    yield lambda *a: ops.selective_scan(a[0] * 2, *a[1:]) + 1, tuple(s.values())


def test_operators_in_compiled_functions(gpu):
    for f, leaves in _cases(_gen(1)):
        torch._dynamo.reset()
        leaves = [v.detach().requires_grad_() for v in leaves]
        want = f(*leaves)
        dy = torch.ones_like(want)
        wants = [want.detach(), *torch.autograd.grad(want, leaves, dy)]
        h = torch.compile(f, backend="eager")
        for _ in range(3):
            got = h(*leaves)
            gots = [got.detach(), *torch.autograd.grad(got, leaves, dy)]
            assert all(torch.equal(p, q) for p, q in zip(wants, gots))
        with torch.no_grad():
            assert torch.equal(h(*leaves), wants[0])
    torch._dynamo.reset()


def test_a_compiled_loss(gpu):
    m, _ = _model(1)
    x = torch.randint(0, 256, (2, 50), generator=_gen(2), device="cuda")
    params = list(m.parameters())
    want = m.loss(x)
    grads = torch.autograd.grad(want, params)
    torch._dynamo.reset()
    h = torch.compile(lambda x: m.loss(x), backend="eager")
    for _ in range(2):
        got = h(x)
        assert torch.equal(got, want) and all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(got, params), grads))
    torch._dynamo.reset()
