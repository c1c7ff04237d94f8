"""The 64-bit formulas that the operators are checked against: their gradients against torch's autograd and against
differences, on the CPU."""
import torch
import torch.nn.functional as F

import ops_ref as R

T = torch.float64


def _r(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + 7 * len(shape) + sum(shape)), dtype=T) * scale


def _same(a, b):
    assert torch.allclose(a, b, rtol=1e-9, atol=1e-11), float((a - b).abs().max())


def test_norm():
    x, w, b, dy = _r(5, 9).requires_grad_(), _r(9).requires_grad_(), _r(9, seed=3).requires_grad_(), _r(5, 9, seed=4)
    y = F.layer_norm(x, (9,), w, b)
    g = torch.autograd.grad(y, (x, w, b), dy)
    ref = R.norm(x, w, b, dy)
    for k, v in zip(("y", "dx", "dw", "db"), (y, *g)):
        _same(ref[k][0], v.detach())
        assert (ref[k][1] >= ref[k][0].abs() - 1e-12).all()


def test_loss():
    x, t = _r(6, 11).requires_grad_(), torch.tensor([0, 3, -100, 10, 5, 5])
    for reduction in ("mean", "sum"):
        y = F.cross_entropy(x, t, reduction=reduction, ignore_index=-100)
        ref = R.loss(x, t, -100, reduction, 2.5)
        _same(ref["y"][0], y.detach())
        _same(ref["dx"][0], torch.autograd.grad(y, x, torch.tensor(2.5, dtype=T))[0])
    y = F.cross_entropy(x, t, reduction="none", ignore_index=-100)
    up = _r(6)
    ref = R.loss(x, t, -100, "none", up)
    _same(ref["y"][0], y.detach())
    _same(ref["dx"][0], torch.autograd.grad(y, x, up)[0])


def test_conv():
    x, w, b, st, dy = (_r(2, 7, 3).requires_grad_(), _r(3, 1, 4).requires_grad_(), _r(3).requires_grad_(), _r(2, 3, 3, seed=1),
                       _r(2, 7, 3, seed=2))
    for silu in (True, False):
        y = F.conv1d(torch.cat([st, x], 1).transpose(1, 2), w, b, groups=3).transpose(1, 2)
        y = F.silu(y) if silu else y
        g = torch.autograd.grad(y, (x, w, b), dy)
        ref = R.conv(x, w, b, silu, st, None, dy)
        _same(ref["y"][0], y.detach())
        for k, v in zip(("dx", "dw", "db"), g):
            _same(ref[k][0].reshape(v.shape), v)
        _same(ref["state"][0], x.detach()[:, -3:])


def _scan_torch(u, delta, A, B, C, D, z, bias, h, ends):
    ys = []
    dt = F.softplus(delta + bias)
    for t in range(u.shape[1]):
        new = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * B[:, t, None]
        live = (t < ends)[:, None]
        h = torch.where(live[..., None], new, h)
        ys.append(torch.where(live, ((h * C[:, t, None]).sum(2) + D * u[:, t]) * F.silu(z[:, t]), torch.zeros_like(u[:, t])))
    return torch.stack(ys, 1), h


def test_scan():
    n, length, c = 3, 6, 4
    leaves = [_r(n, length, c), _r(n, length, c, seed=1), -torch.exp(_r(c, 16)), _r(n, length, 16, seed=2), _r(n, length, 16, seed=3),
              _r(c), _r(n, length, c, seed=4), _r(c, seed=5)]
    for v in leaves:
        v.requires_grad_()
    h0, lens, dy = _r(n, 16, c), torch.tensor([6, 0, 4]), _r(n, length, c, seed=6)
    y, h = _scan_torch(*leaves, h0.transpose(1, 2), lens)
    g = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    ref = R.scan(*leaves, h0, lens, dy)
    _same(ref["y"][0], y.detach())
    _same(ref["state"][0], h.detach().transpose(1, 2))
    for k, v in zip(("du", "ddelta", "dA", "dB", "dC", "dD", "dz", "dbias"), g):
        _same(ref[k][0], v)
        assert (ref[k][1] >= ref[k][0].abs() - 1e-12).all()
    # and against differences: a central step of 1e-6 is off by about 1e-9 of the values
    for leaf, k in ((leaves[2], "dA"), (leaves[3], "dB"), (leaves[1], "ddelta")):
        step = _r(*leaf.shape, seed=9)
        moved = [[v if v is not leaf else (v + s * 1e-6 * step) for v in leaves] for s in (1, -1)]
        hi, lo = ((R.scan(*m, h0, lens)["y"][0] * dy).sum() for m in moved)
        assert abs((hi - lo) / 2e-6 - (ref[k][0] * step).sum()) < 1e-6 * ref[k][1].sum()
