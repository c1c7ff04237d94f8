"""Linear attention where a row's last access of 16 bytes would pass its end, and rows at every element's address: against 64 bits under
the bounds of test_gpu_attention.py, and bit for bit against aligned rows with nothing beside them."""
import pytest
import torch

from boa_amd import ops
from test_gpu_attention import BF, F16, F32, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("key", [*range(1, 18), 63, 65, 66, 127])
def test_every_end_of_a_row(gpu, key, dtype):
    _check(2, 70, 2, 1, key, 61 + key % 13, dtype, "token", ragged=True, state=True, seed=key)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("key,value", [(64, 64), (9, 71), (2, 3), (24, 72), (128, 5)])
@pytest.mark.parametrize("before", [0, 1, 2, 3, 5])
def test_rows_beside_what_is_no_number(gpu, before, key, value, dtype):
    """Each row is a part of one that holds NaN around it; the state stands at any float32's address."""
    n, length, heads, groups = 2, 100, 4, 2
    x, dy, _, s = _inputs(n, length, heads, groups, key, value, dtype, "token", seed=before, state=True)
    x, dy, s = {k: t.cuda() for k, t in x.items()}, dy.cuda(), s.cuda()

    def beside(t):
        out = torch.full((*t.shape[:-1], t.shape[-1] + before + 1), float("nan"), dtype=t.dtype, device="cuda")
        out = out[..., before:before + t.shape[-1]]
        return out.copy_(t)

    def run(q, k, v, g, dy, s):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, g)]
        y, last = ops.linear_attention(*leaves, state=s, return_state=True)
        return [y.detach(), last, *torch.autograd.grad(y, leaves, dy)]

    want = run(*x.values(), dy, s)
    q, k, v, g = x.values()
    got = run(beside(q), beside(k), beside(v), g, beside(dy), s)
    for a, b in zip(want, got):
        assert torch.equal(a, b)

    state = s.clone()
    want = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state=state)
    buf = torch.full((s.numel() + 16,), float("nan"), device="cuda")
    at = buf[before:before + s.numel()].view(s.shape).copy_(s)
    got = ops.linear_attention_step(beside(q)[:, 0], beside(k)[:, 0], beside(v)[:, 0], g[:, 0], state=at)
    assert torch.equal(got, want) and torch.equal(at, state)
    assert buf[:before].isnan().all() and buf[before + s.numel():].isnan().all()


@pytest.mark.parametrize("value", [1, 2, 3, 5, 63, 65, 66, 67, 130])
def test_single_tokens_of_every_width(gpu, value):
    n, heads, groups, key = 3, 4, 2, 20
    x, _, _, s = _inputs(n, 1, heads, groups, key, value, F32, "token", seed=value, state=True)
    want_s = s.double() * x["log_decay"][:, 0, :, None, None].double().exp()
    k, q = (x[name][:, 0].double().repeat_interleave(heads // groups, 1) for name in "kq")
    add = k[..., None] * x["v"][:, 0].double()[:, :, None]
    size = s.double().abs() + add.abs()  # the decay is at most 1
    want_s = want_s + add
    got_s = s.cuda()
    got = ops.linear_attention_step(*(t[:, 0].cuda() for t in x.values()), state=got_s).cpu().double()
    # a state: the power (its exponent below 1: two roundings), the product, the sum; y: its terms' products, their sum over 20
    # keys, the scale
    assert ((got_s.cpu().double() - want_s).abs() <= 6 * 2.0 ** -24 * size).all()
    terms = (q.abs()[..., None] * size).sum(-2) * key ** -0.5
    want = (q[..., None] * want_s).sum(-2) * key ** -0.5
    assert ((got - want).abs() <= (6 + key + 3) * 2.0 ** -24 * terms).all()
