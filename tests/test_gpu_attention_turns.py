"""Linear attention's gradient where one workgroup takes the heads of a group in turn (from 1024 workgroups on), and what is not finite
there: bounds of test_gpu_attention.py."""
import math

import pytest
import torch

from boa_amd import ops
from test_gpu_attention import BF, F16, F32, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,decay,dtype", [
    ((600, 65, 4, 1, 9, 9), "token", F32), ((600, 65, 4, 1, 9, 9), "head", BF), ((300, 65, 6, 2, 16, 8), "token", BF),
    ((300, 65, 6, 2, 16, 8), "token", F16), ((130, 130, 8, 2, 64, 70), "token", BF), ((520, 65, 4, 1, 80, 5), "head", F32),
    ((520, 65, 4, 1, 80, 5), "token", BF),
])
def test_heads_in_turn(gpu, size, decay, dtype):
    _check(*size, dtype, decay, ragged=True, state=True, seed=1)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("value", [8, 70])
def test_what_is_not_a_number_stays_in_its_head_and_sequence(gpu, value, bad, dtype):
    n, length, heads, at = 520, 70, 4, 37
    x, dy, _, _ = _inputs(n, length, heads, 1, 12, value, dtype, "token", 2)
    leaves = [t.cuda().requires_grad_() for t in x.values()]
    dy = dy.cuda()
    want = torch.autograd.grad(ops.linear_attention(*leaves), leaves, dy)
    for column in (3, value - 1):
        wrong = dy.clone()
        wrong[5, at, 1, column] = bad
        dq, dk, dv, dg = torch.autograd.grad(ops.linear_attention(*leaves), leaves, wrong)
        others = [i for i in range(n) if i != 5]
        for got, w in zip((dq, dk, dv, dg), want):
            assert torch.equal(got[others], w[others])
        heads_of = [0, 2, 3]
        columns = [c for c in range(value) if c != column]
        assert torch.equal(dv[5][:, heads_of], want[2][5][:, heads_of]) and torch.equal(dv[5][..., columns], want[2][5][..., columns])
        assert torch.equal(dg[5][:, heads_of], want[3][5][:, heads_of])
        assert torch.equal(dq[5, at + 1:], want[0][5, at + 1:]) and torch.equal(dk[5, at + 1:], want[1][5, at + 1:])
        assert not torch.isfinite(dv[5, :at + 1, 1, column]).any()
        wrong = x["v"].cuda()
        wrong[5, at, 1, column] = bad
        y = ops.linear_attention(leaves[0].detach(), leaves[1].detach(), wrong, leaves[3].detach())
        clean = ops.linear_attention(*(t.detach() for t in leaves))
        assert torch.equal(y[others], clean[others]) and torch.equal(y[5][..., columns], clean[5][..., columns])
        assert torch.equal(y[5][:, heads_of], clean[5][:, heads_of]) and torch.equal(y[5, :at], clean[5, :at])
        assert not torch.isfinite(y[5, at:, 1, column]).any()
