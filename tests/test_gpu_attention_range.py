"""Linear attention at the ends of float32's range: what is finite in the definition's own order of operations comes out finite."""
import pytest
import torch

from boa_amd import ops
from test_gpu_attention import BF, F16, F32
from test_gpu_attention_bits import WAYS, _run

pytestmark = pytest.mark.gpu

TOP = torch.finfo(F32).max
NEAR = 255.75 * 2.0 ** 120  # finite, and nearer to 2^128 than to the largest bfloat16


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("large", [TOP, -TOP, NEAR, 3.4e38, 3.39e38])
def test_states_near_the_largest_number(gpu, large, way, dtype):
    n, heads, key, value = way
    forward, _ = _run(*way, dtype, 2, q={0: (2.0 ** -10,), 1: (0.0, -2.0 ** -10)})
    state = torch.zeros(n, heads, key, value, device="cuda")
    state[:, :, 0] = state[:, :, 1] = large
    want = (torch.tensor(large) * 2.0 ** -10).to(dtype).item()
    y = forward(state)
    assert (y[:, 0] == want).all() and (y[:, 1] == -want).all()


BIG = (255.0 * 2.0 ** 60, 0.75 * 2.0 ** 60)  # times 2^60, summed: NEAR
ONE = (2.0 ** 60, 2.0 ** 60)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("way", WAYS)
def test_scores_near_the_largest_number(gpu, way, dtype):
    small = 2.0 ** -20
    want = torch.tensor(NEAR * small).to(dtype).item()
    forward, _ = _run(*way, dtype, 2, q={1: ONE}, k={0: BIG}, v={0: (small,)})
    y = forward()
    assert (y[:, 1, 0, 0] == want).all() and not y[:, 0].any() and not y[..., 1:].any()
    for which, at, rows in (("v", 0, dict(q={1: ONE}, k={0: BIG}, dy={1: (small,)})), ("q", 1, dict(v={0: BIG}, dy={1: ONE}, k={0: (small,)})),
                            ("k", 0, dict(v={0: BIG}, dy={1: ONE}, q={1: (small,)}))):
        _, grads = _run(*way, dtype, 2, **rows)
        got = grads()[which]
        assert (got[:, at, 0, 0] == want).all() and torch.isfinite(got).all(), which


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("way", WAYS)
def test_states_gradients_near_the_largest_number(gpu, way, dtype):
    small = 2.0 ** -20
    want = torch.tensor(NEAR * small).to(dtype).item()
    q, dy = {64: BIG[:1], 65: BIG[1:]}, {64: ONE[:1], 65: ONE[:1]}
    _, grads = _run(*way, dtype, 70, q=q, dy=dy, k={t: (small,) for t in range(64)})
    dv = grads()["v"]
    assert (dv[:, :64, 0, 0] == want).all() and not dv[..., 1:].any()
    _, grads = _run(*way, dtype, 70, q=q, dy=dy, v={t: (small,) for t in range(64)})
    dk = grads()["k"]
    assert (dk[:, :64, 0, 0] == want).all() and not dk[..., 1:].any()
    # and of states before a chunk, in the gradient of q
    _, grads = _run(*way, dtype, 70, k=q, v=dy, dy={t: (small,) for t in range(66, 70)})
    dq = grads()["q"]
    assert (dq[:, 66:70, 0, 0] == want).all() and not dq[..., 1:].any()


# One head by itself and heads in turn, one and several tiles of keys and values, many pieces and one of the length.
SHAPES = [(1, 70, 1, 5, 6), (2, 200, 2, 100, 70), (1100, 70, 4, 5, 6)]


def _ordinary(n, length, heads, key, value, dtype):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()  # noqa: E731
    return dict(q=r(n, length, 1, key), k=r(n, length, 1, key), v=r(n, length, heads, value), log_decay=-torch.rand(n, length, heads, generator=g).cuda())


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_large_state_that_is_forgotten(gpu, shape, dtype):
    """Behind a decay to nothing a state of any size is as none: in y, and in the gradients of q and of the decay."""
    n, length, heads, key, value = shape
    x = _ordinary(*shape, dtype)
    x["log_decay"][:, 0] = -float("inf")
    x["q"][:, 0] = 200.0  # 200 times such a state is infinite
    leaves = [t.requires_grad_() for t in x.values()]
    dy = torch.full((n, length, heads, value), 100.0, dtype=dtype, device="cuda")
    state = torch.full((n, heads, key, value), 3e38, device="cuda")
    state[:, :, ::2] *= -1.0

    def run(state):
        y, last = ops.linear_attention(**x, state=state, return_state=True)
        return [y.detach(), last, *torch.autograd.grad(y, leaves, dy)]

    # in float16 the right results can be infinite: dk of position 0 is 200 / sqrt(5) times the sum over the heads of dy . v, which is
    # 100 times a sum of 24 normal numbers
    for got, want in zip(run(state), run(None)):
        assert not torch.isnan(want).any() and (dtype is F16 or torch.isfinite(want).all()) and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_large_gradient_of_a_state_that_is_forgotten(gpu, shape, dtype):
    """Positions before a decay to nothing have no gradient from behind it, however large that is."""
    n, length, heads, key, value = shape
    x = _ordinary(*shape, dtype)
    big = 2.0 ** (15 if dtype is F16 else 63)  # in float16 products of inputs are far from the end of the range
    at, last = 63, length - 1
    x["log_decay"][:, at] = -float("inf")
    x["q"][:, last], x["k"][:, last], x["v"][:, last] = big, 0.0, 0.0
    x["k"][:, at], x["v"][:, at] = 0.0, 0.0
    x["k"][:, :at] = x["v"][:, :at] = 200.0
    leaves = [t.requires_grad_() for t in x.values()]
    dy = torch.zeros(n, length, heads, value, dtype=dtype, device="cuda")
    dy[:, last] = big
    dq, dk, dv, dg = torch.autograd.grad(ops.linear_attention(**x, scale=1.0), leaves, dy)
    for t in (dq, dk, dv, dg):
        assert torch.isfinite(t[:, :at]).all() and not t[:, :at].any()
    assert not dg[:, at].any()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("way", WAYS)
def test_a_large_state_times_a_small_scale_and_decay(gpu, way, dtype):
    n, heads, key, value = way
    half = {F32: 2.0 ** -24, BF: 2.0 ** -8}[dtype]
    x = dict(q=torch.zeros(n, 2, 1, key, dtype=dtype, device="cuda"), k=torch.zeros(n, 2, 1, key, dtype=dtype, device="cuda"),
             v=torch.zeros(n, 2, heads, value, dtype=dtype, device="cuda"), log_decay=torch.zeros(n, 2, heads, device="cuda"))
    x["q"][:, :, :, 0] = 4.0
    x["log_decay"][:, 1] = -60.0
    state = torch.full((n, heads, key, value), 3e38, device="cuda")
    y = ops.linear_attention(**x, scale=0.25, state=state).double()
    for t, want in enumerate((3e38, 3e38 * float(torch.tensor(-60.0, dtype=torch.float64).exp()))):
        # the power: 60 log2(e) = 87 rounded to float32 is off by 2^-18, so 2^e by ln 2 of that and its own rounding
        assert ((y[:, t] - want).abs() <= want * (half * (1 + 2.0 ** -6) + 2.0 ** -18 + 4 * 2.0 ** -24)).all()
    got = ops.linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"][:, 0], state=state, scale=0.25).double()
    assert ((got - 3e38).abs() <= 3e38 * (half * (1 + 2.0 ** -6) + 4 * 2.0 ** -24)).all() and (state == 3e38).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("way", WAYS)
def test_large_scores_that_are_forgotten(gpu, way, dtype):
    """Products of a query and a key beyond the range, with a decay to nothing between them."""
    n, heads, key, value = way
    big = (2.0 ** 70,) * 3
    for rows in (dict(q={1: big}, k={0: big}, v={0: (1.0, 2.0)}, dy={1: (3.0, 4.0)}), dict(v={0: big}, dy={1: big}, k={0: (1.0,)}, q={1: (2.0,)})):
        x = {name: torch.zeros(n, 2, *((1, key) if name in "qk" else (heads, value)), dtype=dtype, device="cuda") for name in ("q", "k", "v", "dy")}
        for name, at in rows.items():
            for t, v in at.items():
                x[name][:, t, :, :len(v)] = torch.tensor(v, device="cuda").to(dtype)
        dy = x.pop("dy")
        decay = torch.zeros(n, 2, heads, device="cuda")
        decay[:, 1] = -float("inf")
        leaves = [t.requires_grad_() for t in (*x.values(), decay)]
        y = ops.linear_attention(*leaves, scale=1.0)
        assert not y[:, 1].any()
        for t in torch.autograd.grad(y, leaves, dy):
            assert not t.any()


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_no_number_is_not_forgotten(gpu, bad, shape, dtype):
    """0 times an infinity or NaN is NaN: such a state, key or value reaches every position behind it, an upstream gradient every one
    before."""
    n, length, heads, key, value = shape
    x = _ordinary(*shape, dtype)
    x["log_decay"][:, 9] = -float("inf")
    for name in ("k", "v"):
        y = dict(x, **{name: x[name].clone()})
        y[name][0, 4, 0, 1] = bad
        got = ops.linear_attention(**y)
        assert not torch.isfinite(got[0, 9:, 0, 1]).any() and torch.isfinite(got[1:]).all() and torch.isfinite(got[0, :4]).all()
    state = torch.zeros(n, heads, key, value, device="cuda")
    state[0, 0, 1, 1] = bad
    got, last = ops.linear_attention(**x, state=state, return_state=True)
    assert not torch.isfinite(got[0, 9:, 0, 1]).any() and not torch.isfinite(last[0, 0, 1, 1])
    leaves = [t.requires_grad_() for t in x.values()]
    dy = torch.ones(n, length, heads, value, dtype=dtype, device="cuda")
    dy[0, 12, 0, 1] = bad
    _, dk, dv, _ = torch.autograd.grad(ops.linear_attention(*leaves), leaves, dy)
    assert not torch.isfinite(dv[0, :9, 0, 1]).any() and not torch.isfinite(dk[0, :9, 0]).any() and torch.isfinite(dv[1:]).all()
