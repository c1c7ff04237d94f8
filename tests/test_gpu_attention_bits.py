"""Linear attention computes in float32 whatever its inputs' type: what is made on the way (a state, the scores, their gradients) keeps
all 24 bits where it meets inputs of 16.  Exact cases, in which two values that agree in their first 20 bits cancel, and random ones
under the bounds of test_gpu_attention.py without its allowance for products of fewer bits."""
import pytest
import torch

from boa_amd import ops
from test_gpu_attention import BF, F16, F32, _c, _inputs, _magnitudes
import more_ops_ref as ref

pytestmark = pytest.mark.gpu

LONG, SHORT = (1.0, 2.0 ** -9, 2.0 ** -20), (1.0, 2.0 ** -9, 0.0)  # their sums differ by the last bit but three of float32
LAST = 2.0 ** -20
# one head by itself, with up to 64 and with more keys; heads of a group in turn (1024 workgroups and more)
WAYS = [(1, 1, 5, 6), (2, 1, 100, 70), (1100, 4, 5, 6)]


def _run(n, heads, key, value, dtype, length, **rows):
    """Zeros but for the values given per name and position, of head 0 of every sequence; no decay, a scale of 1."""
    x = {name: torch.zeros(n, length, *((1, key) if name in "qk" else (heads, value)), dtype=dtype, device="cuda") for name in ("q", "k", "v", "dy")}
    for name, at in rows.items():
        for t, v in at.items():
            x[name][:, t, 0, :len(v)] = torch.tensor(v, device="cuda").to(dtype)
    dy = x.pop("dy")
    leaves = {name: t.requires_grad_() for name, t in x.items()}
    decay = torch.zeros(heads, device="cuda")

    def forward(state=None):
        return ops.linear_attention(**leaves, log_decay=decay, scale=1.0, state=state)

    return forward, lambda: dict(zip(leaves, torch.autograd.grad(forward(), list(leaves.values()), dy)))


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("way", WAYS)
def test_the_state_in_y(gpu, way, dtype):
    n, heads, key, value = way
    forward, _ = _run(*way, dtype, 2, q={0: (1.0, -1.0), 1: (-1.0, 1.0)})
    state = torch.zeros(n, heads, key, value, device="cuda")
    state[:, :, 0], state[:, :, 1] = sum(LONG), sum(SHORT)
    y = forward(state)
    assert (y[:, 0] == LAST).all() and (y[:, 1] == -LAST).all()


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("way", WAYS)
def test_scores_in_y(gpu, way, dtype):
    forward, _ = _run(*way, dtype, 3, q={2: (1.0, 1.0, 1.0)}, k={0: LONG, 1: SHORT}, v={0: (1.0,), 1: (-1.0,)})
    y = forward()
    assert (y[:, 2, 0, 0] == LAST).all() and not y[:, :2].any() and not y[..., 1:].any() and not y[:, :, 1:].any()


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("way", WAYS)
def test_a_states_gradient_in_the_values(gpu, way, dtype):
    two = {64 + i: (LONG[i], SHORT[i]) for i in range(3)}
    _, grads = _run(*way, dtype, 70, q=two, dy={t: (1.0,) for t in two}, k={t: (1.0, -1.0) for t in range(64)})
    dv = grads()["v"]
    assert (dv[:, :64, 0, 0] == LAST).all() and not dv[:, 64:].any() and not dv[..., 1:].any()


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("which,rows,at", [
    ("v", dict(q={1: LONG, 2: SHORT}, k={0: (1.0, 1.0, 1.0)}, dy={1: (1.0,), 2: (-1.0,)}), 0),
    ("q", dict(v={0: LONG, 1: SHORT}, dy={2: (1.0, 1.0, 1.0)}, k={0: (1.0,), 1: (-1.0,)}), 2),
    ("k", dict(dy={1: LONG, 2: SHORT}, v={0: (1.0, 1.0, 1.0)}, q={1: (1.0,), 2: (-1.0,)}), 0),
])
def test_scores_in_the_gradients(gpu, which, rows, at, way, dtype):
    _, grads = _run(*way, dtype, 3, **rows)
    got = grads()[which][:, :, 0, 0]
    assert (got[:, at] == LAST).all()


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1, 1), (2, 9, 2, 2, 3, 2), (2, 130, 4, 2, 64, 64), (1, 200, 2, 1, 100, 130), (600, 65, 4, 1, 9, 9)])
def test_random_ones_without_allowance(gpu, size, dtype):
    n, length, heads, groups, key, value = size
    x, dy, lens, s = _inputs(*size, dtype, "token", seed=31, ragged=True, state=True)
    leaves = [t.cuda().requires_grad_() for t in x.values()]
    y, last = ops.linear_attention(*leaves, state=s.cuda(), lens=lens.cuda(), return_state=True)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    want = ref.attention_grads(*x.values(), key ** -0.5, dy, lens, s)
    terms = _magnitudes(x, dy, key ** -0.5, lens, s)
    c = _c(length, key, value, x["log_decay"])
    more = c + heads // groups * -(-value // 64)
    for got, w, t, roundings in zip((y, last, *grads), (*want[:2], *want[2]), (*terms[:2], *terms[2]), (c, c, more, more, more, c + 64)):
        half = {F32: 2.0 ** -24, BF: 2.0 ** -8, F16: 2.0 ** -11}[got.dtype]
        tiny = 2.0 ** -25 if got.dtype == F16 else 2.0 ** -100
        off = (got.detach().cpu().double() - w).abs()
        assert (off <= half * w.abs() * (1 + 2.0 ** -6) + roundings * 2.0 ** -24 * t + tiny).all()
