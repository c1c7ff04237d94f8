"""Linear attention at the ends of float32's range: what is finite in the definition's own order of operations comes out finite."""
import pytest
import torch

from boa_amd import ops
from test_gpu_attention import BF, F32
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
