"""The 64-bit restatements themselves, on the CPU: gradients against differences, drawn symbols against a search of all."""
import itertools
import math

import pytest
import torch

import more_ops_ref as ref


@pytest.mark.parametrize("per_head", [False, True])
def test_gradients_against_differences(per_head):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    n, length, heads, groups, key, value = 2, 6, 4, 2, 3, 2
    leaves = [r(n, length, groups, key), r(n, length, groups, key), r(n, length, heads, value), -r(*((heads,) if per_head else (n, length, heads))).abs()]
    lens, state = torch.tensor([6, 4]), r(n, heads, key, value)
    up = r(n, length, heads, value)
    _, _, grads = ref.attention_grads(*leaves, 0.7, up, lens, state)
    f = lambda *x: float((ref.attention(*x, 0.7, lens, state)[0] * up).sum())  # noqa: E731
    for i, (x, d) in enumerate(zip(leaves, grads)):
        for at in itertools.islice(itertools.product(*map(range, x.shape)), 0, None, 5):
            h, moved = 1e-6, []
            for s in (h, -h):
                y = x.clone()
                y[at] += s
                moved.append(f(*leaves[:i], y, *leaves[i + 1:]))
            assert abs((moved[0] - moved[1]) / (2 * h) - float(d[at])) <= 1e-7 * (1 + abs(float(d[at])))


def test_attention_is_the_sum_over_pairs():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, d = r(1, 7, 1, 3), r(1, 7, 1, 3), r(1, 7, 1, 2), -r(1, 7, 1).abs()
    y, _ = ref.attention(q, k, v, d, 1.0)
    for i in range(7):
        want = sum(math.exp(float(d[0, j + 1:i + 1].sum())) * float(q[0, i, 0] @ k[0, j, 0]) * v[0, j, 0] for j in range(i + 1))
        assert torch.allclose(y[0, i, 0], want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("x,u,kw,want", [
    ([0.0, 0.0, 0.0, 0.0], 0.0, {}, 0), ([0.0, 0.0, 0.0, 0.0], 0.25, {}, 1), ([0.0, 0.0, 0.0, 0.0], 0.999, {}, 3),
    ([0.0, 0.0, 0.0, 0.0], 0.999, dict(top_k=2), 1), ([0.0, 0.0, 0.0, 0.0], 0.999, dict(top_p=0.5), 1),
    ([0.0, 0.0, 0.0, 0.0], 0.999, dict(top_p=0.500001), 2), ([0.0, math.log(0.5), 0.0], 0.5, dict(min_p=0.75), 2),
    ([1.0, 3.0, 3.0], 0.9, dict(temperature=0.0), 1), ([-math.inf, 2.0], 0.0, {}, 1), ([-math.inf, -math.inf], 0.5, {}, -1),
    ([math.nan, 1.0], 0.5, {}, -1), ([math.inf, 5.0, math.inf], 0.6, {}, 2), ([0.0, 1.0], math.nan, {}, -1)])
def test_drawn_symbols(x, u, kw, want):
    assert ref.sample(x, u, **kw)[0] == want
