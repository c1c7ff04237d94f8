"""The scan's vectorised 64-bit reference and its bound (scan_ref.py), on the CPU: against the position by position formulas, against
differences of rounding in float32, and that the bound sees what is kept in 16 bits."""
import pytest
import torch
import torch.nn.functional as F

import ops_ref as R
import scan_ref as S

F32 = torch.float32


def inputs(n, length, c, seed=0, dtype=F32, state=True):
    g = torch.Generator().manual_seed(seed + length + c)
    r = lambda *s, scale=1.0, mean=0.0: (torch.randn(s, generator=g) * scale + mean).to(dtype)  # noqa: E731
    s = {"u": r(n, length, c), "delta": r(n, length, c, scale=0.5),
         "A": (-torch.exp(r(c, 16, scale=0.1)) * torch.arange(1, 17)).float(), "B": r(n, length, 16), "C": r(n, length, 16),
         "D": r(c).float(), "z": r(n, length, c), "delta_bias": r(c, mean=-2.0).float()}
    return s, (r(n, 16, c).float() if state else None), r(n, length, c)


NAMES = {"u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "delta_bias": "dbias"}


@pytest.mark.parametrize("absent", [(), ("z",), ("D", "delta_bias"), ("z", "D", "delta_bias", "state")])
@pytest.mark.parametrize("ends", [None, (9, 0, 4)])
def test_values(absent, ends):
    s, state, dy = inputs(3, 9, 5)
    s = {k: None if k in absent else v for k, v in s.items()}
    state = None if "state" in absent else state
    lens = None if ends is None else torch.tensor(ends, dtype=torch.int32)
    if lens is not None:
        for k in ("u", "delta", "B", "C"):
            s[k][1, 0:], s[k][2, 4:] = float("nan"), float("nan")
    got = S.scan(**s, state=state, lens=lens, dy=dy)
    want = R.scan(*s.values(), state=state, lens=lens, dy=dy)
    assert set(got) == set(want)
    for k, (value, _) in want.items():
        assert torch.allclose(got[k][0], value, rtol=1e-12, atol=1e-12), k
        assert (got[k][1] >= 0).all() and got[k][1].isfinite().all(), k


def rounded(s, state, dy, at=None, every=64, keep=None):
    """Outputs and gradients by float32 operations one after the other, with autograd; `at`: the type that the state is rounded to
    behind every so many positions; keep: the type that the adjoint is rounded to at the same places."""
    leaves = {k: v.detach().clone().requires_grad_() for k, v in s.items()}
    u, delta, A, B, C, D, z, bias = leaves.values()
    dt = F.softplus(delta + bias)
    h, ys = state.transpose(1, 2), []
    for t in range(u.shape[1]):
        h = torch.exp(dt[:, t, :, None] * A) * h + B[:, t, None] * (dt[:, t] * u[:, t])[..., None]
        if t % every == every - 1:
            if at is not None:
                h = h + (h.to(at).float() - h).detach()
            if keep is not None:
                h.register_hook(lambda v: v.to(keep).float())
        ys.append(((h * C[:, t, None]).sum(-1) + D * u[:, t]) * F.silu(z[:, t]))
    y = torch.stack(ys, 1)
    grads = torch.autograd.grad(y, tuple(leaves.values()), dy)
    return {"y": y.detach(), "state": h.detach().transpose(1, 2), **{NAMES[k]: v for k, v in zip(leaves, grads)}}


@pytest.mark.parametrize("n,length,c", [(1, 300, 70), (2, 1000, 20), (3, 40, 5)])
def test_float32_is_within_the_bound(n, length, c):
    s, state, dy = inputs(n, length, c)
    ref, got = S.scan(**s, state=state, dy=dy), rounded(s, state, dy)
    for k, v in got.items():
        assert S.worst(v, ref[k]) <= 1, (k, S.worst(v, ref[k]))


@pytest.mark.parametrize("kept", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,length,c", [(1, 700, 70), (2, 2300, 10)])
def test_states_in_16_bits_are_not(n, length, c, kept):
    """With the widest chunks that the tests on the GPU have.  The state behind the last whole chunk, the outputs and gradients behind
    such states and adjoints, dB and dC in between: all exceed it."""
    s, state, dy = inputs(n, length, c)
    ref = S.scan(**s, state=state, dy=dy, chunk=264, parts=n * 128)
    got = rounded(s, state, dy, at=kept)
    for k in ("y", "dC", "dz"):
        assert S.worst(got[k], ref[k]) > 1, (k, S.worst(got[k], ref[k]))
    got = rounded(s, state, dy, keep=kept)
    for k in ("du", "ddelta", "dB"):
        assert S.worst(got[k], ref[k]) > 1, (k, S.worst(got[k], ref[k]))


@pytest.mark.parametrize("name", ["u", "delta", "A", "B", "C", "D", "z", "delta_bias"])
def test_inputs_in_16_bits_are_not(name):
    s, state, dy = inputs(1, 700, 70)
    ref = S.scan(**s, state=state, dy=dy, chunk=264, parts=128)
    for kept in (torch.bfloat16, torch.float16):
        got = S.scan(**{**s, name: s[name].to(kept).float()}, state=state, dy=dy)
        assert S.worst(got["y"][0].float(), ref["y"]) > 1, kept


def test_partial_sums_in_16_bits_are_not():
    """Of the parameters' gradients (a part for each of 10 chunks of 64 positions) and of dB and dC (a part for each block of channels)."""
    s, state, dy = inputs(1, 640, 130)
    ref = S.scan(**s, state=state, dy=dy, chunk=64, parts=10)
    cut = lambda v: v.to(torch.float16).double()  # noqa: E731
    full = S.scan(**s, state=state, dy=dy)
    parts = [S.scan(**{k: v[..., lo:lo + 64] if k in ("u", "delta", "z", "D", "delta_bias") else v[lo:lo + 64] if k == "A" else v
                       for k, v in s.items()}, state=state[..., lo:lo + 64], dy=dy[..., lo:lo + 64]) for lo in (0, 64, 128)]
    for k in ("dB", "dC"):
        whole = sum(p[k][0] for p in parts)
        assert torch.allclose(whole, full[k][0], rtol=1e-9, atol=1e-9)
        assert S.worst(sum(cut(p[k][0]) for p in parts).float(), ref[k]) > 1, k
    each = full["ddelta"][0].reshape(10, 64, 130).sum(1)
    assert S.worst(sum(cut(p) for p in each).float(), ref["dbias"]) > 1
