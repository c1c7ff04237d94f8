"""The selective scan on every way that its length is split, against scan_ref.py's formulas in 64 bits under the bound carried along the
recurrences (which states, adjoints or partial sums kept in 16 bits exceed: test_scan_ref.py).

The split follows from sizes and lens alone; each case says how many chunks it is meant to have forward and backward, and the
workspace's size how many it has.  A chunk of 64 positions is the shortest; from 33 chunks on they are joined by a kernel of its
own, 32 of them in each of its wavefronts; 128 are the most."""
import pytest
import torch

import scan_ref as S
from boa_amd import _native, ops

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = {"u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "delta_bias": "dbias"}


def split(n, length, c, lens):
    """Chunks forward and backward, and the most positions that one of them may have."""
    packed = ops._SCAN.pack(0, c, n, length, *[0] * 18, 4096 if lens else 0, *[0] * 25)
    size = _native.load_cdll().boa_selective_scan_work_bytes
    fwd, bwd = size(packed, 0) // 4, size(packed, 1) // 4 - -(-c // 64) * n * -(-length // 8) * 256
    fwd = fwd // (n * 17 * c) or 1
    bwd = bwd // (n * 35 * c) if bwd > n * 18 * c else 1
    longest = max((length - 1) // (k - 1) // 8 * 8 if k > 1 else length for k in (fwd, bwd))
    return fwd, bwd, longest


def inputs(n, length, c, dtype, seed, gate=True, params=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, scale=1.0, mean=0.0: torch.randn(s, generator=g, device="cuda") * scale + mean  # noqa: E731
    s = {"u": r(n, length, c).to(dtype), "delta": r(n, length, c, scale=0.5).to(dtype),
         "A": -torch.exp(r(c, 16, scale=0.1)) * torch.arange(1, 17, device="cuda"), "B": r(n, length, 16).to(dtype),
         "C": r(n, length, 16).to(dtype), "D": r(c), "z": r(n, length, c).to(dtype), "delta_bias": r(c, mean=-2.0)}
    if not gate:
        s["z"] = None
    if not params:
        s["D"] = s["delta_bias"] = None
    return s, r(n, 16, c), r(n, length, c).to(dtype)


def check(n, length, c, dtype, lens=None, gate=True, params=True, state=True, seed=0):
    s, h0, dy = inputs(n, length, c, dtype, seed + length + c, gate, params)
    h0 = h0 if state else None
    fwd, bwd, longest = split(n, length, c, lens is not None)
    if lens is not None:
        lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        behind = torch.arange(length, device="cuda") >= lens[:, None]
        for t in (s["u"], s["delta"], s["B"], s["C"], s["z"], dy):
            if t is not None:
                t[behind] = float("nan")
    leaves = {k: v.requires_grad_() for k, v in s.items() if v is not None}
    y, end = ops.selective_scan(**s, state=h0, lens=lens, return_state=True)
    got = {"y": y.detach(), "state": end}
    got.update({NAMES[k]: v for k, v in zip(leaves, torch.autograd.grad(y, tuple(leaves.values()), dy))})
    with torch.no_grad():
        assert torch.equal(ops.selective_scan(**s, state=h0, lens=lens), y)  # with and without what the gradient needs
    ref = S.scan(**s, state=h0, lens=lens, dy=dy, chunk=longest if max(fwd, bwd) > 1 else 0, parts=n * bwd)
    off = {k: S.worst(v, ref[k]) for k, v in got.items()}
    assert all(v <= 1 for v in off.values()), off
    if lens is not None:
        for k, v in got.items():
            if v.ndim == 3 and k != "state":
                assert not v[behind].any(), k
        assert h0 is None or torch.equal(end[lens <= 0], h0[lens <= 0])
    print(" ".join(f"{k}={v:.2f}" for k, v in off.items()), end=" ")


# name: batch, length, channels, lens, chunks forward and backward
SPLITS = {
    "joined by four wavefronts, the last one in part": (1, 9000, 70, None, 125, 125),
    "joined by three": (2, 5700, 70, None, 90, 90),
    "128 chunks": (1, 16384, 33, None, 128, 128),
    "joined, chunks of odd multiples of 8, ends on their borders": (2, 9211, 70, (9211, 72 * 50), 128, 128),
    "joined, ends one before and one behind a border": (3, 8500, 9, (72 * 32 - 1, 72 * 64 + 1, 72 * 96), 119, 119),
    "not joined, chunks beyond 64": (32, 1600, 128, None, 23, 16),
    "not joined, padded": (64, 1600, 130, tuple([0, 1600, 80, 79, 81, 1, 8, 1520, 1521, 1519, 799, 160] + [37 * i for i in range(1, 41)] + [1599] * 12), 20, 20),
    "two chunks of a batch that almost fills the card": (600, 150, 65, None, 2, 1),
    "a batch that fills the card": (800, 90, 65, None, 1, 1),
    "a batch that fills the card, padded": (2100, 70, 65, tuple((i * 31) % 71 for i in range(2100)), 1, 1),
}


def test_the_cases_are_split_as_they_are_meant_to_be(gpu):
    for name, (n, length, c, lens, fwd, bwd) in SPLITS.items():
        assert split(n, length, c, lens is not None)[:2] == (fwd, bwd), name


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("name", SPLITS)
def test_split(gpu, name, dtype):
    n, length, c, lens, _, _ = SPLITS[name]
    check(n, length, c, dtype, lens)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("gate,params,state", [(False, True, True), (True, False, False), (False, False, True)])
@pytest.mark.parametrize("n,length,c,lens", [(1, 2300, 40, None), (2, 2500, 130, (2500, 130)), (2, 4700, 70, (4700, 0))])
def test_joined_without_gate_or_parameters(gpu, n, length, c, lens, gate, params, state, dtype):
    assert split(n, length, c, lens is not None)[0] > 32
    check(n, length, c, dtype, lens, gate, params, state)


def test_chunks_of_a_few_hundred_positions(gpu):
    """Of a batch of 32 workgroups: 47 chunks of 176 forward, joined, and 32 of 264 backward, not joined."""
    assert split(2, 8197, 1024, False) == (47, 32, 264)
    check(2, 8197, 1024, F32)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("n,length,c", [(1, 1, 1), (2, 2, 3), (2, 7, 5), (3, 8, 64), (2, 9, 65), (1, 40, 130), (2, 100, 33), (1, 129, 64),
                                        (1, 700, 70), (4, 65, 256)])
def test_small(gpu, n, length, c, dtype):
    check(n, length, c, dtype, state=False)
    check(n, length, c, dtype, tuple((length, 0, 1, length // 2)[i % 4] for i in range(n)))


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("n,c", [(1, 1), (3, 5), (1, 512), (300, 65), (64, 1024)])
def test_steps(gpu, n, c, dtype):
    s, state, _ = inputs(n, 12, c, dtype, n + c)
    ref, st = S.scan(**s, state=state), state.clone()
    for t in range(12):
        at = {k: v[:, t] if k in ("u", "delta", "B", "C", "z") else v for k, v in s.items()}
        y = ops.selective_scan_step(**at, state=st)
        assert S.worst(y, (ref["y"][0][:, t], ref["y"][1][:, t])) <= 1
    assert S.worst(st, ref["state"]) <= 1
