"""Drawn symbols against a restatement in 64 bits, which also says how near a row's choice was to another one: sums of the same
weights in another order differ by some 1e-16 of all of them per symbol, so rows within 1e-11 of a border are left out (there are
hardly any, which is checked)."""
import math

import pytest
import torch

import more_ops_ref as ref
from boa_amd import ops

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def _want(x, u, **kw):
    each = lambda i: {k: (v[i].item() if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}  # noqa: E731
    rows = [ref.sample(x[i].tolist(), u[i].item(), **each(i)) for i in range(len(x))]
    return torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows])


def _check(x, u, least_sure=0.99, **kw):
    got = ops.sample(x.cuda(), u.cuda(), **{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    assert got.dtype == torch.int64 and got.shape == u.shape
    want, near = _want(x.float(), u, **kw)
    sure = near > 1e-11
    assert sure.double().mean() >= least_sure
    assert torch.equal(got.cpu()[sure], want[sure])
    return got


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("v", [1, 2, 3, 63, 64, 65, 255, 256, 257, 260, 1000, 1024, 1025, 2048, 4093, 4096])
def test_every_size(gpu, v, dtype):
    g = torch.Generator().manual_seed(v)
    n = 40 if v <= 1024 else 12
    x = (3 * torch.randn(n, v, generator=g)).to(dtype)
    u = torch.rand(n, generator=g)
    _check(x, u)
    _check(x, u, temperature=0.7, top_k=max(1, v // 3))
    _check(x, u, temperature=1.3, top_p=0.8)
    _check(x, u, min_p=0.05)
    _check(x, u, temperature=0.9, top_k=max(1, v // 2), top_p=0.9, min_p=0.01)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,v", [(1, 256), (5, 256), (4097, 256), (300, 100), (37, 1500)])
def test_limits_of_each_row(gpu, n, v, dtype):
    g = torch.Generator().manual_seed(n)
    r = lambda: torch.rand(n, generator=g)  # noqa: E731
    x = (2 * torch.randn(n, v, generator=g)).to(dtype)
    t = r() * 2
    t[r() < 0.2] = 0.0
    _check(x, r(), temperature=t, top_k=torch.randint(-1, v + 5, (n,), generator=g, dtype=torch.int32), top_p=r() * 1.2, min_p=r() ** 4)


def test_equal_logits_count_in_the_symbols_order(gpu):
    """Weights of 1, whose sums are exact: the borders themselves."""
    for v in (256, 100, 1024, 2000):
        x = torch.zeros(64, v)
        u = torch.arange(64) / 64
        for kw in (dict(), dict(top_k=7), dict(top_p=0.5), dict(top_k=64, top_p=0.25), dict(top_p=1 / 1024), dict(min_p=1.0)):
            got = ops.sample(x.cuda(), u.cuda(), **kw).cpu()
            kept = min(kw.get("top_k", v), v)
            kept = math.ceil(kept * kw.get("top_p", 1.0))
            assert torch.equal(got, (u.double() * kept).floor().long()), (v, kw)
    x = torch.full((3, 256), -5.0)
    x[0, 9] = x[0, 200] = x[1, 255] = x[2, 0] = 4.0
    assert ops.sample(x.cuda(), torch.full((3,), 0.9).cuda(), temperature=0.0).tolist() == [9, 255, 0]
    assert ops.sample(x.cuda(), torch.full((3,), 0.9).cuda(), top_k=1).tolist() == [9, 255, 0]
    assert ops.sample(x.cuda(), torch.full((3,), 0.4).cuda(), top_k=2).tolist() == [9, 255, 0]
    assert ops.sample(x.cuda(), torch.full((3,), 0.6).cuda(), top_k=2).tolist() == [200, 255, 0]
    # many bfloat16 logits are equal; a zero of either sign is one
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-3, 4, (500, 256), generator=g).to(BF)
    x[:, ::3] *= -1.0
    for kw in (dict(top_k=50), dict(top_p=0.6), dict(top_k=100, top_p=0.3), dict(temperature=0.0)):
        _check(x, torch.rand(500, generator=g), least_sure=0.95, **kw)


def test_rows_that_are_masked(gpu):
    x = torch.randn(7, 256)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 77] = -3e38
    x[2, 5] = math.nan
    x[3, 3] = math.inf
    x[3, 200] = math.inf
    x[4, :] = torch.finfo(F32).min
    x[5, 1::2] = -math.inf
    u = torch.full((7,), 0.75)
    for kw in (dict(), dict(top_k=100), dict(top_p=0.9), dict(temperature=0.3, top_k=90, top_p=0.5, min_p=0.01), dict(temperature=1e-30),
               dict(temperature=math.inf)):
        got = _check(x, u, least_sure=1.0, **kw).tolist()
        kept = math.ceil(kw.get("top_k", 256) * kw.get("top_p", 1.0))
        assert got[4] == int(0.75 * kept) and got[3] == (3 if kw.get("top_p") == 0.5 else 200)
        assert got[0] == -1 and got[1] == 77 and got[2] == -1 and got[5] % 2 == 0
    assert ops.sample(x.cuda(), u.cuda(), temperature=0.0).tolist()[:4] == [-1, 77, -1, 3]
    wide = torch.randn(5, 3001)
    wide[0] = -math.inf
    wide[1, 3000] = math.nan
    wide[2, :3000] = -math.inf
    assert ops.sample(wide.cuda(), u[:5].cuda(), top_p=0.9).tolist()[:3] == [-1, -1, 3000]


def test_numbers_at_the_ends(gpu):
    x = torch.randn(6, 256)
    x[:, 0] = x[:, 255] = -math.inf
    below_one = 1 - 2.0 ** -24
    got = ops.sample(x.cuda(), torch.tensor([0.0, below_one, 1.0, 7.0, -1.0, math.nan]).cuda())
    assert got.tolist() == [1, 254, 254, 254, 1, -1]
    nan = torch.full((6,), math.nan, device="cuda")
    u = torch.full((6,), 0.5, device="cuda")
    for name in ("temperature", "top_p", "min_p"):
        assert ops.sample(x.cuda(), u, **{name: nan}).tolist() == [-1] * 6


def test_leading_shapes_and_strides(gpu):
    g = torch.Generator().manual_seed(2)
    x, u = torch.randn(4, 6, 256, generator=g), torch.rand(4, 6, generator=g)
    want = ops.sample(x.cuda(), u.cuda(), top_p=0.9)
    assert want.shape == (4, 6)
    assert torch.equal(ops.sample(x[2, 3].cuda(), u[2, 3].cuda(), top_p=0.9), want[2, 3])
    wide = torch.nn.functional.pad(x.cuda(), (3, 2))[..., 3:-2]
    assert torch.equal(ops.sample(wide, u.cuda(), top_p=0.9), want)
    assert torch.equal(ops.sample(x.cuda()[:, -1], u.cuda()[:, -1], top_p=0.9), want[:, -1])
    assert torch.equal(ops.sample(x.cuda().transpose(0, 2).contiguous().transpose(0, 2), u.cuda().t().contiguous().t(), top_p=0.9), want)
    assert ops.sample(torch.empty(0, 256, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)
    limit = torch.tensor([0.9], device="cuda").expand(4, 6)
    assert torch.equal(ops.sample(x.cuda(), u.cuda(), top_p=limit), ops.sample(x.cuda(), u.cuda(), top_p=float(limit[0, 0])))


def test_from_a_graph_and_on_another_stream(gpu):
    g = torch.Generator().manual_seed(3)
    x, u = torch.randn(700, 256, generator=g).cuda(), torch.rand(700, generator=g).cuda()
    run = lambda: ops.sample(x, u, temperature=0.8, top_k=40, top_p=0.9, min_p=0.01)  # noqa: E731
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run()
    for _ in range(3):
        u.copy_(torch.rand(700, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run())
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert torch.equal(out, run())


def test_drawn_as_often_as_the_weights_say(gpu):
    """65536 draws by evenly spaced numbers: each symbol's share is its probability to within one of them."""
    x = torch.randn(16, generator=torch.Generator().manual_seed(4))
    n = 65536
    got = ops.sample(x.cuda().expand(n, 16), (torch.arange(n) / n).cuda())
    share = torch.bincount(got.cpu(), minlength=16).double() / n
    assert (share - torch.softmax(x.double(), 0)).abs().max() <= 1.0 / n + 1e-12
