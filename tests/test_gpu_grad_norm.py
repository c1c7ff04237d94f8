"""The norm of gradients together and their clipping, against 64 bits.  Sums are in 64 bits and rounded once: the norm is off by half
a step of float32 (2^-24) and what 64-bit sums lose; a scaled gradient by the factor's rounding, the product's and its own."""
import math

import pytest
import torch

from boa_amd import ops

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF: 2.0 ** -8, F16: 2.0 ** -11}


def _params(shapes, seed=0, dtypes=(F32,), scale=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, shape in enumerate(shapes):
        dt = dtypes[i % len(dtypes)]
        p = torch.nn.Parameter(torch.zeros(shape, dtype=dt, device="cuda"))
        p.grad = (scale * torch.randn(shape, generator=g)).to(dt).cuda()
        out.append(p)
    return out


def _norm(params, p=2.0):
    grads = [q.grad.double().flatten() for q in params if q.grad is not None]
    return float(torch.linalg.vector_norm(torch.cat(grads), p)) if grads else 0.0


def _near(got, want):
    """Within a step of float32; infinite where that cannot hold it."""
    got = float(got)
    return got == math.inf if want >= (2 - 2.0 ** -24) * 2.0 ** 127 else abs(got - want) <= 2.0 ** -23 * want


def _check(params, max_norm, norm_type=2.0):
    before = [None if p.grad is None else p.grad.clone() for p in params]
    want = _norm(params, norm_type)
    if any(p.grad is not None for p in params):
        assert _near(ops.grad_norm(params, norm_type=norm_type), want)
    got = ops.clip_grad_norm_(params, max_norm, norm_type=norm_type)
    assert got.shape == () and got.dtype == F32 and _near(got, want)
    f = min(1.0, max_norm / (want + 1e-6))
    for p, b in zip(params, before):
        if b is None:
            assert p.grad is None
            continue
        if f == 1.0:
            assert torch.equal(p.grad, b)
            continue
        x = b.double() * f
        tiny = 2.0 ** -25 if p.dtype == F16 else 2.0 ** -149
        assert ((p.grad.double() - x).abs() <= x.abs() * (HALF[p.dtype] + 4 * 2.0 ** -24) + tiny).all()


SHAPES = [(256, 256), (1,), (3, 5, 7), (1000,), (0,), (512, 1, 4), (), (4097,)]


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [(F32,), (BF,), (F16,), (F32, BF, F16)])
@pytest.mark.parametrize("max_norm", [1.0, 0.0, 1e4, math.inf])
def test_sizes_and_types(gpu, dtypes, max_norm, norm_type):
    _check(_params(SHAPES, 1, dtypes), max_norm, norm_type)


@pytest.mark.parametrize("count", [1, 2, 179, 180, 181, 400])
def test_more_tensors_than_a_launch_takes(gpu, count):
    _check(_params([(1 + 37 * i % 300,) for i in range(count)], count, (F32, BF)), 0.5)


def test_more_blocks_than_workgroups(gpu):
    _check(_params([(40_000_001,), (17,), (5000, 4097)], 2, (BF, F32), scale=0.1), 1.0)
    _check(_params([(40_000_001,), (17,), (5000, 4097)], 2, (F16, F32), scale=0.1), 1.0, math.inf)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_views_at_every_offset_of_one_buffer(gpu, dtype):
    """What lies beside a gradient stays as it is."""
    sizes = [1, 2, 3, 5, 8, 13, 31, 64, 100, 257, 1023, 4096, 4099, 20000]
    g = torch.Generator().manual_seed(3)
    buf = torch.randn(sum(sizes) + 2 * len(sizes) + 7, generator=g).to(dtype).cuda()
    kept, at, params = buf.clone(), 1, []
    inside = torch.zeros(len(buf), dtype=torch.bool)
    for n in sizes:
        p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device="cuda"))
        p.grad = buf[at:at + n]
        inside[at:at + n] = True
        params.append(p)
        at += n + (at % 3)
    _check(params, 0.25)
    assert torch.equal(buf[~inside], kept[~inside]) and not torch.equal(buf[inside], kept[inside])


def test_large_and_small_values_stay_in_range(gpu):
    for scale, dtype in ((1e30, F32), (1e-30, F32), (6e4, F16), (1e-7, F16), (1e38, BF)):
        params = _params([(1000,), (33,)], 4, (dtype,))
        for i, p in enumerate(params):
            x = torch.rand(p.shape, generator=torch.Generator().manual_seed(i)) * 2 - 1
            p.grad.copy_(x * scale)
        _check(params, 1.0)
        _check(params, 1.0, math.inf)


def test_what_is_not_a_number(gpu):
    params = _params([(100,), (7,)], 5)
    params[0].grad[50] = math.nan
    assert math.isnan(ops.grad_norm(params)) and math.isnan(ops.grad_norm(params, norm_type=math.inf))
    assert math.isnan(ops.clip_grad_norm_(params, 1.0)) and all(p.grad.isnan().all() for p in params)
    params = _params([(100,), (7,)], 5)
    params[1].grad[3] = -math.inf
    assert float(ops.clip_grad_norm_(params, 1.0)) == math.inf
    assert not params[0].grad.any() and params[1].grad[3].isnan() and not params[1].grad[:3].any()


def test_gradients_that_are_not_contiguous_and_those_that_are_missing(gpu):
    params = _params([(64, 32), (5, 6, 7), (10,), (3,)], 6)
    params[0].grad = params[0].grad.t().contiguous().t()
    params[1].grad = torch.randn(7, 6, 10, device="cuda")[..., ::2].permute(2, 1, 0)
    params[3].grad = None
    _check(params, 0.1)
    only = _params([(9,)], 7)
    _check(only, 0.1)
    want = _norm(only)
    assert abs(float(ops.grad_norm(only[0])) - want) <= 2.0 ** -23 * want  # a tensor by itself
    assert float(ops.clip_grad_norm_((p for p in only), 1e9)) == float(ops.grad_norm(only))  # an iterator
    assert float(ops.clip_grad_norm_([params[3]], 1.0)) == 0.0 and float(ops.grad_norm([])) == 0.0
    assert float(ops.clip_grad_norm_(_params([(0,), (0, 5)]), 1.0)) == 0.0
    params[2].grad = torch.randn(1, device="cuda").expand(10)
    ops.grad_norm(params)
    before = params[0].grad.clone()
    with pytest.raises(ValueError, match="share memory"):
        ops.clip_grad_norm_(params, 0.1)
    assert torch.equal(before, params[0].grad)


def test_gradients_that_share_memory_are_refused(gpu):
    params = _params([(100,), (100,)], 8)
    buf = torch.randn(150, device="cuda")
    params[0].grad, params[1].grad = buf[:100], buf[50:]
    before = buf.clone()
    with pytest.raises(ValueError, match="share memory"):
        ops.clip_grad_norm_(params, 0.1)
    with pytest.raises(ValueError, match="share memory"):
        ops.clip_grad_norm_([params[0], params[0]], 0.1)
    assert torch.equal(buf, before)
    ops.grad_norm(params)


def test_a_gradient_given_twice_that_is_not_contiguous_is_refused(gpu):
    p, = _params([(64, 32)], 8)
    p.grad = p.grad.t().contiguous().t()
    before = p.grad.clone()
    with pytest.raises(ValueError, match="share memory"):
        ops.clip_grad_norm_([p, p], 0.1)
    assert torch.equal(p.grad, before)
    p.grad = p.grad.t().contiguous().t()
    q = torch.nn.Parameter(torch.zeros(32, 64, device="cuda"))
    q.grad = p.grad.t()
    with pytest.raises(ValueError, match="share memory"):
        ops.clip_grad_norm_([q, p], 0.1)
    assert torch.equal(p.grad, before)


def test_autograd_sees_that_gradients_were_scaled(gpu):
    p, = _params([(10,)], 9)
    version = p.grad._version
    ops.clip_grad_norm_([p], 0.1)
    assert p.grad._version == version + 1
    version = p.grad._version
    ops.grad_norm([p])
    assert p.grad._version == version


def test_the_same_bits_from_a_graph_and_on_another_stream(gpu):
    params = _params([(100_000,), (333,), (64, 64)], 10, (F32, BF))
    start = [p.grad.clone() for p in params]

    def run():
        for p, s in zip(params, start):
            p.grad.copy_(s)
        return ops.clip_grad_norm_(params, 0.5)

    norm = run()
    want = [p.grad.clone() for p in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run()
    for _ in range(3):
        for p in params:
            p.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, norm) and all(torch.equal(p.grad, w) for p, w in zip(params, want))
    with torch.cuda.stream(side):
        assert torch.equal(run(), norm)
    torch.cuda.synchronize()
    assert all(torch.equal(p.grad, w) for p, w in zip(params, want))
