"""Linear attention with a decay for each head, and its single-token form, against 64 bits on the CPU.

Bounds: a result is a sum of products of inputs and of powers of the decay.  With every input replaced by its magnitude the
reference gives the sum of the terms' magnitudes, T (its gradients those of the gradients' terms), and a float32 computation of
them is off by at most c 2^-24 T, c the roundings that a term passes: a dot product over the key and one over the values, up to 64
positions of a chunk twice, a state's update per chunk, and of each power the rounding of its exponent, which is at most its
magnitude.  bfloat16 products on the way keep 16 bits at least (2^-16 of a term, twice).  The result's own rounding is half a step.
A power or product below float32's smallest normal number, 2^-126, may come out as zero: that is off by 2^-126 times the other
factors of its term, and all terms of a result have less than 2^26 of those here (up to 700 positions, 128 keys, four inputs of up to
5): 2^-100."""
import math

import pytest
import torch

import more_ops_ref as ref
from boa_amd import ops

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def _inputs(n, length, heads, groups, key, value, dtype, decay, seed=0, ragged=False, state=False, low=-0.3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x = dict(q=r(n, length, groups, key).to(dtype), k=r(n, length, groups, key).to(dtype), v=r(n, length, heads, value).to(dtype))
    shape = (heads,) if decay == "head" else (n, length, heads)
    x["log_decay"] = low * torch.rand(shape, generator=g)
    lens = None
    if ragged:
        lens = torch.randint(0, length + 1, (n,), generator=g, dtype=torch.int32)
        lens[0] = length
        if n > 1:
            lens[-1] = 0
    s = r(n, heads, key, value) if state else None
    return x, r(n, length, heads, value).to(dtype), lens, s


def _bound(got, want, terms, c):
    own = {F32: 2.0 ** -24, BF: 2.0 ** -8, F16: 2.0 ** -11}[got.dtype]
    mid = 2.0 ** -15 if got.dtype == BF else 0.0
    tiny = 2.0 ** -25 if got.dtype == F16 else 2.0 ** -100  # half a step of the smallest float16 numbers; what underflows
    off = (got.detach().cpu().double() - want).abs()
    over = off - (own * want.abs() * (1 + 2.0 ** -6) + (c * 2.0 ** -24 + mid) * terms + tiny)
    assert not torch.isnan(got).any()
    assert (over <= 0).all(), f"{int((over > 0).sum())} of {off.numel()} beyond, at most {float((off / (terms + 1e-300)).max()):.3g} of the terms"


def _c(length, key, value, g):
    chunks = -(-length // 64)
    exponents = min(64 * float(g.clamp(min=-2.5).abs().max()) * 1.4427, 200.0)  # a power below 2^-200 is nothing
    return key + value + 2 * 64 + 6 * chunks + 3 * exponents + 20


def _magnitudes(x, dy, scale, lens, s):
    """The terms' magnitudes: of y and the state, and of the gradients."""
    return ref.attention_grads(*(t.detach().abs() if name != "log_decay" else t for name, t in x.items()), abs(scale), dy.abs(), lens,
                               None if s is None else s.abs())


def _check(n, length, heads, groups, key, value, dtype, decay, ragged=False, state=False, scale=None, seed=0, low=-0.3, change=None):
    x, dy, lens, s = _inputs(n, length, heads, groups, key, value, dtype, decay, seed, ragged, state, low)
    if change is not None:
        change(x)
    gx = {k: t.cuda().requires_grad_() for k, t in x.items()}
    gl, gs = (None if t is None else t.cuda() for t in (lens, s))
    y, last = ops.linear_attention(**gx, scale=scale, state=gs, lens=gl, return_state=True)
    assert y.shape == dy.shape and y.dtype == dtype and y.is_contiguous() and last.dtype == F32
    grads = torch.autograd.grad(y, list(gx.values()), dy.cuda())
    with torch.no_grad():
        plain = ops.linear_attention(**{k: t.detach() for k, t in gx.items()}, scale=scale, state=gs, lens=gl)
    assert torch.equal(plain, y)
    sc = key ** -0.5 if scale is None else scale
    want = ref.attention_grads(*x.values(), sc, dy, lens, s)
    terms = _magnitudes(x, dy, sc, lens, s)
    c = _c(length, key, value, x["log_decay"])
    _bound(y, want[0], terms[0], c)
    _bound(last, want[1], terms[1], c)
    for got, w, t, name in zip(grads, want[2], terms[2], x):
        assert got.dtype == x[name].dtype and got.shape == x[name].shape
        # the decay of a head: one more sum over all positions; dg: float32 whatever the inputs, by way of three parts (24 bits)
        _bound(got, w, t, (c + 64 + n * length ** 0.5) if name == "log_decay" else c + heads // groups * -(-value // 64))
    if lens is not None:
        behind = torch.arange(length)[None] >= lens[:, None]
        for t in (y, *grads[:3]) + ((grads[3],) if decay == "token" else ()):
            assert not t.detach().cpu()[behind].any()


SIZES = [(1, 1, 1, 1, 1, 1), (2, 2, 3, 3, 5, 7), (1, 63, 2, 1, 64, 64), (2, 64, 2, 2, 16, 64), (1, 65, 4, 2, 64, 32), (3, 129, 4, 1, 17, 33),
         (2, 200, 6, 3, 64, 64), (1, 130, 2, 2, 128, 64), (1, 150, 2, 1, 100, 130), (2, 70, 3, 3, 5, 300), (1, 700, 1, 1, 40, 64)]


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradient(gpu, size, dtype):
    _check(*size, dtype, "token", seed=1)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("size", SIZES[1::2])
def test_a_decay_of_the_head(gpu, size, dtype):
    _check(*size, dtype, "head", seed=2, scale=0.37)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("size", [(4, 3, 2, 2, 8, 8), (5, 130, 2, 1, 64, 64), (4, 257, 2, 2, 33, 65)])
def test_padded_batches_that_go_on_from_states(gpu, size, decay, dtype):
    _check(*size, dtype, decay, ragged=True, state=True, seed=3)


def test_many_sequences_need_no_split(gpu):
    """1100 workgroups: a sequence is walked by one of them, which starts from the caller's state."""
    _check(275, 70, 4, 4, 8, 8, F32, "token", ragged=True, state=True, seed=4)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("low", [0.0, -5.0, -300.0])
def test_slow_and_fast_decays(gpu, low, dtype):
    _check(2, 200, 2, 2, 32, 32, dtype, "token", seed=5, low=low)


def test_a_decay_to_nothing_forgets_and_leaves_what_follows_exact(gpu):
    """-inf, and steps so large that a sum of logarithms in 32 bits would lose the small ones behind them."""
    def change(x):
        x["log_decay"][:, 10] = -math.inf
        x["log_decay"][:, 70] = -1e4
        x["log_decay"][:, 71:90] = -1e-3

    x, dy, lens, s = _inputs(2, 140, 2, 2, 16, 16, F32, "token", 6, state=True)
    change(x)
    gx = {k: t.cuda().requires_grad_() for k, t in x.items()}
    y, last = ops.linear_attention(**gx, state=s.cuda(), return_state=True)
    grads = torch.autograd.grad(y, list(gx.values()), dy.cuda())
    x["log_decay"] = x["log_decay"].clamp(min=-1e3)  # zero in 64 bits too, and the reference's gradient a number
    want, terms = ref.attention_grads(*x.values(), 0.25, dy, lens, s), _magnitudes(x, dy, 0.25, lens, s)
    c = _c(140, 16, 16, x["log_decay"])
    _bound(y, want[0], terms[0], c)
    _bound(last, want[1], terms[1], c)
    for got, w, t in zip(grads, want[2], terms[2]):
        _bound(got, w, t, c + 100)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_single_tokens_and_whole_sequences_agree(gpu, dtype):
    for heads, groups, key, value, decay in ((4, 2, 64, 64, "token"), (3, 3, 17, 65, "head"), (2, 1, 128, 33, "token"), (1, 1, 1, 1, "head")):
        n, length = 3, 9
        x, dy, _, s = _inputs(n, length, heads, groups, key, value, dtype, decay, 7, state=True)
        state = s.cuda()
        gx = {k: t.cuda() for k, t in x.items()}
        ys = []
        for t in range(length):
            version = state._version
            g = gx["log_decay"] if decay == "head" else gx["log_decay"][:, t]
            ys.append(ops.linear_attention_step(gx["q"][:, t], gx["k"][:, t], gx["v"][:, t], g, state=state))
            assert state._version == version + 1
        want, terms = ref.attention_grads(*x.values(), key ** -0.5, dy, None, s), _magnitudes(x, dy, key ** -0.5, None, s)
        c = _c(length, key, value, x["log_decay"])
        _bound(torch.stack(ys, 1), want[0], terms[0], c)
        _bound(state, want[1], terms[1], c)


def test_steps_of_many_sequences(gpu):
    x, dy, _, s = _inputs(1500, 1, 3, 3, 20, 24, BF, "token", 8, state=True)
    state = s.cuda()
    y = ops.linear_attention_step(*(t[:, 0].cuda() for t in x.values()), state=state)
    want, terms = ref.attention_grads(*x.values(), 20 ** -0.5, dy, None, s), _magnitudes(x, dy, 20 ** -0.5, None, s)
    _bound(y, want[0][:, 0], terms[0][:, 0], 200)
    _bound(state, want[1], terms[1], 200)


def test_a_prompt_in_two_halves_is_the_whole(gpu):
    x, dy, _, s = _inputs(2, 300, 2, 2, 32, 48, F32, "token", 9, state=True)
    gx = {k: t.cuda() for k, t in x.items()}
    half = lambda a, b: {k: t[:, a:b] for k, t in gx.items()}  # noqa: E731
    y0, s0 = ops.linear_attention(**half(0, 77), state=s.cuda(), return_state=True)
    y1, s1 = ops.linear_attention(**half(77, 300), state=s0, return_state=True)
    want, terms = ref.attention_grads(*x.values(), 32 ** -0.5, dy, None, s), _magnitudes(x, dy, 32 ** -0.5, None, s)
    _bound(torch.cat([y0, y1], 1), want[0], terms[0], _c(300, 32, 48, x["log_decay"]))
    _bound(s1, want[1], terms[1], _c(300, 32, 48, x["log_decay"]))


def test_nothing_to_do(gpu):
    s = torch.randn(2, 3, 5, 6, device="cuda")
    empty = lambda n, length: dict(q=torch.zeros(n, length, 3, 5, device="cuda"), k=torch.zeros(n, length, 3, 5, device="cuda"),  # noqa: E731
                                   v=torch.zeros(n, length, 3, 6, device="cuda"), log_decay=torch.zeros(3, device="cuda", requires_grad=True))
    y, last = ops.linear_attention(**empty(2, 0), state=s, return_state=True)
    assert y.shape == (2, 0, 3, 6) and torch.equal(last, s) and last.data_ptr() != s.data_ptr()
    x = empty(2, 0)
    assert not ops.linear_attention(**x, return_state=True)[1].any()
    ops.linear_attention(**x).sum().backward()
    assert torch.equal(x["log_decay"].grad, torch.zeros(3, device="cuda"))
    x = empty(0, 5)
    ops.linear_attention(**x).sum().backward()
    assert torch.equal(x["log_decay"].grad, torch.zeros(3, device="cuda"))
    # sequences of length zero, with NaN in them
    x = {k: t.detach().new_full((2, 70, *t.shape[2:]), math.nan) for k, t in empty(2, 1).items() if k != "log_decay"}
    g = torch.full((2, 70, 3), math.nan, device="cuda")
    y, last = ops.linear_attention(**x, log_decay=g, state=s, lens=torch.zeros(2, dtype=torch.int32, device="cuda"), return_state=True)
    assert not y.any() and torch.equal(last, s)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides(gpu, dtype):
    """q, k and v as columns of one projection's rows, as [batch, heads, length, d], with gaps, at odd offsets, and not contiguous in
    the last dimension: the bits of contiguous ones."""
    n, length, heads, key, value = 2, 100, 3, 24, 40
    x, dy, _, _ = _inputs(n, length, heads, heads, key, value, dtype, "token", 10)
    gx = {k: t.cuda() for k, t in x.items()}

    def run(q, k, v, g, dy):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, g)]
        y = ops.linear_attention(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))

    want = run(*gx.values(), dy.cuda())
    rows = torch.cat([t.flatten(2) for t in (gx["q"], gx["k"], gx["v"])], 2)
    a, b = heads * key, 2 * heads * key
    ways = [(rows[..., :a].unflatten(2, (heads, key)), rows[..., a:b].unflatten(2, (heads, key)), rows[..., b:].unflatten(2, (heads, value)),
             gx["log_decay"], dy.cuda())]
    ways.append(tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (*gx.values(), dy.cuda())))
    ways.append(tuple(torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in (*gx.values(), dy.cuda())))
    ways.append(tuple(t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (*gx.values(), dy.cuda())))
    for way in ways:
        for w, got in zip(want, run(*way)):
            assert torch.equal(w, got)
    expanded = gx["log_decay"][:1, :1].expand(n, length, heads)
    for w, got in zip(run(*list(gx.values())[:3], expanded.contiguous(), dy.cuda()), run(*list(gx.values())[:3], expanded, dy.cuda())):
        assert torch.equal(w, got)


def test_offsets_beyond_32_bits(gpu):
    """Sequences 2^31 + 64 values apart (8.6 GB of bfloat16)."""
    apart = 2 ** 31 + 64
    buf = torch.empty(apart + 4096 * 3, dtype=BF, device="cuda")
    x, dy, _, _ = _inputs(2, 20, 2, 2, 8, 8, BF, "token", 11)
    gx = {k: t.cuda() for k, t in x.items()}
    want = ops.linear_attention(**gx)
    views = [torch.as_strided(buf, (2, 20, 2, 8), (apart, 16, 8, 1), 4096 * i) for i in range(3)]
    for view, name in zip(views, "qkv"):
        view.copy_(gx[name])
    leaves = [v.requires_grad_() for v in (torch.as_strided(buf, (2, 20, 2, 8), (apart, 16, 8, 1), 4096 * i) for i in range(3))]
    y = ops.linear_attention(*leaves, gx["log_decay"])
    assert torch.equal(y, want)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    gx = [t.requires_grad_() for t in list(gx.values())[:3]]
    for a, b in zip(got, torch.autograd.grad(ops.linear_attention(*gx, x["log_decay"].cuda()), gx, dy.cuda())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_a_number_reaches_only_what_comes_behind_it(gpu, bad, dtype):
    """Forward: a position's key, value or query reaches its own and later positions.  Backward: an upstream gradient reaches the
    gradients of its own and earlier positions' keys and values, and its own query's."""
    at = 37
    x, dy, _, _ = _inputs(2, 100, 2, 2, 20, 12, dtype, "token", 12)
    x, dy = {k: t.cuda() for k, t in x.items()}, dy.cuda()
    clean = ops.linear_attention(**x)
    for name in ("q", "k", "v"):
        y = dict(x, **{name: x[name].clone()})
        y[name][0, at, 1, 3] = bad
        got = ops.linear_attention(**y)
        assert torch.equal(got[:, :at], clean[:, :at]) and torch.equal(got[1], clean[1]) and torch.equal(got[0, :, 0], clean[0, :, 0])
        assert not torch.isfinite(got[0, at, 1]).all()
        if name == "q":
            assert torch.equal(got[0, at + 1:], clean[0, at + 1:])
        else:
            if name == "v":
                other = [c for c in range(12) if c != 3]
                assert torch.equal(got[..., other], clean[..., other])
            assert not torch.isfinite(got[0, at + 1, 1, 3])
    leaves = [t.requires_grad_() for t in x.values()]
    want = torch.autograd.grad(ops.linear_attention(*leaves), leaves, dy)
    dy = dy.clone()
    dy[0, at, 1, 3] = bad
    got = torch.autograd.grad(ops.linear_attention(*leaves), leaves, dy)
    for g, w, name in zip(got, want, x):
        assert torch.equal(g[1], w[1]) and torch.equal(g[0, :, 0], w[0, :, 0]), name
        assert not torch.isfinite(g[0, at, 1]).all(), name
        assert torch.equal(g[0, at + 1:], w[0, at + 1:]), name


def test_padding_may_hold_anything(gpu):
    x, dy, lens, _ = _inputs(3, 150, 2, 1, 30, 20, F32, "token", 13, ragged=True)
    lens[1] = 70

    def run(x, dy):
        leaves = [t.cuda().requires_grad_() for t in x.values()]
        y, s = ops.linear_attention(*leaves, lens=lens.cuda(), return_state=True)
        return (y, s, *torch.autograd.grad(y, leaves, dy.cuda()))

    want = run(x, dy)
    behind = torch.arange(150)[None] >= lens[:, None]
    for t in (*x.values(), dy):
        t[behind] = math.nan
    for a, b in zip(want, run(x, dy)):
        assert torch.equal(a, b)


def test_the_same_bits_again_on_another_stream_and_from_a_graph(gpu):
    x, dy, lens, s = _inputs(2, 400, 4, 2, 64, 64, BF, "token", 14, ragged=True, state=True)
    gx = [t.cuda().requires_grad_() for t in x.values()]
    dy, lens, s = dy.cuda(), lens.cuda(), s.cuda()
    one = [t[:, 0].detach() for t in gx]

    def run():
        y, last = ops.linear_attention(*gx, state=s, lens=lens, return_state=True)
        return [y.detach(), last, *torch.autograd.grad(y, gx, dy), ops.linear_attention_step(*one, state=s.clone())]

    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(want, run()):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run()
    for i in range(4):
        for t in out:
            t.zero_()
        with torch.no_grad():
            gx[2].mul_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        for a, b, w in zip(out, eager, want):
            assert torch.equal(a, b)
            assert i % 2 == 0 or torch.equal(a, w)


def test_two_streams_at_once(gpu):
    """Each call has workspaces of its own."""
    calls = []
    for seed in (20, 21):
        x, dy, _, _ = _inputs(1, 3000, 4, 4, 64, 64, F32, "token", seed)
        calls.append(([t.cuda().requires_grad_() for t in x.values()], dy.cuda()))

    def run(leaves, dy):
        y = ops.linear_attention(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = [run(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        got = []
        for c, st in zip(calls, streams):
            with torch.cuda.stream(st):
                got.append(run(*c))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradients_of_some_inputs_only(gpu):
    x, dy, _, _ = _inputs(1, 80, 2, 2, 8, 8, F32, "head", 15)
    gx = {k: t.cuda() for k, t in x.items()}
    leaves = [t.requires_grad_() for t in gx.values()]
    want = torch.autograd.grad(ops.linear_attention(*leaves), leaves, dy.cuda())
    for i, name in enumerate(gx):
        one = {k: t.detach() for k, t in gx.items()}
        one[name].requires_grad_()
        got, = torch.autograd.grad(ops.linear_attention(**one), [one[name]], dy.cuda())
        assert torch.equal(got, want[i])
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(ops.linear_attention(*leaves), leaves, dy.cuda(), create_graph=True)
