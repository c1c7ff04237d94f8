"""The training operators on the GPU against their formulas in 64 bits (ops_ref.py).

Tolerance of a value: half a step of its type relative to it (one rounding when it is stored), and N * 2^-24 of its magnitude
(the same sums over absolute values), N the number of float32 roundings on the longest way to it:
  layer norm   a row's sums add d / 64 values per lane and 6 times across lanes; two such sums and a dozen operations
  loss         the same, and exp's argument, whose rounding counts by its size (|x - m| log2 e)
  convolution  16 operations; sums over batch and positions add one rounding each
  scan         per position 6 roundings, and dt's (some 8 of them) in exp(dt A) by their size |dt A|; sums over channels,
               batch and positions add one each
"""
import math

import pytest
import torch

import ops_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAN = float("nan")


@pytest.fixture(scope="module")
def ops(gpu):
    from boa_amd import ops as o

    return o


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)


def _check(name, got, ref, n, dtype=None):
    value, mag = ref
    dtype = dtype or got.dtype
    assert got.shape == value.shape and got.dtype == dtype, (name, got.shape, value.shape, got.dtype)
    got = got.detach().to("cpu", torch.float64)
    nan = torch.isnan(value)
    assert torch.equal(torch.isnan(got), nan), f"{name}: NaN in other places"
    tol = torch.finfo(dtype).eps / 2 * value.abs() + n * 2.0 ** -24 * mag + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    over = ((got - value).abs() / tol)[~nan]
    assert over.numel() == 0 or over.max() <= 1, f"{name}: {float(over.max()):.3g} times the tolerance"


# ---- layer norm -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 17), (7, 63), (33, 64), (130, 100), (257, 256), (1000, 256), (63, 512),
                                    (9, 1000), (5, 1025), (4, 2048), (3, 2100), (2, 4096), (3, 4095)])
def test_norm(ops, rows, d, dtype):
    g = _gen(rows + d)
    x, w, b, dy = _randn(g, rows, d, dtype=dtype, scale=2, mean=0.5), _randn(g, d), _randn(g, d), _randn(g, rows, d, dtype=dtype)
    for t in (x, w, b):
        t.requires_grad_()
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b), y)
    ref = R.norm(x, w, b, dy)
    n = 4 * (d / 64 + 8) + 16
    _check("y", y, ref["y"], n, dtype)
    _check("dx", dx, ref["dx"], 2 * n, dtype)
    _check("dw", dw, ref["dw"], n + rows, torch.float32)
    _check("db", db, ref["db"], rows, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d,params", [(41, 384, 4), (41, 768, 4), (11, 1152, 4), (11, 1536, 4), (9, 2500, 4), (6, 4000, 4),
                                           (20011, 64, 4), (17001, 200, 4), (4501, 1152, 4), (2101, 2500, 4), (2101, 2501, 4),
                                           (50, 256, 1), (50, 512, 2), (9, 2048, 3)])
def test_norm_widths_loops_and_parameters_anywhere(ops, rows, d, params, dtype):
    """More widths, rows that take several steps of a workgroup, parameters that begin at any multiple of 4 bytes."""
    g = _gen(rows * d)
    x, dy = _randn(g, rows, d, dtype=dtype, scale=2, mean=0.5).requires_grad_(), _randn(g, rows, d, dtype=dtype)
    w, b = (_randn(g, d + 4)[params:][:d].detach().requires_grad_() for _ in range(2))
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ref = R.norm(x, w, b, dy)
    n = 4 * (d / 64 + 8) + 16
    _check("y", y, ref["y"], n, dtype)
    _check("dx", dx, ref["dx"], 2 * n, dtype)
    _check("dw", dw, ref["dw"], n + rows, torch.float32)
    _check("db", db, ref["db"], rows, torch.float32)


def test_norm_without_parameters_and_odd_layouts(ops):
    g = _gen(1)
    wide = _randn(g, 6, 5, 300)
    for x in (wide[..., :256], wide[..., 1:258], wide.transpose(0, 1)[..., 4:260], wide[..., ::2], wide[:, :1].expand(6, 5, 300)):
        x = x.detach().requires_grad_()
        d = x.shape[-1]
        y = ops.layer_norm(x)
        dy = _randn(g, 5, 6, d).transpose(0, 1) if y.shape[0] == 6 else _randn(g, *y.shape)
        dx, = torch.autograd.grad(y, (x,), dy)
        ref = R.norm(x.reshape(-1, d), None, None, dy.reshape(-1, d))
        n = 4 * (d / 64 + 8) + 16
        _check("y", y.reshape(-1, d), ref["y"], n)
        _check("dx", dx.reshape(-1, d), ref["dx"], 2 * n)
    w = _randn(g, 300).requires_grad_()
    dw, = torch.autograd.grad(ops.layer_norm(wide, w).sum(), (w,))  # an expanded upstream gradient
    _check("dw", dw, R.norm(wide.reshape(-1, 300), w, None, torch.ones(30, 300))["dw"], 4 * 13 + 16 + 30)
    assert ops.layer_norm(torch.empty(0, 8, device="cuda"), w[:8].detach()).shape == (0, 8)
    e = torch.empty(0, 300, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(ops.layer_norm(e, w).sum(), (e, w))
    assert gx.shape == (0, 300) and not gw.any()


def test_norm_rows_do_not_touch_each_other(ops):
    x = _randn(_gen(2), 9, 256)
    good = ops.layer_norm(x)
    x[4, 3] = NAN
    x[6, 0] = float("inf")
    y = ops.layer_norm(x)
    keep = [i for i in range(9) if i not in (4, 6)]
    assert torch.equal(y[keep], good[keep]) and y[4].isnan().all() and y[6].isnan().all()


# ---- cross entropy ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (9, 5), (65, 63), (300, 256), (1025, 256), (7, 257), (5, 1000), (3, 1024), (4, 2000),
                                    (2, 4096), (3, 4093)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss(ops, rows, v, dtype, reduction):
    g = _gen(rows + v)
    x = _randn(g, rows, v, dtype=dtype, scale=4).requires_grad_()
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    t[rows // 2:rows // 2 + rows // 4] = -100
    up = _randn(g, rows) if reduction == "none" else torch.tensor(3.0, device="cuda")
    y = ops.cross_entropy(x, t, reduction=reduction)
    dx, = torch.autograd.grad(y, (x,), up)
    ref = R.loss(x, t, -100, reduction, up.cpu().double())
    spread = float((x.detach().float().amax(1) - x.detach().float().amin(1)).max()) * 1.5
    n = v / 64 + 24 + 2 * spread
    _check("loss", y, ref["y"], n, torch.float32)
    _check("dx", dx, ref["dx"], n + 8, dtype)


def test_loss_targets(ops):
    g = _gen(3)
    x = _randn(g, 4, 3, 256, scale=3)
    t = torch.randint(0, 256, (4, 3), generator=g, device="cuda")
    want = ops.cross_entropy(x, t)
    assert torch.equal(ops.cross_entropy(x, t.to(torch.uint8)), want) and torch.equal(ops.cross_entropy(x, t.to(torch.int32)), want)
    assert ops.cross_entropy(x, t, reduction="none").shape == (4, 3)
    # no row counts: a mean over nothing, and no gradient
    x = x.reshape(12, 256).requires_grad_()
    none = torch.full((12,), -100, device="cuda")
    y = ops.cross_entropy(x, none)
    assert y.isnan() and not torch.autograd.grad(y, x)[0].any()
    assert ops.cross_entropy(x, none, reduction="sum") == 0
    # a target that is no symbol: NaN there, in its gradient and in the sums; the other rows as they were
    t = t.reshape(12)
    good = torch.autograd.grad(ops.cross_entropy(x, t, reduction="sum"), x)[0]
    t[3], t[5] = 256, -1
    y = ops.cross_entropy(x, t, reduction="none")
    dx, = torch.autograd.grad(y, x, torch.ones(12, device="cuda"))
    for i in range(12):
        assert bool(y[i].isnan()) == (i in (3, 5)) == bool(dx[i].isnan().all())
    keep = [i for i in range(12) if i not in (3, 5)]
    assert torch.equal(dx[keep], good[keep])
    assert ops.cross_entropy(x, t, ignore_index=-1).isnan() and ops.cross_entropy(x[:3], t[:3], ignore_index=-1).isfinite()
    e = torch.empty(0, 5, device="cuda")
    assert ops.cross_entropy(e, none[:0]).isnan() and ops.cross_entropy(e, none[:0], reduction="none").shape == (0,)


def test_loss_extreme_logits(ops):
    inf = float("inf")
    x = torch.zeros(6, 70, device="cuda")
    x[0, 1:] = -inf                               # one symbol allowed
    x[1, 3] = torch.finfo(torch.float32).min      # a mask of the type's lowest value
    x[2] = 1e30
    x[3] = -inf                                   # nothing allowed
    x[4, 7] = NAN
    x[5, 7] = inf
    t = torch.zeros(6, dtype=torch.int64, device="cuda")
    want = torch.nn.functional.cross_entropy(x.cpu().double(), t.cpu(), reduction="none")
    got = ops.cross_entropy(x, t, reduction="none").cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.allclose(got[:3], want[:3], rtol=1e-6)
    x.requires_grad_()
    dx, = torch.autograd.grad(ops.cross_entropy(x, t, reduction="none"), x, torch.ones(6, device="cuda"))
    xc = x.detach().cpu().double().requires_grad_()
    dw, = torch.autograd.grad(torch.nn.functional.cross_entropy(xc, t.cpu(), reduction="none"), xc, torch.ones(6).double())
    assert torch.allclose(dx[:3].cpu().double(), dw[:3], rtol=1e-5, atol=1e-7) and dx[3:].isnan().any(1).all()


def test_loss_strided_rows(ops):
    g = _gen(4)
    wide = _randn(g, 20, 600, scale=3)
    t = torch.randint(0, 200, (20,), generator=g, device="cuda")
    for x in (wide[:, :200], wide[:, 3:203], wide[:, 0:400:2], wide[:1, 8:208].expand(20, 200)):
        x = x.detach().requires_grad_()
        y = ops.cross_entropy(x, t)
        dx, = torch.autograd.grad(y, x)
        ref = R.loss(x, t, -100, "mean", 1.0)
        _check("loss", y, ref["y"], 80)
        _check("dx", dx, ref["dx"], 90)


# ---- convolution ------------------------------------------------------------------------------------
CONV = [(1, 1, 1), (2, 2, 3), (3, 3, 4), (2, 16, 64), (2, 17, 65), (3, 15, 256), (1, 50, 260), (4, 33, 512), (2, 100, 1024), (1, 400, 7)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,length,c", CONV)
@pytest.mark.parametrize("ragged", [False, True])
def test_conv(ops, n, length, c, dtype, ragged):
    g = _gen(n + length + c)
    x, w, b, dy = _randn(g, n, length, c, dtype=dtype), _randn(g, c, 1, 4, scale=0.5), _randn(g, c), _randn(g, n, length, c, dtype=dtype)
    state = _randn(g, n, 3, c, dtype=dtype) if ragged else None
    lens = torch.tensor([(length, 0, 1, length // 2)[i % 4] for i in range(n)], dtype=torch.int32, device="cuda") if ragged else None
    for t in (x, w, b):
        t.requires_grad_()
    y, end = ops.causal_conv(x, w, b, state=state, lens=lens, return_state=True)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        assert torch.equal(ops.causal_conv(x, w, b, state=state, lens=lens), y)
    ref = R.conv(x, w, b, True, state, lens, dy)
    _check("y", y, ref["y"], 16, dtype)
    _check("state", end, ref["state"], 0, dtype)
    _check("dx", dx, ref["dx"], 32, dtype)
    _check("dw", dw[:, 0], ref["dw"], 32 + n * length, torch.float32)
    _check("db", db, ref["db"], 32 + n * length, torch.float32)


def test_conv_without_silu_bias_and_of_no_positions(ops):
    g = _gen(5)
    x, w, dy = _randn(g, 2, 9, 12).requires_grad_(), _randn(g, 12, 4).requires_grad_(), _randn(g, 2, 9, 12)
    y = ops.causal_conv(x, w, silu=False)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ref = R.conv(x, w, None, False, None, None, dy)
    for k, v, n in (("y", y, 16), ("dx", dx, 32), ("dw", dw, 50)):
        _check(k, v, ref[k], n)
    st = _randn(g, 2, 3, 12)
    y, end = ops.causal_conv(x[:, :0].detach(), w.detach(), state=st, return_state=True)
    assert y.shape == (2, 0, 12) and torch.equal(end, st)
    e = x[:, :0].detach().requires_grad_()
    dx, dw = torch.autograd.grad(ops.causal_conv(e, w).sum(), (e, w))
    assert dx.shape == (2, 0, 12) and not dw.any()
    assert ops.causal_conv(x[:0].detach(), w.detach()).shape == (0, 9, 12)


def test_conv_padding_is_not_read(ops):
    g = _gen(6)
    x, w, b, dy = _randn(g, 3, 40, 64), _randn(g, 64, 4).requires_grad_(), _randn(g, 64).requires_grad_(), _randn(g, 3, 40, 64)
    lens = torch.tensor([40, 13, 0], dtype=torch.int32, device="cuda")
    got = []
    for fill in (0.0, NAN):
        for i, n in enumerate(lens.tolist()):
            x[i, n:], dy[i, n:] = fill, fill
        xx = x.clone().requires_grad_()
        y, end = ops.causal_conv(xx, w, b, lens=lens, return_state=True)
        got.append([y, end, *torch.autograd.grad(y, (xx, w, b), dy)])
    assert all(torch.equal(p, q) for p, q in zip(*got))
    assert not got[1][0][1, 13:].any() and not got[1][0][2].any() and not got[1][2][1, 13:].any()
    long = torch.tensor([99, -4, 0], dtype=torch.int32, device="cuda")  # clamped to [0, length]
    x[0] = 1.0
    assert torch.equal(ops.causal_conv(x, w.detach(), lens=long), ops.causal_conv(x, w.detach(), lens=long.clamp(0, 40)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_conv_strided(ops, dtype):
    g = _gen(7)
    wide = _randn(g, 5, 30, 200, dtype=dtype)
    w, b = _randn(g, 96, 4), _randn(g, 96)
    for x in (wide[:, :, :96], wide[:, :, 3:99], wide[:, ::2, 100:196], wide.transpose(0, 1)[:, :, :96], wide[:1, :, :96].expand(5, 30, 96),
              wide[:, :1, :96].expand(5, 30, 96), wide[:, :, ::2][:, :, :96]):
        want = ops.causal_conv(x.contiguous(), w, b)
        assert torch.equal(ops.causal_conv(x, w, b), want)
        xs, xc = x.detach().requires_grad_(), x.contiguous().detach().requires_grad_()
        dy = _randn(g, x.shape[1], x.shape[0], 96, dtype=dtype).transpose(0, 1)
        ds, = torch.autograd.grad(ops.causal_conv(xs, w, b), xs, dy)
        dc, = torch.autograd.grad(ops.causal_conv(xc, w, b), xc, dy.contiguous())
        assert torch.equal(ds, dc)
    v = _randn(g, 1, 30, 96, dtype=dtype).requires_grad_()  # a broadcast input: its gradient is the sum over the copies
    dy = _randn(g, 5, 30, 96, dtype=dtype)
    dv, = torch.autograd.grad(ops.causal_conv(v.expand(5, 30, 96), w, b), v, dy)
    full = R.conv(v.detach().expand(5, 30, 96), w, b, True, None, None, dy)["dx"]
    eps = torch.finfo(dtype).eps / 2
    tol = 6 * eps * full[1].sum(0, keepdim=True) + 40 * 2.0 ** -24 * full[1].sum(0, keepdim=True)  # five roundings, then the sum's
    assert ((dv.cpu().double() - full[0].sum(0, keepdim=True)).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (3, 5), (2, 64), (64, 512), (1000, 130)])
def test_conv_step_is_the_prompts(ops, n, c, dtype):
    """Steps give the bits that the prompt form gives, and leave its state."""
    g = _gen(n + c)
    x, w, b, state = _randn(g, n, 6, c, dtype=dtype), _randn(g, c, 1, 4), _randn(g, c), _randn(g, n, 3, c, dtype=dtype)
    want, end = ops.causal_conv(x, w, b, state=state, return_state=True)
    st = state.clone()
    for t in range(6):
        assert torch.equal(ops.causal_conv_step(x[:, t], st, w, b), want[:, t])
    assert torch.equal(st, end)
    assert torch.equal(ops.causal_conv_step(x[:, 0], state.clone(), w, b, silu=False),
                       ops.causal_conv(x[:, :1], w, b, silu=False, state=state)[:, 0])


# ---- scan -------------------------------------------------------------------------------------------
def _scan_inputs(g, n, length, c, dtype, gate=True, params=True, wide=False):
    rank = -(-c // 32)
    dbc = _randn(g, n, length, rank + 32, dtype=dtype)
    s = {"u": _randn(g, n, length, c, dtype=dtype), "delta": _randn(g, n, length, c, dtype=dtype, scale=0.5),
         "A": -torch.exp(_randn(g, c, 16, scale=0.1)) * torch.arange(1, 17, device="cuda"), "B": dbc[..., rank:rank + 16],
         "C": dbc[..., rank + 16:], "D": None, "z": None, "delta_bias": None}
    if params:
        s["D"], s["delta_bias"] = _randn(g, c), _randn(g, c, mean=-2.0)
    if gate:
        s["z"] = _randn(g, n, length, 2 * c if wide else c, dtype=dtype)[..., :c]
    return s


NAMES = {"u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "delta_bias": "dbias"}


def _ref(s, **kw):
    return R.scan(*(s[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")), **kw)


def _roundings(s):
    n, length, c = s["u"].shape
    bias = 0 if s["delta_bias"] is None else s["delta_bias"]
    most = float((torch.nn.functional.softplus(s["delta"].float() + bias).amax((0, 1))[:, None] * -s["A"]).detach().max()) if length else 0
    return 64 + c + n * length + length * (6 + 10 * most)


SCAN = [(1, 1, 1), (2, 2, 3), (2, 7, 5), (3, 8, 64), (2, 9, 65), (1, 40, 130), (2, 100, 33), (1, 129, 64), (1, 700, 70), (4, 65, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,length,c", SCAN)
def test_scan(ops, n, length, c, dtype):
    g = _gen(n + length + c)
    s = {k: v.detach().requires_grad_() for k, v in _scan_inputs(g, n, length, c, dtype, wide=c % 2 == 0).items()}
    dy = _randn(g, n, length, c, dtype=dtype)
    y, end = ops.selective_scan(**s, return_state=True)
    grads = torch.autograd.grad(y, tuple(s.values()), dy)
    with torch.no_grad():
        assert torch.equal(ops.selective_scan(**s), y)  # with and without what the gradient needs
    ref, k = _ref(s, dy=dy), _roundings(s)
    _check("y", y, ref["y"], k, dtype)
    _check("state", end, ref["state"], k, torch.float32)
    for name, got in zip(s, grads):
        _check(NAMES[name], got, ref[NAMES[name]], 2 * k, s[name].dtype)


@pytest.mark.parametrize("gate,params", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("n,length,c,ends", [(4, 30, 70, (30, 0, 1, 17)), (3, 200, 64, (8, 200, 129)), (1, 300, 40, (265,)), (2, 16, 8, (0, 0))])
def test_scan_of_padded_batches_from_a_state(ops, n, length, c, ends, gate, params):
    g = _gen(length)
    s = {k: None if v is None else v.detach().requires_grad_() for k, v in
         _scan_inputs(g, n, length, c, torch.float32, gate, params).items()}
    state, dy = _randn(g, n, 16, c), _randn(g, n, length, c)
    lens = torch.tensor(ends, dtype=torch.int32, device="cuda")
    y, end = ops.selective_scan(**s, state=state, lens=lens, return_state=True)
    leaves = {k: v for k, v in s.items() if v is not None}
    grads = torch.autograd.grad(y, tuple(leaves.values()), dy)
    ref, k = _ref(s, state=state, lens=lens, dy=dy), _roundings(s)
    _check("y", y, ref["y"], k)
    _check("state", end, ref["state"], k)
    for name, got in zip(leaves, grads):
        _check(NAMES[name], got, ref[NAMES[name]], 2 * k)
    for i, e in enumerate(ends):
        assert not y[i, e:].any() and not grads[0][i, e:].any()
        if e == 0:
            assert torch.equal(end[i], state[i])


@pytest.mark.parametrize("n,length,c,ends", [(1, 2300, 40, None), (2, 2500, 8, (2500, 130)), (3, 2200, 5, (0, 64, 2199))])
def test_scan_of_many_chunks(ops, n, length, c, ends):
    """Lengths that are split into more chunks than a workgroup goes over by itself (33 and more of 64 positions)."""
    g = _gen(length)
    s = {k: v.detach().requires_grad_() for k, v in _scan_inputs(g, n, length, c, torch.float32).items()}
    state, dy = _randn(g, n, 16, c), _randn(g, n, length, c)
    lens = None if ends is None else torch.tensor(ends, dtype=torch.int32, device="cuda")
    y, end = ops.selective_scan(**s, state=state, lens=lens, return_state=True)
    grads = torch.autograd.grad(y, tuple(s.values()), dy)
    ref, k = _ref(s, state=state, lens=lens, dy=dy), _roundings(s)
    # in these units an error at a chunk's border is one of size 1; a state is forgotten within some hundred positions, so no
    # more than 500 positions' roundings add up
    k = k * 500 / length
    _check("y", y, ref["y"], k)
    _check("state", end, ref["state"], k)
    for name, got in zip(s, grads):
        _check(NAMES[name], got, ref[NAMES[name]], 2 * k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_padding_is_not_read(ops, dtype):
    g = _gen(8)
    n, length, c = 4, 150, 70
    s, dy = _scan_inputs(g, n, length, c, dtype), _randn(g, n, length, c, dtype=dtype)
    lens = torch.tensor([150, 77, 8, 0], dtype=torch.int32, device="cuda")
    got = []
    for fill in (0.0, NAN):
        for k in ("u", "delta", "B", "C", "z"):
            for i, e in enumerate(lens.tolist()):
                s[k][i, e:] = fill
        for i, e in enumerate(lens.tolist()):
            dy[i, e:] = fill
        leaf = {k: v.detach().requires_grad_() for k, v in s.items()}
        y, end = ops.selective_scan(**leaf, lens=lens, return_state=True)
        got.append([y, end, *torch.autograd.grad(y, tuple(leaf.values()), dy)])
    assert all(torch.equal(p, q) for p, q in zip(*got)) and all(bool(t.isfinite().all()) for t in got[1])
    s = _scan_inputs(g, 3, 20, c, dtype)
    odd = torch.tensor([99, -1, 20], dtype=torch.int32, device="cuda")  # clamped to [0, length]
    assert torch.equal(ops.selective_scan(**s, lens=odd), ops.selective_scan(**s, lens=odd.clamp(0, 20).long()))


def test_scan_sequences_do_not_touch_each_other(ops):
    g = _gen(9)
    s = _scan_inputs(g, 3, 90, 70, torch.float32)
    good = ops.selective_scan(**s)
    s["u"][1, 40, 5] = NAN
    y = ops.selective_scan(**s)
    assert torch.equal(y[[0, 2]], good[[0, 2]]) and torch.equal(y[1, :40], good[1, :40]) and y[1, 40:, 5].isnan().all()
    keep = [c for c in range(70) if c != 5]
    assert torch.equal(y[1][:, keep], good[1][:, keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_strided(ops, dtype):
    """Odd row offsets, transposed batches, broadcast rows: the bits of contiguous inputs."""
    g = _gen(10)
    n, length, c = 5, 70, 96
    wide = _randn(g, n, length, 4 * c, dtype=dtype)
    base = _scan_inputs(g, n, length, c, dtype)
    views = {"u": wide[..., 1:c + 1], "delta": wide[..., c:2 * c], "z": wide[..., 2 * c + 3:3 * c + 3]}
    turned = _randn(g, length, n, c, dtype=dtype).transpose(0, 1)
    for change in (views, {"u": turned, "z": turned}, {"B": wide[..., 3:19], "C": wide[..., 20:36]},
                   {"B": wide[:, :1, :16].expand(n, length, 16), "u": wide[:1, :, :c].expand(n, length, c)},
                   {"B": wide[..., 0:32:2], "delta": wide[..., ::4]}):
        s = {**base, **change}
        dy = _randn(g, length, n, c, dtype=dtype).transpose(0, 1)
        got = []
        for make in (lambda v: v.detach(), lambda v: v.contiguous().detach()):
            leaf = {k: make(v).requires_grad_() for k, v in s.items()}
            y = ops.selective_scan(**leaf)
            got.append([y, *torch.autograd.grad(y, tuple(leaf.values()), dy)])
        assert all(torch.equal(p, q) for p, q in zip(*got))


def test_scan_continues(ops):
    """A sequence in two parts, the state handed on, is the sequence in one."""
    g = _gen(11)
    n, length, c = 2, 203, 70
    s = _scan_inputs(g, n, length, c, torch.float32)
    want, end = ops.selective_scan(**s, return_state=True)
    ref, k = _ref(s), _roundings(s)
    for at in (1, 64, 100, 202):
        part = lambda lo, hi: {key: v[:, lo:hi] if key in ("u", "delta", "B", "C", "z") else v for key, v in s.items()}  # noqa: E731
        y0, st = ops.selective_scan(**part(0, at), return_state=True)
        y1, st = ops.selective_scan(**part(at, length), state=st, return_state=True)
        _check("y", torch.cat([y0, y1], 1), ref["y"], k)
        _check("state", st, ref["state"], k)
    y, st = ops.selective_scan(**part(0, 0), state=end, return_state=True)
    assert y.shape == (n, 0, c) and torch.equal(st, end)
    y, st = ops.selective_scan(**part(0, 0), return_state=True)
    assert not st.any()


def test_scan_of_nothing(ops):
    g = _gen(12)
    for n, length in ((0, 5), (2, 0)):
        s = {k: v.detach().requires_grad_() for k, v in _scan_inputs(g, n, length, 8, torch.float32).items()}
        y = ops.selective_scan(**s)
        grads = torch.autograd.grad(y.sum(), tuple(s.values()))
        assert y.shape == (n, length, 8) and all(not v.any() and v.shape == w.shape for v, w in zip(grads, s.values()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (3, 5), (1, 512), (2, 130), (300, 65), (64, 1024)])
def test_scan_step(ops, n, c, dtype):
    g = _gen(n + c)
    s, state = _scan_inputs(g, n, 3, c, dtype), _randn(g, n, 16, c)
    ref, k, st = _ref(s, state=state), _roundings(s), state.clone()
    for t in range(3):
        at = {key: v[:, t] if key in ("u", "delta", "B", "C", "z") else v for key, v in s.items()}
        y = ops.selective_scan_step(**at, state=st)
        _check("y", y, (ref["y"][0][:, t], ref["y"][1][:, t]), k, dtype)
    _check("state", st, ref["state"], k, torch.float32)
    bare = {key: v[:, 0] if key in ("u", "delta", "B", "C") else v for key, v in s.items() if key in ("u", "delta", "A", "B", "C")}
    st = state.clone()
    y = ops.selective_scan_step(**bare, state=st)
    want, end = ops.selective_scan(**{key: v[:, None] if key != "A" else v for key, v in bare.items()}, state=state, return_state=True)
    assert torch.allclose(y.float(), want[:, 0].float(), rtol=2e-2 if dtype != torch.float32 else 1e-5, atol=1e-5)
    assert torch.allclose(st, end, rtol=1e-5, atol=1e-6)


def test_scan_extreme_steps(ops):
    """Steps so long that a state is forgotten at once, and so short that nothing moves."""
    g = _gen(13)
    s = _scan_inputs(g, 2, 80, 64, torch.float32)
    s["delta"][:, ::3] = 60.0
    s["delta"][:, 1::3] = -120.0
    leaf = {k: v.detach().requires_grad_() for k, v in s.items()}
    dy = _randn(g, 2, 80, 64)
    y, end = ops.selective_scan(**leaf, return_state=True)
    grads = torch.autograd.grad(y, tuple(leaf.values()), dy)
    assert y.isfinite().all() and end.isfinite().all() and all(v.isfinite().all() for v in grads)
    ref = _ref(s, dy=dy)
    # dt A reaches 60 * 20: its rounding in the exponent counts by e^-x x, below 0.37 per unit of dt's relative error
    _check("y", y, ref["y"], 80 * 32 + 200)
    _check("state", end, ref["state"], 80 * 32 + 200)


# ---- all of them ------------------------------------------------------------------------------------
def _passes(ops, g, dtype=torch.float32):
    """A pass through every operator as a closure that returns all outputs and gradients, its leaves, and new inputs for it."""
    n, length, c, v = 3, 150, 70, 256
    s = {k: t.detach().requires_grad_() for k, t in _scan_inputs(g, n, length, c, dtype).items()}
    x, w4, b = (_randn(g, n, length, c, dtype=dtype).requires_grad_(), _randn(g, c, 4).requires_grad_(), _randn(g, c).requires_grad_())
    logits = _randn(g, n * length, v, dtype=dtype).requires_grad_()
    t = torch.randint(0, v, (n * length,), generator=g, device="cuda")
    lens = torch.tensor([150, 20, 99], dtype=torch.int32, device="cuda")
    dy = _randn(g, n, length, c, dtype=dtype)
    conv_state, ssm_state = _randn(g, n, 3, c, dtype=dtype), _randn(g, n, 16, c)

    def run():
        out = []
        y = ops.layer_norm(x, w4[:, 0].contiguous(), b)
        out += [y, *torch.autograd.grad(y, (x, w4, b), dy)]
        y, st = ops.causal_conv(x, w4, b, lens=lens, state=conv_state, return_state=True)
        out += [y, st, *torch.autograd.grad(y, (x, w4, b), dy)]
        y, st = ops.selective_scan(**s, lens=lens, state=ssm_state, return_state=True)
        out += [y, st, *torch.autograd.grad(y, tuple(s.values()), dy)]
        y = ops.cross_entropy(logits, t)
        out += [y, *torch.autograd.grad(y, (logits,))]
        with torch.no_grad():
            cs, ss = conv_state.clone(), ssm_state.clone()
            out += [ops.causal_conv_step(x[:, 0], cs, w4, b), cs]
            at = {k: p[:, 0] if k in ("u", "delta", "B", "C", "z") else p for k, p in s.items()}
            out += [ops.selective_scan_step(**at, state=ss), ss]
        return [p.detach() for p in out]

    def renew(seed):
        h = _gen(seed)
        with torch.no_grad():
            for p in (x, logits, s["u"], s["delta"], s["B"], s["C"], s["z"], dy, ssm_state):
                p.copy_(torch.randn(p.shape, generator=h, device="cuda"))

    return run, renew


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_inputs_same_bits(ops, dtype):
    run, _ = _passes(ops, _gen(14), dtype)
    first = run()
    junk = [torch.full((1 << 20,), NAN, device="cuda") for _ in range(8)]  # workspaces come out of dirty memory next
    del junk
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, run()))


def test_on_another_stream(ops):
    run, renew = _passes(ops, _gen(15))
    renew(1)
    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [run() for _ in range(3)]
    s.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(want, g))


def test_two_streams_at_once(ops):
    a, _ = _passes(ops, _gen(16))
    b, _ = _passes(ops, _gen(17))
    want = a(), b()
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = [], []
    for _ in range(4):
        for k, (stream, run) in enumerate(((s, a), (t, b))):
            with torch.cuda.stream(stream):
                got[k].append(run())
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(want[k], g))


def test_captured_passes(ops):
    """Two graphs of all operators, captured one after the other, replayed in turn on changing inputs with eager work between."""
    passes = [_passes(ops, _gen(18)), _passes(ops, _gen(19))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for run, _ in passes:
            run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for run, _ in passes:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for k in range(4):
        for (graph, out), (run, renew) in zip(graphs, passes):
            renew(100 + k)
            want = run()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(want, out)), k


def test_offsets_beyond_32_bits(ops):
    """Rows whose element offsets pass 2^31 and 2^32: a buffer of 2^32 + 2^30 bfloat16 values with a few rows at its ends."""
    big = torch.empty((5 << 30,), dtype=torch.bfloat16, device="cuda")
    c, far = 256, (5 << 30) - 256 * 12
    rows = torch.as_strided(big, (2, 12, c), (far, c, 1))
    g = _gen(20)
    x = _randn(g, 2, 12, c, dtype=torch.bfloat16)
    rows.copy_(x)
    w, b = _randn(g, c, 4), _randn(g, c)
    for a, q in ((rows, x),):
        y, st = ops.causal_conv(a, w, b, return_state=True)
        y2, st2 = ops.causal_conv(q, w, b, return_state=True)
        assert torch.equal(y, y2) and torch.equal(st, st2)
        s = _scan_inputs(g, 2, 12, c, torch.bfloat16)
        far_bc = torch.as_strided(big, (2, 12, 16), (far, c, 1), 0)
        got = []
        for u, bc in ((a, far_bc), (q, x[..., :16].contiguous())):
            leaf = {**s, "u": u, "delta": u, "z": u, "B": bc, "C": bc}
            leaf = {k: v.detach().requires_grad_() for k, v in leaf.items()}
            y = ops.selective_scan(**leaf)
            got.append([y, *torch.autograd.grad(y, tuple(leaf.values()), torch.ones_like(y))])
        assert all(torch.equal(p, r) for p, r in zip(*got))
    flat = torch.as_strided(big, (3, c), (far // 2, 1))
    flat.copy_(_randn(g, 3, c, dtype=torch.bfloat16))
    assert torch.equal(ops.layer_norm(flat), ops.layer_norm(flat.contiguous()))
    t = torch.tensor([0, 5, 255], device="cuda")
    assert torch.equal(ops.cross_entropy(flat, t), ops.cross_entropy(flat.contiguous(), t))


def test_scan_rows_as_far_apart_as_they_may_be(ops):
    """Rows at the largest stride: a block of 16 spans almost 4 GiB, two chunks 27 GB; the bits of contiguous inputs."""
    from boa_amd import _native

    g = _gen(23)
    length, c, far = 100, 64, _native.BOA_SCAN_MAX_ROW_STRIDE
    big = torch.empty((length - 1) * far + 256, device="cuda")
    s = {k: v.detach() for k, v in _scan_inputs(g, 1, length, c, torch.float32).items()}
    state, dy = _randn(g, 1, 16, c), _randn(g, 1, length, c)
    near, spread, at = dict(s), dict(s), 0
    for k in ("u", "delta", "B", "C"):
        spread[k] = torch.as_strided(big, near[k].shape, (far, far, 1), at)
        spread[k].copy_(near[k])
        at += near[k].shape[-1]
    got = []
    for t in (near, spread):
        leaf = {k: v.requires_grad_() for k, v in t.items()}
        y, end = ops.selective_scan(**leaf, state=state, return_state=True)
        got.append([y, end, *torch.autograd.grad(y, tuple(leaf.values()), dy)])
    assert all(torch.equal(p, q) for p, q in zip(*got))
    del big, spread, leaf, got, t, y
    torch.cuda.empty_cache()


def test_differentiable_once(ops):
    x = _randn(_gen(22), 4, 64).requires_grad_()
    g, = torch.autograd.grad(ops.layer_norm(x).square().sum(), x, retain_graph=True)
    assert g.isfinite().all() and not g.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(ops.layer_norm(x).square().sum(), x, create_graph=True)


def test_lengths_of_64_bits(ops):
    """Lengths beyond 32 bits are clamped, not cut."""
    g = _gen(23)
    x, w = _randn(g, 3, 20, 64), _randn(g, 64, 4)
    lens = torch.tensor([1 << 32, (1 << 32) + 7, -(1 << 33)], device="cuda")
    assert torch.equal(ops.causal_conv(x, w, lens=lens), ops.causal_conv(x, w, lens=lens.clamp(0, 20)))
    s = _scan_inputs(g, 3, 20, 64, torch.float32)
    assert torch.equal(ops.selective_scan(**s, lens=lens), ops.selective_scan(**s, lens=lens.clamp(0, 20).int()))


def test_saved_inputs_are_watched(ops):
    """An input changed in place between the passes is an error, as everywhere in torch, never a wrong gradient."""
    g = _gen(21)
    x, w = _randn(g, 2, 9, 64).requires_grad_(), _randn(g, 64, 4).requires_grad_()
    u = x * 1.0
    y = ops.causal_conv(u, w)
    u.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = ops.cross_entropy(x.reshape(-1, 64) * 1.0, torch.zeros(18, dtype=torch.int64, device="cuda"))
    y /= 2
    y.backward()  # the loss itself may be
    assert x.grad.isfinite().all() and math.isfinite(float(y.detach()))


def test_saved_states_are_watched(ops):
    """So is a state that a single-token step has advanced since a backward pass was to read it."""
    g = _gen(22)
    x, w, state = _randn(g, 2, 9, 64).requires_grad_(), _randn(g, 64, 4), _randn(g, 2, 3, 64)
    y = ops.causal_conv(x, w, state=state)
    with torch.no_grad():
        ops.causal_conv_step(x[:, 0], state, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():  # states without a counter
        a, b = torch.zeros(2, 3, 64, device="cuda"), torch.zeros(2, 16, 64, device="cuda")
        ops.causal_conv_step(x[:, 0], a, w)
        B = x[:, 0, :16]
        ops.selective_scan_step(x[:, 0], x[:, 1], -torch.ones(64, 16, device="cuda"), B, B, state=b)
        assert a.abs().sum() > 0 and b.abs().sum() > 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_are_each_as_alone(ops, dtype):
    """More rows, runs and sequences than the workgroups take in one step: the bits of smaller calls."""
    g = _gen(24)
    x = _randn(g, 140003, 40, dtype=dtype, scale=3).requires_grad_()
    t = torch.randint(0, 40, (140003,), generator=g, device="cuda", dtype=torch.uint8)
    up = _randn(g, 140003)
    y = ops.cross_entropy(x, t, reduction="none")
    dx, = torch.autograd.grad(y, (x,), up)
    for at in range(0, 140003, 50000):
        part = x.detach()[at:at + 50000].requires_grad_()
        z = ops.cross_entropy(part, t[at:at + 50000], reduction="none")
        assert torch.equal(z, y[at:at + 50000])
        assert torch.equal(torch.autograd.grad(z, (part,), up[at:at + 50000])[0], dx[at:at + 50000])
    mean = ops.cross_entropy(x.detach(), t)
    # summed in 64 bits, rounded once
    assert abs(float(mean) - float(y.detach().double().mean())) <= (2.0 ** -24 + 2.0 ** -34) * float(mean)

    for c, n, length in ((3, 150001, 2), (8, 9001, 17)):
        w, b = _randn(g, c, 4), _randn(g, c)
        x, dy = _randn(g, n, length, c, dtype=dtype).requires_grad_(), _randn(g, n, length, c, dtype=dtype)
        y = ops.causal_conv(x, w, b)
        dx, = torch.autograd.grad(y, (x,), dy)
        for at in range(0, n, 70000):
            part = x.detach()[at:at + 70000].requires_grad_()
            z = ops.causal_conv(part, w, b)
            assert torch.equal(z, y[at:at + 70000])
            assert torch.equal(torch.autograd.grad(z, (part,), dy[at:at + 70000])[0], dx[at:at + 70000])

    n, c = 20001, 70
    act = [_randn(g, n, c, dtype=dtype) for _ in range(3)] + [_randn(g, n, 16, dtype=dtype) for _ in range(2)]
    A, D, bias, state = -torch.rand(c, 16, device="cuda") * 16, _randn(g, c), _randn(g, c), _randn(g, n, 16, c)
    st = state.clone()
    y = ops.selective_scan_step(act[0], act[1], A, act[3], act[4], D, act[2], bias, state=st)
    for at in range(0, n, 6000):
        u, delta, z, B, C = (v[at:at + 6000] for v in act)
        s = state[at:at + 6000].clone()
        assert torch.equal(ops.selective_scan_step(u, delta, A, B, C, D, z, bias, state=s), y[at:at + 6000])
        assert torch.equal(s, st[at:at + 6000])


def test_scan_of_the_most_channels(ops):
    """65536 channels: each as in a call of its own; dB and dC, here of terms without signs, are the sums over the calls."""
    g = _gen(25)
    n, length, c, step = 1, 60, 65536, 4096 + 64  # 60 positions: never split
    s = {k: v if v is None else (v.abs() if k in "uBC" else v).detach().requires_grad_()
         for k, v in _scan_inputs(g, n, length, c, torch.float32, gate=False).items()}
    s.pop("z")
    dy = _randn(g, n, length, c).abs()
    y, end = ops.selective_scan(**s, return_state=True)
    got = dict(zip(s, torch.autograd.grad(y, tuple(s.values()), dy)))
    sums = {k: torch.zeros(n, length, 16, dtype=torch.float64, device="cuda") for k in "BC"}
    for at in range(0, c, step):
        cut = slice(at, min(at + step, c))
        part = {k: (v if k in "BC" else v[cut] if k in ("A", "D", "delta_bias") else v[..., cut]).detach().requires_grad_()
                for k, v in s.items()}
        z, e = ops.selective_scan(**part, return_state=True)
        assert torch.equal(z, y[..., cut]) and torch.equal(e, end[..., cut])
        for k, v in zip(part, torch.autograd.grad(z, tuple(part.values()), dy[..., cut])):
            if k in "BC":
                sums[k] += v.double()
            else:
                assert torch.equal(v, got[k][cut] if k in ("A", "D", "delta_bias") else got[k][..., cut])
    for k in "BC":  # a butterfly over 64 channels, then 1024 or 65 blocks of them one after another, in 32 bits
        assert ((got[k].double() - sums[k]).abs() <= (6 + 1024 + 6 + 65) * 2.0 ** -24 * sums[k]).all()
