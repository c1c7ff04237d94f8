"""The training pass under autocast: its gradients' errors against those of the same pass in elementary operations, what the second layer
norm does to 16-bit rows, and steps between passes."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from test_gpu_train import _loss64, _model

pytestmark = pytest.mark.gpu


def _plain_loss(m, x, dtype):
    """BoaBytePredictor.loss in elementary operations in float32, rounded where the operators round: their outputs, in 16 bits."""
    inp, tgt = x[:, :-1], x[:, 1:]
    h = F.embedding(inp, m.embedding.weight)
    T = inp.shape[1]
    for block in m.blocks:
        mx, w = block.mamba, block.mamba.in_proj.weight
        a = F.layer_norm(h, h.shape[-1:], block.ln1.weight, block.ln1.bias)
        u, z = F.linear(a, w[:mx.d_inner]), F.linear(a, w[mx.d_inner:])
        past = F.pad(u.float(), (0, 0, 3, 0))
        u = F.silu(sum(past[:, k:k + T] * mx.conv1d.weight[:, 0, k] for k in range(4)) + mx.conv1d.bias).to(dtype)
        dr, B, C = mx.x_proj(u).split([mx.dt_rank, 16, 16], -1)
        dt = F.softplus(F.linear(dr, mx.dt_proj.weight).float() + mx.dt_proj.bias)
        A, B, C, uf = -torch.exp(mx.A_log), B.float(), C.float(), u.float()
        s, ys = torch.zeros(len(x), mx.d_inner, 16, device=x.device), []
        for t in range(T):
            s = torch.exp(dt[:, t, :, None] * A) * s + (dt[:, t] * uf[:, t])[..., None] * B[:, t, None]
            ys.append((s * C[:, t, None]).sum(2) + mx.D * uf[:, t])
        y = mx.out_proj((torch.stack(ys, 1) * F.silu(z.float())).to(dtype))
        h = h + block.ff(F.layer_norm(y, y.shape[-1:], block.ln2.weight, block.ln2.bias))
    return F.cross_entropy(m.head(h).float().reshape(-1, 256), tgt.reshape(-1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_are_no_further_off_than_elementary_operations(gpu, dtype):
    """Both passes round to 16 bits at the same places, some forty one after the other, each rounding as good as independent of the
    other pass's: the 2-norms of their errors, of hundreds of values at least, are then alike.  Twice the other's is allowed; a state, a
    sum or a statistic of the operators in 16 bits would be roundings that the elementary pass has not."""
    m, _ = _model()
    x = torch.from_numpy(np.random.default_rng(4).integers(0, 256, (4, 60))).cuda()
    want, w = _loss64(m, x)
    want.backward()
    scale = 1024.0 if dtype == torch.float16 else 1.0

    def errors(loss_of):
        m.zero_grad()
        with torch.autocast("cuda", dtype=dtype):
            loss = loss_of()
        (loss * scale).backward()
        assert all(p.grad.dtype == torch.float32 for p in m.parameters())
        return {k: float((p.grad.cpu().double() / scale - w[k].grad).norm() / w[k].grad.norm()) for k, p in m.named_parameters()}

    ours, plain = errors(lambda: m.loss(x)), errors(lambda: _plain_loss(m, x, dtype))
    print({k: (round(ours[k], 4), round(plain[k], 4)) for k in ours})
    assert all(ours[k] <= 2 * plain[k] for k in ours), {k: (ours[k], plain[k]) for k in ours if ours[k] > 2 * plain[k]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_norm_of_16_bit_rows_is_the_float32_ones_rounded(gpu, dtype):
    """The second layer norm of a block takes and gives autocast's type: the values of one that gives float32 to a product, which
    would round it, and takes its gradient back from there."""
    from boa_amd import ops

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(70, 256, generator=g, device="cuda").to(dtype)
    w, b = (torch.randn(256, generator=g, device="cuda", requires_grad=True) for _ in range(2))
    dy = torch.randn(70, 256, generator=g, device="cuda").to(dtype)
    got = []
    for widen in (lambda t: t, lambda t: t.float()):
        leaf = x.clone().requires_grad_()
        y = ops.layer_norm(widen(leaf), w, b).to(dtype)
        got.append([y.detach(), *torch.autograd.grad(y, (leaf, w, b), dy)])
    (y, dx, dw, db), (y32, dx32, dw32, db32) = got
    if dtype == torch.bfloat16:
        assert torch.equal(y, y32) and torch.equal(dx, dx32)
    # in float16 the last operation, a fused multiply-add, gives its exact result in 16 bits (v_fma_mixlo_f16) without the float32
    # in between: where that one lies on the border of two float16 values (2^13 float32 values to one step) they may differ, by a step
    for p, q in ((y.float(), y32.float()), (dx.float(), dx32.float())):
        assert ((p - q).abs() <= torch.finfo(dtype).eps * torch.maximum(p.abs(), q.abs()) + 2.0 ** -24).all()
        assert ((p != q).sum() <= p.numel() // 100)
    # the same 70 terms dy xh, and dy, which 16-bit rows are added in pairs and float32 ones singly: either order is off by at most
    # 70 roundings of the sum of magnitudes, and xh is off by less than its double
    xh = (x.double() - x.double().mean(1, keepdim=True)) / x.double().std(1, keepdim=True)
    for p, q, terms in ((dw, dw32, 2 * (dy.double() * xh).abs()), (db, db32, dy.double().abs())):
        assert ((p - q).abs().double() <= 2 * 70 * 2.0 ** -24 * terms.sum(0)).all()


def test_steps_between_passes_of_one_autocast_region(gpu):
    m, _ = _model(1)
    x = torch.from_numpy(np.random.default_rng(8).integers(0, 256, (3, 40))).cuda()
    got = []
    for sample in (False, True):
        m.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            if sample:
                caches = m.init_caches(3, torch.bfloat16)
                for t in range(3):
                    assert not m.train_step(x[:, t], caches).requires_grad
            loss = m.loss(x)
        loss.backward()
        got.append([p.grad.clone() for p in m.parameters()])
    assert all(torch.equal(p, q) for p, q in zip(*got))
