"""The byte model's training pass (model.py train_forward, loss, train_step) on the operators of boa_amd.ops: logits against the
oracle, gradients against the same formulas in 64 bits, and what a training program does with them.

Tolerance: 1e-4 of the largest value, as the logits of the inference path have it (float32 products of up to 1024 terms)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import model_ref, weights_ref

pytestmark = pytest.mark.gpu

REL_TOL = 1e-4


def _model(layers=2, seed=0, d=256):
    from boa_amd import weights as W

    import model as M

    blob = W.seeded_blob(W.Cfg(d_model=d, n_layers=layers), seed)
    return M.BoaConstrictor(d, layers, 256).load_blob(blob).cuda(), blob


def _rel(a, b):
    return float((a.detach().cpu().double() - b.detach().double()).abs().max() / b.detach().double().abs().max())


def _loss64(m, x, lens=None):
    """BoaBytePredictor.loss in 64 bits on the CPU with autograd, position by position."""
    w = {k: v.detach().cpu().double().requires_grad_() for k, v in m.named_parameters()}
    inp, tgt = x[:, :-1].cpu().long(), x[:, 1:].cpu().long()
    h = w["embedding.weight"][inp]
    B, T = inp.shape
    for i, block in enumerate(m.blocks):
        p, q, mx = f"blocks.{i}.", f"blocks.{i}.mamba.", block.mamba
        xz = F.layer_norm(h, h.shape[-1:], w[p + "ln1.weight"], w[p + "ln1.bias"]) @ w[q + "in_proj.weight"].t()
        u, z = xz.chunk(2, -1)
        u = F.silu(F.conv1d(F.pad(u.transpose(1, 2), (3, 0)), w[q + "conv1d.weight"], w[q + "conv1d.bias"], groups=mx.d_inner)).transpose(1, 2)
        dr, Bm, Cm = (u @ w[q + "x_proj.weight"].t()).split([mx.dt_rank, 16, 16], -1)
        dt = F.softplus(dr @ w[q + "dt_proj.weight"].t() + w[q + "dt_proj.bias"])
        A, s, ys = -torch.exp(w[q + "A_log"]), torch.zeros(B, mx.d_inner, 16, dtype=torch.float64), []
        for t in range(T):
            s = torch.exp(dt[:, t, :, None] * A) * s + (dt[:, t] * u[:, t])[..., None] * Bm[:, t, None]
            ys.append((s * Cm[:, t, None]).sum(2) + w[q + "D"] * u[:, t])
        y = (torch.stack(ys, 1) * F.silu(z)) @ w[q + "out_proj.weight"].t()
        y = F.layer_norm(y, y.shape[-1:], w[p + "ln2.weight"], w[p + "ln2.bias"])
        y = F.gelu(y @ w[p + "ff.0.weight"].t() + w[p + "ff.0.bias"])
        h = h + y @ w[p + "ff.2.weight"].t() + w[p + "ff.2.bias"]
    logits = F.relu(h @ w["head.0.weight"].t() + w["head.0.bias"]) @ w["head.2.weight"].t() + w["head.2.bias"]
    if lens is not None:
        tgt = torch.where(torch.arange(1, T + 1) < lens.cpu()[:, None], tgt, torch.full_like(tgt, -100))
    return F.cross_entropy(logits.reshape(-1, 256), tgt.reshape(-1)), w


def test_logits_against_the_oracle_and_the_codecs(gpu):
    m, blob = _model()
    x = torch.from_numpy(np.random.default_rng(1).integers(0, 256, (3, 130)).astype(np.uint8)).cuda()
    got = m.train_forward(x)
    assert got.requires_grad
    ref = model_ref.RefModel(blob, weights_ref.Cfg(n_layers=2)).forward(x.cpu())
    assert _rel(got, ref) <= REL_TOL
    assert _rel(got, m(x).cpu()) <= REL_TOL  # the codec's forward


@pytest.mark.parametrize("ragged", [False, True])
def test_gradients(gpu, ragged):
    m, _ = _model()
    x = torch.from_numpy(np.random.default_rng(2).integers(0, 256, (3, 90))).cuda()
    lens = torch.tensor([90, 33, 1], device="cuda") if ragged else None
    if ragged:
        x[1, 33:], x[2, 1:] = -7, 999  # padding is anything
    loss = m.loss(x, lens)
    loss.backward()
    if ragged:
        x = x.clamp(0, 255)
    want, w = _loss64(m, x, lens)
    want.backward()
    assert _rel(loss, want) <= 1e-6
    for k, p in m.named_parameters():
        assert _rel(p.grad, w[k].grad) <= REL_TOL, k


def test_symbols_outside_the_vocabulary(gpu):
    m, _ = _model(1)
    x = torch.zeros(2, 9, dtype=torch.int64, device="cuda")
    good = m.train_forward(x)
    x[1, 4] = 256
    got = m.train_forward(x)
    assert torch.equal(got[0], good[0]) and torch.equal(got[1, :4], good[1, :4]) and got[1, 4:].isnan().all()
    assert m.loss(x).isnan()
    with pytest.raises(ValueError):
        m.loss(x[:, :1])
    with pytest.raises(ValueError):
        m.train_forward(x[0])


def test_caches(gpu):
    """Bytes in parts, and one by one, continue a sequence; a sequence that ended leaves its cache as it was."""
    m, _ = _model()
    x = torch.from_numpy(np.random.default_rng(3).integers(0, 256, (3, 75))).cuda()
    with torch.no_grad():
        want = m.train_forward(x)
        caches = m.init_caches(3)
        got = [m.train_forward(x[:, :40], caches=caches), m.train_forward(x[:, 40:60], caches=caches)]
        got += [m.train_step(x[:, t], caches)[:, None] for t in range(60, 75)]
        assert _rel(torch.cat(got, 1), want.cpu()) <= REL_TOL
        ended = [[t.clone() for t in c] for c in caches]
        m.train_forward(x[:, :8], lens=torch.tensor([0, 8, 0], device="cuda"), caches=caches)
        for before, after in zip(ended, caches):
            for p, q in zip(before, after):
                assert torch.equal(p[0], q[0]) and torch.equal(p[2], q[2]) and not torch.equal(p[1], q[1])
    loss = F.cross_entropy(m.train_forward(x[:, :20], caches=caches).reshape(-1, 256), x[:, 1:21].reshape(-1))
    loss.backward()  # states carry no gradient, everything else does
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mixed_precision(gpu, dtype):
    """Under autocast the products, the convolution and the scan run in 16 bits; gradients come out as float32.

    Tolerance, in the 2-norm: a rounding of a tensor's values is off by at most half a step of the tensor's norm; about ten lie
    one after the other in each layer, forward and backward, so 40 in two layers; a product by a matrix like these, random with
    entries of one size, makes a relative error of that norm at most twice as large: 80 half steps."""
    tol = 80 * torch.finfo(dtype).eps / 2

    def off(a, b):
        return float((a.float() - b.float()).norm() / b.float().norm())

    m, _ = _model()
    x = torch.from_numpy(np.random.default_rng(4).integers(0, 256, (4, 60))).cuda()
    m.loss(x).backward()
    full = {k: p.grad.clone() for k, p in m.named_parameters()}
    m.zero_grad()
    scale = 1024.0 if dtype == torch.float16 else 1.0
    with torch.autocast("cuda", dtype=dtype):
        loss = m.loss(x)
    (loss * scale).backward()
    for k, p in m.named_parameters():
        assert p.grad.dtype == torch.float32 and off(p.grad / scale, full[k]) <= tol, k
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        caches = m.init_caches(4, dtype)
        want = m.train_forward(x)
        got = [m.train_forward(x[:, :30], caches=caches)] + [m.train_step(x[:, t], caches)[:, None] for t in range(30, 60)]
    assert off(torch.cat(got, 1), want) <= tol


def test_trained_weights_compress(gpu):
    """An optimizer step changes what the codec writes, and what it writes is read back."""
    import codec

    m, _ = _model(1)
    data = np.random.default_rng(5).integers(0, 4, 400).astype(np.uint8)
    before = codec.compress_payload(m, [data])[1].sum()
    opt = torch.optim.SGD(m.parameters(), lr=0.05)
    x = torch.from_numpy(data[None]).cuda()
    for _ in range(3):
        opt.zero_grad()
        m.loss(x).backward()
        opt.step()
    payload, nw, fb, ls = codec.compress_payload(m, [data])
    assert nw.sum() != before
    assert np.array_equal(codec.decompress_payload(m, payload, nw, ls, fb)[0], data)


def test_captured_training_step(gpu):
    """Forward, backward and update as one graph: every replay's loss and weights are the eager step's."""
    eager, _ = _model(1)
    captured, _ = _model(1)
    rng = np.random.default_rng(6)
    x = torch.zeros((2, 70), dtype=torch.uint8, device="cuda")
    params = list(captured.parameters())

    def step(model, ps):
        loss = model.loss(x)
        grads = torch.autograd.grad(loss, ps)
        with torch.no_grad():
            for p, g in zip(ps, grads):
                p.sub_(g, alpha=0.01)
        return loss.detach()

    start = [p.detach().clone() for p in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured, params)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(captured, params)
    with torch.no_grad():
        for p, s in zip(params, start):
            p.copy_(s)
    for _ in range(4):
        x.copy_(torch.from_numpy(rng.integers(0, 256, (2, 70)).astype(np.uint8)))
        want = step(eager, list(eager.parameters()))
        graph.replay()
        torch.cuda.synchronize()
        assert _rel(loss, want.cpu()) <= 1e-6
        for p, q in zip(params, eager.parameters()):
            assert _rel(p, q.cpu()) <= 1e-6


def test_weights_trained_by_a_graph_compress(gpu):
    """The codec does not see what a replayed graph writes; release_engines() makes it look."""
    import codec

    m, _ = _model(1)
    data = np.random.default_rng(7).integers(0, 4, 300).astype(np.uint8)
    w = m.head[2].weight
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        w.mul_(1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        w.mul_(0.5)
    before = codec.compress_payload(m, [data])[0]
    graph.replay()
    m.release_engines()
    got = codec.compress_payload(m, [data])[0]
    other, _ = _model(1)
    with torch.no_grad():
        other.head[2].weight.mul_(0.5)
    want = codec.compress_payload(other, [data])[0]
    assert np.array_equal(got, want) and not np.array_equal(got, before)
