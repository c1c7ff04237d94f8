"""The model goes on with prompts; and linear attention, the loss, the clipping and the drawing used together, as a model of one's
own uses them, against 64 bits on the CPU."""
import math

import pytest
import torch

import model as M
import more_ops_ref as ref
from boa_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def net():
    torch.manual_seed(0)
    return M.BoaConstrictor(256, 2).cuda()


def test_generated_bytes_are_those_of_the_loop_written_out(gpu, net):
    x = torch.randint(0, 256, (3, 20), dtype=torch.uint8)
    u = torch.rand(9, 3).cuda()
    limits = dict(temperature=torch.tensor([0.0, 1.0, 0.7]).cuda(), top_k=torch.tensor([0, 40, 9], dtype=torch.int32).cuda(), top_p=0.9, min_p=0.01)
    got = net.generate(x, 9, u=u, **limits)
    assert got.shape == (3, 9) and got.dtype == torch.int64 and torch.equal(got, net.generate(x.cuda(), 9, u=u, **limits))
    caches = net.init_caches(3)
    with torch.no_grad():
        logits = net.train_forward(x, caches=caches)[:, -1]
        for t in range(9):
            # the prediction for the whole prefix; sums in another order move a logit by some 1e-5 at most
            whole = net.train_forward(torch.cat([x.cuda(), got[:, :t].to(torch.uint8)], 1))[:, -1]
            assert (whole - logits).abs().max() <= 1e-4
            want, near = ref.sample(logits[1].tolist(), u[t, 1].item(), 1.0, 40, 0.9, 0.01)
            assert near < 1e-3 or want == got[1, t]
            assert logits[0, got[0, t]] >= logits[0].max() - 1e-4
            assert torch.equal(ops.sample(logits, u[t], **limits), got[:, t])
            logits = net.train_step(got[:, t], caches)


def test_generated_bytes_by_a_generator_and_under_autocast(gpu, net):
    x = torch.randint(0, 256, (2, 5))
    run = lambda: net.generate(x, 6, generator=torch.Generator("cuda").manual_seed(7))  # noqa: E731
    assert torch.equal(run(), run()) and int(run().min()) >= 0
    with torch.autocast("cuda", torch.bfloat16):
        loss = net.loss(x)
        got = net.generate(x, 6, temperature=0.0)
        loss = loss + net.loss(x)
    assert got.shape == (2, 6) and int(got.min()) >= 0
    loss.backward()
    assert all(p.grad is not None for p in net.parameters())
    net.zero_grad()
    assert net.generate(x, 0).shape == (2, 0) and net.generate(x[:0], 3).shape == (0, 3)
    assert net.generate(x[:, :1], 1).shape == (2, 1)


def test_a_model_that_predicts_nothing_says_so(gpu):
    net = M.BoaConstrictor(256, 1).cuda()
    with torch.no_grad():
        net.head[2].bias[7] = math.nan
    assert net.generate(torch.zeros(2, 3, dtype=torch.uint8), 4).tolist() == [[-1] * 4] * 2


D, HEADS, GROUPS, KEY, VALUE, V = 32, 4, 2, 16, 24, 256


def _weights():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(emb=r(V, D), q=r(GROUPS * KEY, D) * 0.2, k=r(GROUPS * KEY, D) * 0.2, v=r(HEADS * VALUE, D) * 0.2, decay=-r(HEADS).abs() * 0.1,
                out=r(V, HEADS * VALUE) * 0.2)


def _project(w, x):
    h = w["emb"][x.long()]
    split = lambda name, n, d: (h @ w[name].t()).unflatten(-1, (n, d))  # noqa: E731
    return split("q", GROUPS, KEY), split("k", GROUPS, KEY), split("v", HEADS, VALUE)


def test_the_operators_together(gpu):
    """Two clipped training steps of a byte model with one linear attention, then bytes drawn token by token, against the same in 64
    bits: a float32 product of 32 to 96 terms is off by some 1e-6 of its size, and what follows from it by a few times that."""
    x = torch.randint(0, V, (3, 150), generator=torch.Generator().manual_seed(2))
    lens = torch.tensor([150, 60, 101], dtype=torch.int32)
    target = x[:, 1:].clone()
    target[torch.arange(1, 150)[None] >= lens[:, None]] = -100
    w = {k: t.cuda().requires_grad_() for k, t in _weights().items()}
    w64 = {k: t.double().requires_grad_() for k, t in _weights().items()}
    for _ in range(2):
        y = ops.linear_attention(*_project(w, x[:, :-1].cuda()), w["decay"], lens=(lens - 1).cuda())
        loss = ops.cross_entropy(y.flatten(2) @ w["out"].t(), target.cuda())
        loss.backward()
        norm = ops.clip_grad_norm_(w.values(), 0.05)
        y64, _ = ref.attention(*_project(w64, x[:, :-1]), w64["decay"], KEY ** -0.5, lens - 1)
        loss64 = torch.nn.functional.cross_entropy((y64.flatten(2) @ w64["out"].t()).flatten(0, 1), target.flatten())
        loss64.backward()
        norm64 = torch.linalg.vector_norm(torch.cat([t.grad.flatten() for t in w64.values()]))
        assert abs(float(loss) - float(loss64)) <= 1e-5 * float(loss64) and abs(float(norm) - float(norm64)) <= 1e-4 * float(norm64)
        assert float(norm64) > 0.05
        for name in w:
            want = w64[name].grad * (0.05 / (norm64 + 1e-6))
            assert torch.linalg.vector_norm(w[name].grad.cpu().double() - want) <= 1e-4 * torch.linalg.vector_norm(want), name
            with torch.no_grad():
                w[name] -= 10.0 * w[name].grad
                w64[name] -= 10.0 * want
            w[name].grad = w64[name].grad = None
    with torch.no_grad():
        prompt, u = x[:, :70], torch.rand(8, 3, generator=torch.Generator().manual_seed(3))
        y, state = ops.linear_attention(*_project(w, prompt.cuda()), w["decay"], return_state=True)
        logits = y[:, -1].flatten(1) @ w["out"].t()
        text = prompt
        for t in range(8):
            y64, _ = ref.attention(*_project(w64, text), w64["decay"], KEY ** -0.5)
            l64 = y64[:, -1].flatten(1) @ w64["out"].t()
            assert (logits.cpu().double() - l64).abs().max() <= 1e-4 * l64.abs().max()
            token = ops.sample(logits, u[t].cuda(), temperature=0.8, top_k=50, top_p=0.95)
            for i in range(3):
                want, near = ref.sample(l64[i].tolist(), u[t, i].item(), 0.8, 50, 0.95)
                assert near < 1e-3 or want == token[i]
            text = torch.cat([text, token.cpu()[:, None]], 1)
            q, k, v = _project(w, token)
            y = ops.linear_attention_step(q, k, v, w["decay"].detach(), state=state)
            logits = y.flatten(1) @ w["out"].t()
