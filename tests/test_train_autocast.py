"""Single-token steps between training passes of one autocast region (CPU: the operators are stood in for by ones of their shapes,
the library products and autocast's store of cast weights are torch's own)."""
import pytest
import torch
import torch.nn.functional as F

from boa_amd import ops


@pytest.fixture
def model(monkeypatch):
    from model import BoaConstrictor

    monkeypatch.setattr(ops, "layer_norm", lambda x, w, b, eps: F.layer_norm(x.float(), x.shape[-1:], w, b, eps).to(x.dtype))
    monkeypatch.setattr(ops, "causal_conv", lambda x, w, b, **kw: x * w[:, 0, 3] + b)
    monkeypatch.setattr(ops, "causal_conv_step", lambda x, state, w, b: x * w[:, 0, 3] + b)
    monkeypatch.setattr(ops, "selective_scan", lambda u, delta, A, B, C, D, z, bias, **kw: (
        u * (delta + bias + D + A.sum(1)) * z * (B * C).sum(-1, keepdim=True)).to(z.dtype))
    monkeypatch.setattr(ops, "selective_scan_step", lambda u, delta, A, B, C, D, z, bias, state: (u * z).to(z.dtype))
    torch.manual_seed(0)
    return BoaConstrictor(d_model=256, num_layers=2, vocab_size=256, device="cpu")


@pytest.mark.parametrize("step", [
    lambda m, c: m.train_step(torch.zeros(3, dtype=torch.uint8), c),
    lambda m, c: m.blocks[0].step(torch.zeros(3, 256), c[0]),
    lambda m, c: m.blocks[0].mamba.step(torch.zeros(3, 256), c[0])])
def test_weights_cast_by_a_step_do_not_reach_a_training_pass(model, step):
    caches, x = model.init_caches(3, torch.bfloat16), torch.arange(12).reshape(3, 4)
    with torch.autocast("cpu", torch.bfloat16):
        got = step(model, caches)
        assert not got.requires_grad
        assert torch.is_grad_enabled() and torch.is_autocast_cache_enabled()
        loss = model.train_forward(x).float().square().mean()
        step(model, caches)  # and one that finds weights cast with a gradient
    loss.backward()
    assert all(p.grad is not None for p in model.parameters()), [k for k, p in model.named_parameters() if p.grad is None]


def test_a_step_that_raises_leaves_the_settings_as_they_were(model):
    with torch.autocast("cpu", torch.bfloat16), pytest.raises(ValueError):
        model.train_step(torch.zeros(3, dtype=torch.uint8), [])
    assert torch.is_grad_enabled() and torch.is_autocast_cache_enabled()
    with torch.autocast("cpu", torch.bfloat16, cache_enabled=False):
        model.train_step(torch.zeros(3, dtype=torch.uint8), model.init_caches(3))
        assert not torch.is_autocast_cache_enabled()
