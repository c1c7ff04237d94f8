"""64-bit restatements of linear attention, of the clipping of gradients and of the drawing of symbols, on the CPU."""
import math

import torch


def attention(q, k, v, g, scale, lens=None, state=None):
    """Position by position: y [batch, length, heads, value] and the state behind each sequence's end; differentiable."""
    n, length, heads, value = v.shape
    share = heads // q.shape[2]
    q, k = (t.repeat_interleave(share, 2) for t in (q, k))
    g = g.expand(n, length, heads)
    s = torch.zeros((n, heads, q.shape[3], value), dtype=torch.float64) if state is None else state
    ends = torch.full((n,), length) if lens is None else lens
    ys = []
    for t in range(length):
        live = (t < ends)[:, None, None, None]
        new = torch.exp(g[:, t])[..., None, None] * s + k[:, t, :, :, None] * v[:, t, :, None]
        s = torch.where(live, new, s)
        ys.append(torch.where(live[..., 0], scale * (q[:, t, :, :, None] * s).sum(2), torch.zeros_like(v[:, t])))
    return (torch.stack(ys, 1) if ys else torch.zeros_like(v)), s


def attention_grads(q, k, v, g, scale, dy, lens=None, state=None):
    """y, the last state and the gradients of q, k, v, g, in 64 bits."""
    leaves = [t.detach().cpu().double().requires_grad_() for t in (q, k, v, g)]
    y, s = attention(*leaves, scale, None if lens is None else lens.cpu(), None if state is None else state.cpu().double())
    grads = torch.autograd.grad((y * dy.detach().cpu().double()).sum(), leaves) if y.numel() else [torch.zeros_like(t) for t in leaves]
    return y.detach(), s.detach(), grads


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The symbol of one row (a list of floats), and how near its choice was to another one: the least distance of a sum to a border,
    of all the weights."""
    v = len(x)
    if any(math.isnan(t) for t in (u, temperature, top_p, min_p)) or any(map(math.isnan, x)) or max(x) == -math.inf:
        return -1, 1.0
    order = sorted(range(v), key=lambda i: (-x[i], i))
    most = x[order[0]]
    if temperature <= 0 or top_p <= 0 or min_p > 1:
        return order[0], 1.0
    if 0 < top_k < v:
        order = order[:top_k]
    w = {i: 1.0 if x[i] == most else 0.0 if math.isinf(x[i] - most) else math.exp((x[i] - most) / temperature) for i in order}
    total, near = math.fsum(w.values()), 1.0
    exact = all(t in (0.0, 1.0) for t in w.values())  # whole sums, the same in every order
    if top_p < 1:
        kept, s = [], []
        for i in order:
            before = math.fsum(s)
            if kept:
                near = min(near, abs(before - top_p * total) / total)
            if kept and before >= top_p * total:
                break
            kept.append(i)
            s.append(w[i])
        order = kept
    if min_p > 0:
        near = min([near] + [abs(w[i] - min_p) for i in order if w[i] != 1.0])
    kept = sorted(i for i in order if w[i] >= min_p and w[i] > 0)
    total, s = math.fsum(w[i] for i in kept), []
    for i in kept:
        s.append(w[i])
        upto = math.fsum(s)
        near = min(near, abs(upto - u * total) / total) if u > 0 else near
        if upto > u * total:
            break
    return i, 1.0 if exact else near
