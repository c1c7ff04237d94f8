"""The operators of the byte model's training pass and of its streaming by single tokens, as cases that can be timed: the
selective scan, the short causal convolution, layer norm and the cross entropy of the next byte.

Each has a plain form (elementary torch operations in 32 bits, with its gradient written out) and, where `own` is true, the
call that a program makes of `boa_amd.ops`.  Sizes are those of this repository's models (d_model 256 and 512, so 512 and
1024 channels of 16 states; 256 byte values), chunk lengths and chunk counts, and odd ones.
"""
import functools
import math
import os
import sys

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

D_STATE, D_CONV, VOCAB = 16, 4, 256
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST = 16384 * 1024  # positions times channels of the largest scan


def listed():
    return [
        # one token of one stream through the scan: the smallest call there is, where latency counts
        {"name": "scan_step_1x512", "op": "scan", "mode": "step", "batch": 1, "channels": 512, "dtype": "f32"},
        # one token of each of the 1000 chunks of the command line's default, the larger model in bfloat16
        {"name": "scan_step_1000x1024_bf16", "op": "scan", "mode": "step", "batch": 1000, "channels": 1024, "dtype": "bf16"},
        # a few prompts of an odd length, continued from a state and handing one on (bfloat16, the larger model)
        {"name": "scan_prompt_4x4097x1024_bf16", "op": "scan", "mode": "prompt", "batch": 4, "length": 4097, "channels": 1024,
         "dtype": "bf16", "ragged": False},
        # an ordinary training batch of the d_model 256 model: forward and gradient
        {"name": "scan_train_8x1000x512", "op": "scan", "mode": "train", "batch": 8, "length": 1000, "channels": 512,
         "dtype": "f32", "ragged": False},
        # whole chunks of the headline's 16384 bytes: few sequences, so the work has to be split over the length
        {"name": "scan_train_2x16384x512", "op": "scan", "mode": "train", "batch": 2, "length": 16384, "channels": 512,
         "dtype": "f32", "ragged": False},
        # many short chunks of different lengths, padded to the longest, in bfloat16 with the larger model
        {"name": "scan_train_32x500x1024_bf16", "op": "scan", "mode": "train", "batch": 32, "length": 500, "channels": 1024,
         "dtype": "bf16", "ragged": True},
        # one token of 64 streams through the convolution
        {"name": "conv_step_64x512", "op": "conv", "mode": "step", "batch": 64, "channels": 512, "dtype": "f32"},
        # the convolution's forward and gradient on 64 chunks of 1500 bytes, padded
        {"name": "conv_train_64x1500x512", "op": "conv", "mode": "train", "batch": 64, "length": 1500, "channels": 512,
         "dtype": "f32", "ragged": True},
        # layer norm's forward and gradient on an ordinary training batch of the d_model 256 model
        {"name": "norm_train_8000x256", "op": "norm", "mode": "train", "rows": 8000, "width": 256, "dtype": "f32"},
        # and on a large one of the d_model 512 model in bfloat16
        {"name": "norm_train_262144x512_bf16", "op": "norm", "mode": "train", "rows": 262144, "width": 512, "dtype": "bf16"},
        # the loss of an ordinary batch and its gradient
        {"name": "loss_train_8000x256", "op": "loss", "mode": "train", "rows": 8000, "vocab": VOCAB, "dtype": "f32"},
        # and of a large one, logits in bfloat16
        {"name": "loss_train_262144x256_bf16", "op": "loss", "mode": "train", "rows": 262144, "vocab": VOCAB, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "conv", "norm", "loss"])
    c = {"op": op, "mode": "train", "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
    if op == "norm":
        width = rng.choice([256, 512, rng.randint(17, 2100)])
        return {**c, "rows": _log(rng, 3, 262144 * 512 // max(width, 512)), "width": width}
    if op == "loss":
        vocab = rng.choice([VOCAB, VOCAB, rng.randint(5, 1000)])
        return {**c, "rows": _log(rng, 3, 262144 * VOCAB // max(vocab, VOCAB)), "vocab": vocab}
    c["channels"] = rng.choice([512, 1024, rng.randint(33, 1100)])
    c["mode"] = rng.choice(["train", "train", "train", "prompt", "step"])
    if c["mode"] == "step":
        return {**c, "batch": _log(rng, 1, 2000)}
    most = (MOST - (1 << 20)) * (2 if op == "conv" else 1) // c["channels"]
    c["length"] = _log(rng, 2, 16384)
    c["batch"] = _log(rng, 1, max(1, min(256, most // c["length"])))
    c["ragged"] = c["batch"] > 1 and rng.random() < 0.5
    return c


def _lens(case, g):
    """Lengths of a padded batch, the first one whole (None: all of them whole)."""
    if not case["ragged"]:
        return None
    lens = torch.randint(0, case["length"] + 1, (case["batch"],), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = case["length"]
    return lens


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["mode"] == "train"

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(mean)

    s = {"op": case["op"], "mode": case["mode"]}
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        s.update(x=normal(n, d, scale=2.0, mean=0.3).to(dt), w=normal(d, scale=0.2, mean=1.0), b=normal(d, scale=0.2),
                 dy=normal(n, d).to(dt))
        leaves = ("x", "w", "b")
    elif case["op"] == "loss":
        n, v = case["rows"], case["vocab"]
        # next bytes, a few of them behind the end of their chunk; float16 losses are scaled up, as mixed precision does
        t = torch.randint(0, v, (n,), generator=g, device="cuda")
        t[torch.rand(n, generator=g, device="cuda") < 0.1] = -100
        t[0] = 0
        s.update(x=normal(n, v, scale=3.0).to(dt), target=t,
                 dy=torch.tensor(16384.0 if case["dtype"] == "f16" else 1.0, device="cuda"))
        leaves = ("x",)
    else:
        n, c = case["batch"], case["channels"]
        lead = (n,) if case["mode"] == "step" else (n, case["length"])
        s["lens"] = None if case["mode"] == "step" else _lens(case, g)
        s["dy"] = normal(*lead, c).to(dt) if train else None
        if case["op"] == "conv":
            s.update(x=normal(*lead, c).to(dt), w=normal(c, 1, D_CONV, scale=0.3), b=normal(c, scale=0.3),
                     state=None if train else normal(n, D_CONV - 1, c).to(dt))
            leaves = ("x", "w", "b")
        else:
            # as the mixer has them: u out of the convolution, dt as the projection leaves it (its bias apart), B and C as
            # two columns ranges of the same projection's rows
            rank = -(-c // 32)
            dbc = normal(*lead, rank + 2 * D_STATE).to(dt)
            step = torch.exp(torch.rand(c, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
            s.update(u=torch.nn.functional.silu(normal(*lead, c)).to(dt), delta=normal(*lead, c, scale=0.5).to(dt),
                     A=-torch.exp(normal(c, D_STATE, scale=0.1)) * torch.arange(1, D_STATE + 1, device="cuda"),
                     B=dbc[..., rank:rank + D_STATE], C=dbc[..., rank + D_STATE:], D=normal(c, scale=0.1, mean=1.0),
                     z=normal(*lead, c).to(dt), bias=step + torch.log(-torch.expm1(-step)),
                     state=None if train else normal(n, D_STATE, c, scale=0.3))
            leaves = ("u", "delta", "A", "B", "C", "D", "z", "bias")
    if train:
        for k in leaves:
            s[k] = s[k].detach().requires_grad_()
        s["leaves"] = tuple(s[k] for k in leaves)
    return s


@functools.lru_cache(maxsize=1)
def _ops():
    sys.path.insert(0, os.path.join(REPO, "boa-constrictor_amd"))
    from boa_amd import ops
    return ops


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"norm": _norm, "loss": _loss, "conv": _conv, "scan": _scan}[s["op"]](s)


def _own(s):
    op, mode, ops = s["op"], s["mode"], _ops()
    if op == "norm":
        y = ops.layer_norm(s["x"], s["w"], s["b"])
    elif op == "loss":
        y = ops.cross_entropy(s["x"], s["target"], ignore_index=-100)
    elif op == "conv":
        if mode == "step":
            return {"y": ops.causal_conv_step(s["x"], s["state"], s["w"], s["b"]), "state": s["state"]}
        if mode == "prompt":
            y, state = ops.causal_conv(s["x"], s["w"], s["b"], state=s["state"], lens=s["lens"], return_state=True)
            return {"y": y, "state": state}
        y = ops.causal_conv(s["x"], s["w"], s["b"], lens=s["lens"])
    else:
        args = [s[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")]
        if mode == "step":
            return {"y": ops.selective_scan_step(*args, state=s["state"]), "state": s["state"]}
        if mode == "prompt":
            y, state = ops.selective_scan(*args, state=s["state"], lens=s["lens"], return_state=True)
            return {"y": y, "state": state}
        y = ops.selective_scan(*args, lens=s["lens"])
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, s["leaves"], s["dy"]))}


def _norm(s, eps=1e-5):
    dt = s["x"].dtype
    x, w, dy = s["x"].float(), s["w"], s["dy"].float()
    x = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + eps)
    xh = x * rstd
    g = dy * w
    dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) * rstd
    return {"y": (xh * w + s["b"]).to(dt), "grads": [dx.to(dt), (dy * xh).sum(0), dy.sum(0)]}


def _loss(s):
    x, t = s["x"].float(), s["target"]
    kept = t >= 0
    count = kept.sum()
    x = x - x.amax(1, keepdim=True)
    total = torch.exp(x).sum(1, keepdim=True)
    hit = t.clamp(min=0)[:, None] == torch.arange(x.shape[1], device=x.device)
    losses = torch.log(total)[:, 0] - torch.where(hit, x, torch.zeros_like(x)).sum(1)
    dx = (torch.exp(x) / total - hit.float()) * (kept.float() / count * s["dy"])[:, None]
    return {"y": torch.where(kept, losses, torch.zeros_like(losses)).sum() / count, "grads": [dx.to(s["x"].dtype)]}


def _inside(s, n, length):
    """Positions that are not padding, [n, length, 1]."""
    if s["lens"] is None:
        return torch.ones((n, length, 1), dtype=torch.bool, device="cuda")
    return (torch.arange(length, device="cuda") < s["lens"][:, None])[..., None]


def _silu(p):
    """x sigmoid(x) and its derivative."""
    sig = torch.sigmoid(p)
    return p * sig, sig * (1 + p * (1 - sig))


def _conv(s):
    dt, w, k = s["x"].dtype, s["w"][:, 0, :], D_CONV
    x = s["x"].float()
    if s["mode"] == "step":
        past = torch.cat([s["state"].float(), x[:, None]], 1)
        s["state"].copy_(past[:, 1:])
        return {"y": _silu((past * w.t()).sum(1) + s["b"])[0].to(dt), "state": s["state"]}
    n, length, c = x.shape
    inside = _inside(s, n, length)
    x = torch.where(inside, x, torch.zeros_like(x))
    first = torch.zeros((n, k - 1, c), device="cuda") if s["state"] is None else s["state"].float()
    past = torch.cat([first, x], 1)
    taps = [past[:, j:j + length] for j in range(k)]
    y, slope = _silu(s["b"] + taps[0] * w[:, 0] + taps[1] * w[:, 1] + taps[2] * w[:, 2] + taps[3] * w[:, 3])
    y = torch.where(inside, y, torch.zeros_like(y)).to(dt)
    if s["mode"] == "prompt":
        lens = torch.full((n,), length, device="cuda") if s["lens"] is None else s["lens"].long()
        at = (lens[:, None] + torch.arange(k - 1, device="cuda"))[..., None].expand(-1, -1, c)
        return {"y": y, "state": torch.gather(past, 1, at).to(dt)}
    g = torch.where(inside, s["dy"].float() * slope, torch.zeros_like(slope))
    ahead = torch.cat([g, torch.zeros((n, k - 1, c), device="cuda")], 1)
    dx = ahead[:, :length] * w[:, 3] + ahead[:, 1:length + 1] * w[:, 2] + ahead[:, 2:length + 2] * w[:, 1] + ahead[:, 3:] * w[:, 0]
    dx = torch.where(inside, dx, torch.zeros_like(dx))
    dw = torch.stack([(g * t).sum(1).sum(0) for t in taps], 1)[:, None]
    return {"y": y, "grads": [dx.to(dt), dw, g.sum(1).sum(0)]}


def _recurrence(a, b):
    """h_t = a_t h_(t-1) + b_t along dimension 1, by doubling: after each round an element sums twice as many positions."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _scan(s):
    dt = s["u"].dtype
    u, delta, B, C, z = (s[k].float() for k in ("u", "delta", "B", "C", "z"))
    A, D = s["A"], s["D"]
    p = delta + s["bias"]
    step = p.clamp(min=0) + torch.log1p(torch.exp(-p.abs()))
    if s["mode"] == "step":
        h = torch.exp(step[:, None] * A.t()) * s["state"] + (step * u)[:, None] * B[..., None]
        s["state"].copy_(h)
        return {"y": (((h * C[..., None]).sum(1) + D * u) * _silu(z)[0]).to(dt), "state": s["state"]}
    n, length, c = u.shape
    inside = _inside(s, n, length)
    zero = torch.zeros_like(u)
    u, step, z = (torch.where(inside, v, zero) for v in (u, step, z))
    B, C = (torch.where(inside, v, torch.zeros_like(v)) for v in (B, C))
    a = torch.exp(step[..., None] * A)
    b = (step * u)[..., None] * B[:, :, None]
    if s["state"] is not None:
        b[:, 0] += a[:, 0] * s["state"].transpose(1, 2)
    h = _recurrence(a, b)
    y0 = (h * C[:, :, None]).sum(3) + D * u
    gate, slope = _silu(z)
    y = torch.where(inside, y0 * gate, zero).to(dt)
    if s["mode"] == "prompt":
        return {"y": y, "state": h[:, -1].transpose(1, 2).contiguous()}
    del b
    dy = torch.where(inside, s["dy"].float(), zero)
    g, dz = dy * gate, dy * y0 * slope
    # dh_t = C_t g_t + a_(t+1) dh_(t+1): the same recurrence from the end
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    dh = _recurrence(later, (g[..., None] * C[:, :, None]).flip(1)).flip(1)
    del later
    dC = (g[..., None] * h).sum(2)
    dB = (dh * (step * u)[..., None]).sum(2)
    dhB = (dh * B[:, :, None]).sum(3)
    kept = dh * a
    kept[:, 1:] *= h[:, :-1]
    kept[:, 0] = 0
    dstep = u * dhB + (kept * A).sum(3)
    dA = (kept * step[..., None]).sum(1).sum(0)
    ddelta = torch.where(inside, dstep * torch.sigmoid(p), zero)
    du = torch.where(inside, step * dhB + D * g, zero)
    return {"y": y, "grads": [du.to(dt), ddelta.to(dt), dA, dB.to(dt), dC.to(dt), (g * u).sum(1).sum(0), dz.to(dt),
                              ddelta.sum(1).sum(0)]}


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    train = case["mode"] == "train"
    if case["op"] == "norm":  # x, dy in; y, dx out; weight, bias and their gradients; per-row values kept in between do not count
        n, d = case["rows"], case["width"]
        return {"bytes": 4 * n * d * es + 16 * d, "flops": 18 * n * d}
    if case["op"] == "loss":  # logits in, gradient out, targets
        n, v = case["rows"], case["vocab"]
        return {"bytes": 2 * n * v * es + 8 * n, "flops": 7 * n * v}
    n, c = case["batch"], case["channels"]
    positions = n * case.get("length", 1)
    if case["op"] == "conv":
        state = 0 if train else 2 * n * (D_CONV - 1) * c * es
        weights = c * (D_CONV + 1) * 4 * (2 if train else 1)
        return {"bytes": positions * c * es * (4 if train else 2) + state + weights,
                "flops": positions * c * (2 * D_CONV + 4 + (4 * D_CONV + 10 if train else 0))}
    # u, delta, z in, y out; with the gradient dy in and those of u, delta, z out; B, C and theirs
    state = 0 if train else 2 * n * D_STATE * c * 4
    weights = c * (D_STATE + 2) * 4 * (2 if train else 1)
    return {"bytes": positions * es * (c * (8 if train else 4) + D_STATE * (4 if train else 2)) + state + weights,
            "flops": positions * c * ((7 + (15 if train else 0)) * D_STATE + (40 if train else 15))}


def exact(case, seed):
    """The operators' definitions in 64 bits, position by position."""
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in prepare(case, seed).items()}
    return {"norm": _exact_norm, "loss": _exact_loss, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](s)


def _exact_norm(s):
    leaves = [s[k].requires_grad_() for k in ("x", "w", "b")]
    x, w, b = leaves
    y = (x - x.mean(1)[:, None]) / torch.sqrt(x.var(1, unbiased=False)[:, None] + 1e-5) * w + b
    return {"y": y.detach(), "grads": list(torch.autograd.grad((y * s["dy"]).sum(), leaves))}


def _exact_loss(s):
    x = s["x"].requires_grad_()
    rows = torch.nonzero(s["target"] != -100)[:, 0]
    y = (torch.logsumexp(x[rows], 1) - x[rows, s["target"][rows]]).mean()
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, [x], s["dy"]))}


def _ends(s, n, length):
    return [length] * n if s["lens"] is None else s["lens"].tolist()


def _exact_conv(s):
    x, w, b = s["x"], s["w"][:, 0, :], s["b"]
    step = s["mode"] == "step"
    x = x[:, None] if step else x
    n, length, c = x.shape
    first = s["state"] if s["state"] is not None else x.new_zeros((n, D_CONV - 1, c))
    y, dx, dw, db, state = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b), torch.empty_like(first)
    for i, end in enumerate([1] * n if step else _ends(s, n, length)):
        row = torch.cat([first[i], x[i, :end]])
        wins = row.unfold(0, D_CONV, 1) if end else row.new_zeros((0, c, D_CONV))  # [end, c, taps]
        p = torch.einsum("tck,ck->tc", wins, w) + b
        y[i, :end] = p / (1 + torch.exp(-p))
        state[i] = row[end:]
        if s["mode"] == "train" and end:
            sig = 1 / (1 + torch.exp(-p))
            g = s["dy"][i, :end] * (sig + p * sig * (1 - sig))
            db += g.sum(0)
            dw += torch.einsum("tck,tc->ck", wins, g)
            back = row.new_zeros((end + D_CONV - 1, c))
            for k in range(D_CONV):
                back[k:k + end] += g * w[:, k]
            dx[i, :end] = back[D_CONV - 1:]
    if s["mode"] == "train":
        return {"y": y, "grads": [dx, dw[:, None], db]}
    return {"y": y[:, 0] if step else y, "state": state}


def _exact_scan(s):
    names = ("u", "delta", "B", "C", "z")
    u, delta, B, C, z = (s[k][:, None] if s["mode"] == "step" else s[k] for k in names)
    A, D = s["A"], s["D"]
    n, length, c = u.shape
    ends = torch.tensor(_ends(s, n, length) if s["mode"] != "step" else [1] * n, device="cuda")
    dt = torch.logaddexp(delta + s["bias"], torch.zeros_like(s["bias"]))
    h = s["state"].transpose(1, 2) if s["state"] is not None else u.new_zeros((n, c, D_STATE))
    train = s["mode"] == "train"
    y0, kept = torch.zeros_like(u), []
    for t in range(length):
        if train:
            kept.append(h)
        new = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * B[:, t, None]
        h = torch.where((t < ends)[:, None, None], new, h)
        y0[:, t] = torch.einsum("bcn,bn->bc", h, C[:, t]) + D * u[:, t]
    valid = (torch.arange(length, device="cuda") < ends[:, None])[..., None]
    sig = 1 / (1 + torch.exp(-z))
    y = torch.where(valid, y0 * z * sig, torch.zeros_like(y0))
    if not train:
        return {"y": y[:, 0] if s["mode"] == "step" else y, "state": h.transpose(1, 2).contiguous()}
    dy = torch.where(valid, s["dy"], torch.zeros_like(y0))
    g = dy * z * sig
    dz = dy * y0 * (sig + z * sig * (1 - sig))
    du, ddt, dB, dC, dA = (torch.zeros_like(v) for v in (u, u, B, C, A))
    dh = torch.zeros_like(h)
    for t in reversed(range(length)):
        live = (t < ends)[:, None, None]
        before = kept.pop()
        decay = torch.exp(dt[:, t, :, None] * A)
        now = decay * before + (dt[:, t] * u[:, t])[..., None] * B[:, t, None]
        into = torch.where(live, dh + g[:, t, :, None] * C[:, t, None], torch.zeros_like(dh))
        dC[:, t] = torch.einsum("bcn,bc->bn", now, g[:, t])
        dB[:, t] = torch.einsum("bcn,bc->bn", into, dt[:, t] * u[:, t])
        du[:, t] = dt[:, t] * torch.einsum("bcn,bn->bc", into, B[:, t]) + D * g[:, t]
        flow = into * decay * before
        ddt[:, t] = u[:, t] * torch.einsum("bcn,bn->bc", into, B[:, t]) + (flow * A).sum(2)
        dA += (flow * dt[:, t, :, None]).sum(0)
        dh = torch.where(live, into * decay, dh)
    ddelta = torch.where(valid, ddt / (1 + torch.exp(-(delta + s["bias"]))), torch.zeros_like(ddt))
    return {"y": y, "grads": [torch.where(valid, du, torch.zeros_like(du)), ddelta, dA, dB, dC, (g * u).sum((0, 1)), dz,
                              ddelta.sum((0, 1))]}
