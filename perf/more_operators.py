"""Operators beside the byte model's training pass and its streaming, as cases that can be timed: linear attention with a decay
for each head (whole sequences, their gradient, single tokens), the clipping of gradients by their global norm, and the
drawing of next bytes from logits.

Each has a plain form (elementary torch operations in 32 bits, sums and the angles of long decays in 64, gradients written
out) and, where `own` is true, the call that a program makes of `boa_amd.ops`.  Sizes are those of this repository's models
(d_model 256 and 512, so 512 and 1024 inner channels: 8 and 16 heads of 64; 256 byte values; 8 and 16 layers), chunk lengths
and chunk counts, and odd ones.
"""
import functools
import math
import os
import sys

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

VOCAB = 256
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST = 2 * 16384 * 8 * 64 * 64  # positions times heads times state values of the largest training pass
CHUNK = 64                      # positions that the plain form takes at once


def listed():
    return [
        # one token of one stream through a mixer of 8 heads: the smallest call there is, where latency counts
        {"name": "attention_step_1x8", "op": "attention", "mode": "step", "batch": 1, "heads": 8, "groups": 8, "key": 64, "value": 64,
         "decay": "token", "dtype": "f32"},
        # one token of each of the 1000 chunks of the command line's default, the larger model's 16 heads in bfloat16
        {"name": "attention_step_1000x16_bf16", "op": "attention", "mode": "step", "batch": 1000, "heads": 16, "groups": 16,
         "key": 64, "value": 64, "decay": "token", "dtype": "bf16"},
        # a few prompts of an odd length, continued from a state and handing one on; a fixed decay for each head
        {"name": "attention_prompt_4x4097x16_bf16", "op": "attention", "mode": "prompt", "batch": 4, "length": 4097, "heads": 16,
         "groups": 16, "key": 64, "value": 64, "decay": "head", "dtype": "bf16", "ragged": False},
        # an ordinary training batch of the d_model 256 model's size: forward and gradient
        {"name": "attention_train_8x1000x8", "op": "attention", "mode": "train", "batch": 8, "length": 1000, "heads": 8, "groups": 8,
         "key": 64, "value": 64, "decay": "token", "dtype": "f32", "ragged": False},
        # whole chunks of the headline's 16384 bytes: few sequences, so the work has to be split over the length
        {"name": "attention_train_2x16384x8", "op": "attention", "mode": "train", "batch": 2, "length": 16384, "heads": 8,
         "groups": 8, "key": 64, "value": 64, "decay": "token", "dtype": "f32", "ragged": False},
        # many short chunks of different lengths, padded to the longest, in bfloat16; four heads share their queries and keys
        {"name": "attention_train_32x500x16_bf16", "op": "attention", "mode": "train", "batch": 32, "length": 500, "heads": 16,
         "groups": 4, "key": 64, "value": 64, "decay": "token", "dtype": "bf16", "ragged": True},
        # the gradients of a model of one layer: little memory, so latency counts
        {"name": "clip_256x1", "op": "clip", "d_model": 256, "layers": 1, "dtype": "f32"},
        # of the headline's model
        {"name": "clip_256x8", "op": "clip", "d_model": 256, "layers": 8, "dtype": "f32"},
        # of the larger model, kept in bfloat16
        {"name": "clip_512x16_bf16", "op": "clip", "d_model": 512, "layers": 16, "dtype": "bf16"},
        # the next byte of one stream
        {"name": "sample_1x256", "op": "sample", "rows": 1, "vocab": VOCAB, "dtype": "f32", "limits": "one"},
        # of the headline's 4096 chunks
        {"name": "sample_4096x256", "op": "sample", "rows": 4096, "vocab": VOCAB, "dtype": "f32", "limits": "one"},
        # of 16384 chunks, logits in bfloat16 (many of them equal), each stream with its own temperature and limits
        {"name": "sample_16384x256_bf16", "op": "sample", "rows": 16384, "vocab": VOCAB, "dtype": "bf16", "limits": "rows"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "clip", "sample"])
    c = {"op": op, "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
    if op == "clip":
        return {**c, "d_model": rng.choice([256, 512, rng.randint(33, 500)]), "layers": _log(rng, 1, 16)}
    if op == "sample":
        vocab = rng.choice([VOCAB, VOCAB, rng.randint(2, 1000)])
        return {**c, "rows": _log(rng, 1, 16384 * VOCAB // max(vocab, VOCAB)), "vocab": vocab, "limits": rng.choice(["one", "rows"])}
    c["mode"] = rng.choice(["train", "train", "train", "prompt", "step"])
    share = rng.choice([1, 1, 2, 4])
    c["groups"] = rng.randint(1, 16 // share)
    c["heads"] = c["groups"] * share
    c["key"], c["value"] = (rng.choice([64, 64, 128, rng.randint(5, 128)]) for _ in range(2))
    c["decay"] = rng.choice(["token", "token", "head"])
    each = c["heads"] * max(64, c["key"]) * max(64, c["value"])
    if c["mode"] == "step":
        return {**c, "batch": _log(rng, 1, max(1, min(2000, 1000 * 16 * 64 * 64 // each)))}
    c["length"] = _log(rng, 2, min(16384, MOST // each))
    c["batch"] = _log(rng, 1, max(1, min(128, MOST // (each * c["length"]))))
    c["ragged"] = c["batch"] > 1 and rng.random() < 0.5
    return c


def _shapes(d, layers):
    """The parameters of this repository's model."""
    di, r, f = 2 * d, -(-d // 16), 4 * d
    block = [(d,), (d,), (2 * di, d), (di, 1, 4), (di,), (r + 32, di), (di, r), (di,), (di, 16), (di,), (d, di), (d,), (d,),
             (f, d), (f,), (d, f), (d,)]
    return [(VOCAB, d)] + block * layers + [(d, d), (d,), (VOCAB, d), (VOCAB,)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(mean)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    if case["op"] == "clip":
        # gradients of different sizes, one behind the other in one buffer, as a bucket for all of them has them; float16 ones
        # are scaled up, as mixed precision does
        shapes = _shapes(case["d_model"], case["layers"])
        flat = torch.empty(sum(math.prod(shape) for shape in shapes), dtype=dt, device="cuda")
        params, at = [], 0
        for n, shape in enumerate(shapes):
            p = torch.nn.Parameter(torch.zeros(shape, dtype=dt, device="cuda"))
            p.grad = flat[at:at + p.numel()].view(shape)
            p.grad.copy_(normal(*shape, scale=(64.0 if case["dtype"] == "f16" else 0.01) * (1 + n % 5)))
            params.append(p)
            at += p.numel()
        return {"op": "clip", "params": params, "flat": flat, "max_norm": 1.0}
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        s = {"op": "sample", "x": normal(n, v, scale=3.0).to(dt), "u": uniform(n)}
        if case["limits"] == "one":
            return {**s, "temperature": 0.8, "top_k": max(1, v // 5), "top_p": 0.95, "min_p": 0.002}
        top_k = torch.randint(0, v + 1, (n,), generator=g, device="cuda", dtype=torch.int32)  # 0: no limit
        temperature = uniform(n) * 1.5
        temperature[uniform(n) < 0.1] = 0.0  # some take the likeliest byte
        return {**s, "temperature": temperature, "top_k": top_k, "top_p": 0.3 + uniform(n) * 0.7, "min_p": uniform(n) * 0.05}

    n, heads, groups, key, value = (case[k] for k in ("batch", "heads", "groups", "key", "value"))
    train, step = case["mode"] == "train", case["mode"] == "step"
    lead = (n,) if step else (n, case["length"])
    if case["decay"] == "head":
        decay = torch.log1p(-torch.exp2(-4.0 - 4.0 * torch.arange(heads, device="cuda") / heads))
    else:  # from steps of 0.001 to 0.1 and rates of 1 to 16, as the scan's are
        rate = 1.0 + 15.0 * uniform(heads)
        decay = -torch.exp(uniform(*lead, heads) * math.log(100.0) + math.log(1e-3)) * rate
    s = {"op": "attention", "mode": case["mode"], "q": normal(*lead, groups, key).to(dt), "k": normal(*lead, groups, key).to(dt),
         "v": normal(*lead, heads, value).to(dt), "decay": decay, "lens": None, "state": None}
    if not train:
        s["state"] = normal(n, heads, key, value, scale=3.0)
        return s
    if case["ragged"]:
        s["lens"] = torch.randint(0, case["length"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["lens"][0] = case["length"]
    s["dy"] = normal(*lead, heads, value).to(dt)
    for name in ("q", "k", "v", "decay"):
        s[name] = s[name].detach().requires_grad_()
    s["leaves"] = tuple(s[name] for name in ("q", "k", "v", "decay"))
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
        return {"clip": _clip, "sample": _sample, "attention": _attention}[s["op"]](s)


def _own(s):
    ops = _ops()
    if s["op"] == "clip":
        return {"norm": ops.clip_grad_norm_(s["params"], s["max_norm"]), "grads": s["flat"]}
    if s["op"] == "sample":
        return {"token": ops.sample(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])}
    args = [s[k] for k in ("q", "k", "v", "decay")]
    if s["mode"] == "step":
        return {"y": ops.linear_attention_step(*args, state=s["state"]), "state": s["state"]}
    if s["mode"] == "prompt":
        y, state = ops.linear_attention(*args, state=s["state"], return_state=True)
        return {"y": y, "state": state}
    y = ops.linear_attention(*args, lens=s["lens"])
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, s["leaves"], s["dy"]))}


def _clip(s):
    grads = [p.grad for p in s["params"]]
    norm = torch.stack([(g.float() * g.float()).sum(dtype=torch.float64) for g in grads]).sum().sqrt()
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    [g.copy_(g.float() * scale) for g in grads]
    return {"norm": norm.float(), "grads": s["flat"]}


def _sample(s):
    """Weights of the symbols in 64 bits: what is cut off and what is drawn goes by whole sums next to a border."""
    n, v = s["x"].shape

    def column(t):
        return (t.double() if isinstance(t, torch.Tensor) else torch.full((n,), t, dtype=torch.float64, device="cuda"))[:, None]

    t, k, p, least = (column(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    x = s["x"].double()
    # the largest first, the lowest index first among equals
    order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((order.values - order.values[:, :1]) / torch.where(t > 0, t, 1.0))
    at = torch.arange(v, device="cuda")
    w = torch.where((k > 0) & (at >= k) | (t <= 0) & (at > 0), 0.0, w)
    before = torch.cumsum(w, 1) - w
    w = torch.where((before < p * w.sum(1, keepdim=True)) & (w >= least), w, 0.0)
    w[:, 0] = 1.0
    w = torch.zeros_like(w).scatter_(1, order.indices, w)
    upto = torch.cumsum(w, 1)
    drawn = upto > s["u"].double()[:, None] * upto[:, -1:]
    return {"token": torch.where(drawn, at, v).amin(1)}


def _heads(t, heads):
    """[batch, length, groups, d] of the positions in 32 bits as [batch, heads, chunks, CHUNK, d], zeros behind the end."""
    t = t.float().repeat_interleave(heads // t.shape[2], 2).transpose(1, 2)
    t = torch.nn.functional.pad(t, (0, 0, 0, -t.shape[2] % CHUNK))
    return t.reshape(t.shape[0], heads, -1, CHUNK, t.shape[3])


def _back(t, length, groups):
    """The reverse, summed over the heads that share a group."""
    n, heads, d = t.shape[0], t.shape[1], t.shape[4]
    t = t.reshape(n, heads, -1, d)[:, :, :length].transpose(1, 2)
    return t.reshape(n, length, groups, heads // groups, d).sum(3)


def _attention(s):
    dt, q, k, v, g = s["q"].dtype, s["q"], s["k"], s["v"], s["decay"]
    heads, groups, scale = v.shape[-2], q.shape[-2], q.shape[-1] ** -0.5
    if s["mode"] == "step":
        q, k = (t.float().repeat_interleave(heads // groups, 1) for t in (q, k))
        h = torch.exp(g)[..., None, None] * s["state"] + k[..., None] * v.float()[:, :, None]
        s["state"].copy_(h)
        return {"y": ((q * scale)[..., None] * h).sum(2).to(dt), "state": s["state"]}
    n, length = v.shape[:2]
    inside = torch.ones((n, length, 1, 1), dtype=torch.bool, device="cuda")
    if s["lens"] is not None:
        inside = (torch.arange(length, device="cuda") < s["lens"][:, None])[..., None, None]
    q, k, v = (_heads(torch.where(inside, t, torch.zeros_like(t)), heads) for t in (q, k, v))
    q = q * scale
    g = torch.where(inside[..., 0], g.double(), 0.0)
    g = _heads(g[..., None], heads)[..., 0].double()  # [batch, heads, chunks, CHUNK]
    total = torch.cumsum(g.reshape(n, heads, -1), 2).reshape(g.shape)  # log of the decay up to and with a position
    start = total[..., :1] - g[..., :1]  # before the chunk
    end = total[..., -1:]
    causal = torch.ones((CHUNK, CHUNK), dtype=torch.bool, device="cuda").tril()
    w = torch.exp(torch.where(causal, total[..., :, None] - total[..., None, :], -math.inf)).float()
    into, out = torch.exp(total - start).float()[..., None], torch.exp(end - total).float()[..., None]
    chunks = g.shape[2]
    # from the end of one chunk to the start of another
    apart = start[..., 0][..., :, None] - end[..., 0][..., None, :]
    join = torch.exp(torch.where(torch.ones_like(apart, dtype=torch.bool).tril(-1), apart, -math.inf)).float()
    own_states = (k * out).transpose(-1, -2).contiguous() @ v  # [.., key, value] that a chunk leaves
    flat = own_states.shape[:3] + (-1,)
    states = (join @ own_states.reshape(flat)).reshape(own_states.shape)  # before each chunk
    if s["state"] is not None:
        states = states + torch.exp(start).float()[..., None] * s["state"][:, :, None]
    a = (q @ k.transpose(-1, -2).contiguous()) * w
    y = a @ v + (q * into) @ states
    y = _back(y, length, heads)
    y = torch.where(inside, y, torch.zeros_like(y)).to(dt)
    if s["mode"] == "prompt":
        last = torch.exp(end - start).float()[:, :, -1, :, None] * states[:, :, -1] + own_states[:, :, -1]
        return {"y": y, "state": last}
    dy = s["dy"]
    dy = _heads(torch.where(inside, dy, torch.zeros_like(dy)), heads)
    own_grads = (q * into).transpose(-1, -2).contiguous() @ dy
    grads = (join.transpose(-1, -2).contiguous() @ own_grads.reshape(flat)).reshape(own_grads.shape)  # for the state behind each chunk
    qk, dyv = q @ k.transpose(-1, -2).contiguous(), dy @ v.transpose(-1, -2).contiguous()
    da = dyv * w
    dq_far = into * (dy @ states.transpose(-1, -2).contiguous())
    dk_far = out * (v @ grads.transpose(-1, -2).contiguous())
    dq = da @ k + dq_far
    dk = da.transpose(-1, -2).contiguous() @ q + dk_far
    dv = a.transpose(-1, -2).contiguous() @ dy + out * (k @ grads)
    # what depends on the decay of a position: every pair that it lies between, in this chunk, from before it, to behind it
    m = qk * dyv * w
    rows, columns = m.sum(-1) + (q * dq_far).sum(-1), m.sum(-2)
    later = (rows - columns).flip(-1).cumsum(-1).flip(-1)
    over = (k * dk_far).sum(-1)
    earlier = over.cumsum(-1) - over
    through = torch.exp(end - start).float()[..., 0] * (states * grads).sum((-1, -2))
    dg = _back((later + earlier + through[..., None])[..., None], length, heads)[..., 0]
    dg = torch.where(inside[..., 0], dg, torch.zeros_like(dg))
    dg = dg.sum(1).sum(0) if s["decay"].ndim == 1 else dg
    return {"y": y, "grads": [_back(dq * scale, length, groups).to(dt), _back(dk, length, groups).to(dt),
                              _back(dv, length, heads).to(dt), dg]}


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "clip":
        count = sum(math.prod(shape) for shape in _shapes(case["d_model"], case["layers"]))
        return {"bytes": 2 * count * es, "flops": 3 * count}
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * (v * es + 12 + (16 if case["limits"] == "rows" else 0)), "flops": 8 * n * v}
    n, heads, groups, key, value = (case[k] for k in ("batch", "heads", "groups", "key", "value"))
    positions, train = n * case.get("length", 1), case["mode"] == "train"
    decay = 4 * heads * (1 if case["decay"] == "head" else positions) * (2 if train else 1)
    state = 0 if train else 2 * n * heads * key * value * 4
    # q, k, v in, y out; with the gradient dy in and those of q, k, v out
    rows = positions * es * (groups * key * (4 if train else 2) + heads * value * (4 if train else 2))
    # a state's update and its product with q, per position; backward both again with their gradients
    return {"bytes": rows + decay + state, "flops": positions * heads * key * value * (14 if train else 4)}


def exact(case, seed):
    """The operators' definitions in 64 bits: attention with all pairs of positions at once, its gradient by differentiation.
    Symbols are whole numbers and have no such value."""
    s = prepare(case, seed)
    if case["op"] == "sample":
        return None
    if case["op"] == "clip":
        grads = s["flat"].double()
        norm = torch.dot(grads, grads) ** 0.5
        return {"norm": norm, "grads": grads * min(1.0, s["max_norm"] / (norm.item() + 1e-6))}
    q, k, v, g = (s[name].detach().double() for name in ("q", "k", "v", "decay"))
    heads, share = v.shape[-2], v.shape[-2] // q.shape[-2]
    scale = 1.0 / math.sqrt(q.shape[-1])
    if case["mode"] == "step":
        q, k = (t.repeat_interleave(share, 1) for t in (q, k))
        state = torch.exp(g)[..., None, None] * s["state"].double() + torch.einsum("bhn,bhp->bhnp", k, v)
        return {"y": torch.einsum("bhn,bhnp->bhp", q * scale, state), "state": state}
    n, length = v.shape[:2]
    ends = [length] * n if s["lens"] is None else s["lens"].tolist()
    train = case["mode"] == "train"
    y, state = torch.zeros_like(v), None if train else torch.zeros_like(s["state"], dtype=torch.float64)
    grads = [torch.zeros_like(t) for t in (q, k, v, g)]
    for b in range(n):
        for h in range(heads):
            at = slice(0, ends[b])
            parts = [q[b, at, h // share], k[b, at, h // share], v[b, at, h], g[h].expand(ends[b]) if g.ndim == 1 else g[b, at, h]]
            parts = [t.clone().requires_grad_(train) for t in parts]
            qh, kh, vh, gh = parts
            upto = gh.cumsum(0)
            pairs = (upto[:, None] - upto[None]).masked_fill_(torch.ones((ends[b], ends[b]), dtype=torch.bool, device="cuda").triu_(1), -math.inf)
            yh = (pairs.exp_() * (qh @ kh.t())) @ vh * scale
            if not train:
                first = s["state"][b, h].double()
                yh = yh + upto.exp()[:, None] * (qh @ first) * scale
                state[b, h] = (upto[-1].exp() * first + (kh * (upto[-1] - upto).exp()[:, None]).t() @ vh) if ends[b] else first
            elif ends[b]:
                dq, dk, dv, dg = torch.autograd.grad(yh, parts, s["dy"][b, at, h].double())
                grads[0][b, at, h // share] += dq
                grads[1][b, at, h // share] += dk
                grads[2][b, at, h] = dv
                if g.ndim == 1:
                    grads[3][h] += dg.sum()
                else:
                    grads[3][b, at, h] = dg
            y[b, at, h] = yh.detach()
    return {"y": y, "grads": grads} if train else {"y": y, "state": state}
