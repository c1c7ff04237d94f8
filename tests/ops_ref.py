"""The training operators from their formulas in 64 bits (CPU, position by position), each result with its magnitude: the same
sums over absolute values, in whose units rounding errors are bounded."""
import torch

F64 = torch.float64


def d(t):
    return None if t is None else t.detach().to("cpu", F64)


def ends_of(lens, n, length):
    return [length] * n if lens is None else [max(0, min(length, int(v))) for v in lens.tolist()]


def norm(x, w, b, dy, eps=1e-5):
    x, dy = d(x), d(dy)
    n, k = x.shape
    w = torch.ones(k, dtype=F64) if w is None else d(w)
    b = torch.zeros(k, dtype=F64) if b is None else d(b)
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh, xm = (x - mean) * rstd, ((x - mean).abs() + x.abs().mean(1, keepdim=True)) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    dxm = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xm * (g.abs() * xm).mean(1, keepdim=True))
    return {"y": (xh * w + b, xm * w.abs() + b.abs()), "dx": (dx, dxm), "dw": ((dy * xh).sum(0), (dy.abs() * xm).sum(0)),
            "db": (dy.sum(0), dy.abs().sum(0))}


def loss(x, target, ignore, reduction, up):
    """up: the upstream gradient, one value or one per row."""
    x, t = d(x), target.cpu().long()
    v = x.shape[1]
    kept = t != ignore
    bad = kept & ((t < 0) | (t >= v))
    m = x.max(1, keepdim=True).values
    e = torch.exp(x - m)
    p = e / e.sum(1, keepdim=True)
    xt = x.gather(1, t.clamp(0, v - 1)[:, None])[:, 0]
    each = torch.log(e.sum(1)) + m[:, 0] - xt
    mag = 1 + torch.log(e.sum(1)).abs() + m[:, 0].abs() + xt.abs()
    each = torch.where(bad, torch.full_like(each, float("nan")), each)
    each, mag = torch.where(kept, each, torch.zeros_like(each)), torch.where(kept, mag, torch.zeros_like(mag))
    hit = torch.zeros_like(x).scatter_(1, t.clamp(0, v - 1)[:, None], 1.0)
    scale = torch.as_tensor(up, dtype=F64).reshape(-1, 1).expand(len(x), 1) / (kept.sum() if reduction == "mean" else 1)
    dx = (p - hit) * scale
    dx = torch.where(bad[:, None], torch.full_like(dx, float("nan")), dx)
    dx = torch.where(kept[:, None], dx, torch.zeros_like(dx))
    y = (each, mag) if reduction == "none" else (each.sum() / (kept.sum() if reduction == "mean" else 1),
                                                 mag.sum() / (kept.sum() if reduction == "mean" else 1))
    return {"y": y, "dx": (dx, (p + hit) * scale.abs())}


def conv(x, w, b, silu=True, state=None, lens=None, dy=None):
    x, w, dy, state = d(x), d(w).reshape(-1, 4), d(dy), d(state)
    n, length, c = x.shape
    b = torch.zeros(c, dtype=F64) if b is None else d(b)
    state = torch.zeros(n, 3, c, dtype=F64) if state is None else state
    z = torch.zeros(n, length, c, dtype=F64)
    y, ym, dx, dxm, end_state = z.clone(), z.clone(), z.clone(), z.clone(), torch.zeros_like(state)
    dw, db = torch.zeros(2, c, 4, dtype=F64), torch.zeros(2, c, dtype=F64)
    for i, end in enumerate(ends_of(lens, n, length)):
        row = torch.cat([state[i], x[i, :end]])
        end_state[i] = row[end:end + 3]
        win = torch.stack([row[k:k + end] for k in range(4)], -1)
        p, pm = (win * w).sum(-1) + b, (win * w).abs().sum(-1) + b.abs()
        sig = torch.sigmoid(p)
        y[i, :end], ym[i, :end] = (p * sig, pm) if silu else (p, pm)
        if dy is None:
            continue
        slope = sig + p * sig * (1 - sig) if silu else torch.ones_like(p)
        g, gm = dy[i, :end] * slope, dy[i, :end].abs() * (1 + pm)
        db += torch.stack([g.sum(0), gm.sum(0)])
        dw += torch.stack([(g[..., None] * win).sum(0), (gm[..., None] * win.abs()).sum(0)])
        for k in range(4):  # position t's window holds position t - 3 + k
            s = 3 - k
            if end > s:
                dx[i, :end - s] += g[s:] * w[:, k]
                dxm[i, :end - s] += gm[s:] * w[:, k].abs()
    out = {"y": (y, ym), "state": (end_state, torch.zeros_like(end_state))}
    if dy is not None:
        out.update(dx=(dx, dxm), dw=(dw[0], dw[1]), db=(db[0], db[1]))
    return out


def scan(u, delta, A, B, C, D=None, z=None, bias=None, state=None, lens=None, dy=None):
    u, delta, A, B, C, z, dy, state = (d(t) for t in (u, delta, A, B, C, z, dy, state))
    n, length, c = u.shape
    D = torch.zeros(c, dtype=F64) if D is None else d(D)
    bias = torch.zeros(c, dtype=F64) if bias is None else d(bias)
    h0 = torch.zeros(n, 16, c, dtype=F64) if state is None else state
    zero = torch.zeros(n, length, c, dtype=F64)
    res = {k: (zero.clone(), zero.clone()) for k in ("y", "du", "ddelta", "dz")}
    res.update({k: (torch.zeros(n, length, 16, dtype=F64), torch.zeros(n, length, 16, dtype=F64)) for k in ("dB", "dC")})
    res.update({k: (torch.zeros(s, dtype=F64), torch.zeros(s, dtype=F64)) for k, s in (("dA", (c, 16)), ("dD", c), ("dbias", c))})
    res["state"] = (h0.clone(), h0.abs())
    for i, end in enumerate(ends_of(lens, n, length)):
        h, hm = h0[i].t(), h0[i].t().abs()  # [c, 16]
        pre = delta[i, :end] + bias
        dt = torch.logaddexp(pre, torch.zeros_like(pre))
        sig = torch.sigmoid(pre)
        gate = torch.sigmoid(z[i, :end]) * z[i, :end] if z is not None else torch.ones(end, c, dtype=F64)
        zs = torch.sigmoid(z[i, :end]) if z is not None else None
        past, y0s, y0m = [], [], []
        for t in range(end):
            past.append((h, hm))
            e, x = torch.exp(dt[t, :, None] * A), (dt[t] * u[i, t])[:, None] * B[i, t]
            h, hm = e * h + x, e * hm + x.abs()
            y0s.append(h @ C[i, t] + D * u[i, t])
            y0m.append(hm @ C[i, t].abs() + (D * u[i, t]).abs())
            res["y"][0][i, t], res["y"][1][i, t] = y0s[t] * gate[t], y0m[t] * gate[t].abs()
        res["state"][0][i], res["state"][1][i] = h.t(), hm.t()
        if dy is None:
            continue
        dh, dhm = torch.zeros(c, 16, dtype=F64), torch.zeros(c, 16, dtype=F64)
        for t in range(end - 1, -1, -1):
            e, x = torch.exp(dt[t, :, None] * A), (dt[t] * u[i, t])[:, None] * B[i, t]
            g, (before, bm) = dy[i, t] * gate[t], past[t]
            now, nm = e * before + x, e * bm + x.abs()
            dh, dhm = dh + g[:, None] * C[i, t], dhm + (g[:, None] * C[i, t]).abs()
            flow, fm = dh * e * before, dhm * e * bm
            sB, sm = dh @ B[i, t], dhm @ B[i, t].abs()
            for k, v, m in (("dC", g @ now, g.abs() @ nm), ("dB", (dt[t] * u[i, t]) @ dh, (dt[t] * u[i, t]).abs() @ dhm),
                            ("du", dt[t] * sB + D * g, dt[t] * sm + (D * g).abs()),
                            ("ddelta", sig[t] * (u[i, t] * sB + (flow * A).sum(1)),
                             sig[t] * (u[i, t].abs() * sm + (fm * A.abs()).sum(1)))):
                res[k][0][i, t], res[k][1][i, t] = v, m
            if z is not None:
                slope = zs[t] * (1 + z[i, t] * (1 - zs[t]))
                res["dz"][0][i, t], res["dz"][1][i, t] = dy[i, t] * y0s[t] * slope, dy[i, t].abs() * y0m[t] * (1 + z[i, t].abs())
            for k, v, m in (("dA", flow * dt[t][:, None], fm * dt[t][:, None]), ("dD", g * u[i, t], (g * u[i, t]).abs()),
                            ("dbias", res["ddelta"][0][i, t], res["ddelta"][1][i, t])):
                res[k][0].add_(v)
                res[k][1].add_(m)
            dh, dhm = dh * e, dhm * e
    keep = ["y", "state"] + (["du", "ddelta", "dB", "dC", "dA", "dD", "dbias"] + (["dz"] if z is not None else []) if dy is not None else [])
    return {k: res[k] for k in keep}
