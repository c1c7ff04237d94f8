"""The selective scan and its gradient from the formulas in 64 bits, all positions' terms at once and only the two recurrences
position by position (on any device), each result with a bound of what float32 arithmetic may be off by.

The bound is carried along the recurrences, so that it counts a rounding by what it does to the result.  Unit: e = 2^-24, a
rounding to nearest in float32; a hardware exponential, logarithm or reciprocal is off by one unit in the last place, 2 e.
  pre = delta + bias is rounded once; exp(-|pre|) has its argument's two roundings (2 |pre| e) and 2 e; softplus from it is off by
    rho e dt, rho = 3 |pre| + 12 (|pre| of pre's own rounding, as softplus' <= softplus; 2 |pre| + 2 of the exponential; 8 of
    the logarithm, the reciprocal and their products; the last sum), and sigmoid(pre) by rs e, rs = 3 |pre| + 8
  exp(dt A): its argument's rounding counts by the argument's size, |dt A| (rho + 3) e, and 2 e of the exponential.  Where the length
    is split, a chunk's decay is exp of a sum of up to `chunk` steps, added one by one (and 32 such sums): |dt A| (chunk + 32) e more for
    each of its positions
  h = exp(dt A) h + B dt u: three roundings of B dt u, one each of the product and the sum, two where chunks meet
  z sigmoid(z) is off by rg e, rg = 2 |z| + 6
  sums: one rounding per addition on the longest way to the result, in the magnitudes of what is added: 16 states 4 + 4, the
    lanes of a wavefront 6, blocks of channels one by one, positions as the comments below say
Magnitudes are the same sums over absolute values.  Terms of second order are left out; the bound is taken 2^-6 wider for them.
"""
import torch

E24 = 2.0 ** -24


def _rows(t, live):
    """[length, batch, ...] in 64 bits, zeros behind the ends (whatever is there)."""
    t = t.detach().double().transpose(0, 1)
    return torch.where(live, t, torch.zeros((), dtype=t.dtype, device=t.device))


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, *, state=None, lens=None, dy=None, chunk=0, parts=1):
    """{name: (value, bound in units of 2^-24)}.  chunk: positions that are summed before chunks are joined; parts: partial sums
    that the parameters' gradients are added from (sequences times chunks)."""
    n, length, c = u.shape
    dev = u.device
    zero = torch.zeros((), dtype=torch.float64, device=dev)
    ends = torch.full((n,), length, device=dev) if lens is None else lens.to(dev).long().clamp(0, length)
    live = (torch.arange(length, device=dev)[:, None] < ends)[..., None]  # [length, batch, 1]
    u, delta, B, C = (_rows(t, live) for t in (u, delta, B, C))
    z = None if z is None else _rows(z, live)
    A = A.detach().double()
    D = torch.zeros(c, dtype=A.dtype, device=dev) if D is None else D.detach().double()
    bias = torch.zeros(c, dtype=A.dtype, device=dev) if delta_bias is None else delta_bias.detach().double()
    h0 = torch.zeros(n, c, 16, dtype=A.dtype, device=dev) if state is None else state.detach().double().transpose(1, 2)
    cblocks = -(-c // 64)

    pre = torch.where(live, delta + bias, zero)
    rho, rs = 3 * pre.abs() + 12, 3 * pre.abs() + 8
    dt = torch.where(live, torch.logaddexp(pre, zero), zero)
    sig = torch.where(live, torch.sigmoid(pre), zero)
    dtu = dt * u
    arg = dt[..., None] * A                                     # [length, batch, channels, 16]
    e = torch.exp(arg)
    x = dtu[..., None] * B[:, :, None]
    once = arg.abs() * (rho[..., None] + 3) + 2                 # of one exponential
    split = once + arg.abs() * (chunk + 32 if chunk else 0)

    h, hm, he = (torch.empty_like(x) for _ in range(3))         # behind each position: value, magnitude, bound
    p, pm, pe = h0, h0.abs(), torch.zeros_like(h0)
    for t in range(length):
        torch.addcmul(x[t], e[t], p, out=h[t])
        torch.addcmul(x[t].abs(), e[t], pm, out=hm[t])
        now = e[t] * (pe + pm * split[t]) + x[t].abs() * (rho[t, ..., None] + 3) + 4 * hm[t]
        torch.where(live[t, ..., None], now, pe, out=he[t])     # behind the end the state stays as it is
        p, pm, pe = h[t], hm[t], he[t]
    out = {"state": (p.transpose(1, 2), pe.transpose(1, 2))}

    gate, rg = (torch.ones_like(u), torch.zeros_like(u)) if z is None else (z * torch.sigmoid(z), 2 * z.abs() + 6)
    Ca, Ba, Du = C.abs()[:, :, None], B.abs()[:, :, None], D * u
    y0, y0m = (h * C[:, :, None]).sum(-1) + Du, (hm * Ca).sum(-1) + Du.abs()
    y0e = ((he + 12 * hm) * Ca).sum(-1) + 8 * Du.abs()
    here = lambda t: torch.where(live, t, zero)  # noqa: E731
    out["y"] = (here(y0 * gate), here(gate.abs() * (y0e + (rg + 1) * y0m)))

    if dy is not None:
        dy = _rows(dy, live)
        g = dy * gate
        ge = g.abs() * (rg + 2) if z is not None else torch.zeros_like(g)
        d, dm, de = (torch.empty_like(x) for _ in range(3))     # adjoint of h at each position, its own output's part included
        p = pm = pe = torch.zeros_like(h0)                      # the adjoint behind it, on its way back
        for t in range(length - 1, -1, -1):
            own = g[t, ..., None] * C[t, :, None]
            torch.add(own, p, out=d[t])
            torch.add(own.abs(), pm, out=dm[t])
            torch.add(Ca[t] * (ge[t] + g[t].abs())[..., None] + pe, 4 * dm[t], out=de[t])
            p, pm, pe = e[t] * d[t], e[t] * dm[t], e[t] * (de[t] + dm[t] * split[t])
        ga, dtua, ua = g.abs()[..., None], dtu.abs()[..., None], u.abs()
        over = 8 + cblocks                                      # lanes, then blocks of channels
        out["dC"] = ((g[..., None] * h).sum(2), (ga * he + (ge[..., None] + (1 + over) * ga) * hm).sum(2))
        out["dB"] = ((dtu[..., None] * d).sum(2), (dtua * (de + (rho[..., None] + 3 + over) * dm)).sum(2))
        sB, sBm, sBe = (d * B[:, :, None]).sum(-1), (dm * Ba).sum(-1), ((de + 12 * dm) * Ba).sum(-1)
        out["du"] = (dt * sB + D * g, dt * (sBe + (rho + 3) * sBm) + D.abs() * (ge + 4 * g.abs()))
        before = lambda t, first: torch.cat([first[None], t[:-1]])  # noqa: E731
        hb, hbm, hbe = before(h, h0), before(hm, h0.abs()), before(he, torch.zeros_like(h0))
        w, wm = d * e * hb, dm * e * hbm
        we = e * (de * hbm + dm * (hbe + hbm * once)) + 3 * wm
        Aa = A.abs()
        sw, swm, swe = (w * A).sum(-1), (wm * Aa).sum(-1), ((we + 14 * wm) * Aa).sum(-1)
        ddm = sig * (ua * sBm + swm)
        out["ddelta"] = (sig * (u * sB + sw), sig * (ua * (sBe + 2 * sBm) + swe) + (rs + 3) * ddm)
        if z is not None:
            s = torch.sigmoid(z)
            slope, r = s + z * s * (1 - s), 2 * z.abs() + 6
            slope_e = z.abs() * s * ((r + 1) * (1 - s) + s * r + 1) + s * r + slope.abs()
            out["dz"] = (dy * y0 * slope, dy.abs() * (y0e * slope.abs() + y0m * (slope_e + 3 * slope.abs())))
        # 64 positions in one register, those sums of a chunk in another, then every eighth of the parts
        tail = parts / 8 + 32
        deep = 64 + chunk / 64 + tail if chunk else 64 + length / 64 + tail
        out["dA"] = ((w * dt[..., None]).sum((0, 1)), (dt[..., None] * (we + (rho[..., None] + 2 + deep) * wm)).sum((0, 1)))
        # a wavefront has every fourth position of a chunk in one register
        deep = (chunk or length) / 4 + 8 + tail
        out["dD"] = ((g * u).sum((0, 1)), (ua * (ge + (1 + deep) * g.abs())).sum((0, 1)))
        out["dbias"] = (out["ddelta"][0].sum((0, 1)), (out["ddelta"][1] + deep * ddm).sum((0, 1)))
    turn = ("y", "du", "ddelta", "dz", "dB", "dC")
    return {k: (v.transpose(0, 1), b.transpose(0, 1)) if k in turn else (v, b) for k, (v, b) in out.items()}


def worst(got, ref, dtype=None):
    """The largest error in units of what is allowed: the float32 bound, and half a step of the type that the result is rounded to."""
    value, bound = ref
    dtype = dtype or got.dtype
    info = torch.finfo(dtype)
    assert got.shape == value.shape and got.dtype == dtype, (got.shape, value.shape, got.dtype)
    if not got.numel():
        return 0.0
    bound = (1 + 2.0 ** -6) * E24 * bound
    allowed = info.eps / 2 * (value.abs() + bound) * (dtype != torch.float32) + bound + E24 * value.abs() + info.tiny * info.eps
    over = (got.detach().to(value.device).double() - value).abs() / allowed
    return float(over.max()) if not over.isnan().any() else float("nan")
