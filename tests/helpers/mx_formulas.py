"""The block seam and the microscaled formats written out in 64 bits, for the operators' tests (any device)."""
import math

import torch

D = torch.float64
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step of the type, relative
MAX = {4: 6.0, 8: 448.0}


def grid(bits):
    if bits == 4:
        return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=D)
    sub = [m / 8 * 2.0 ** -6 for m in range(8)]
    return torch.tensor(sub + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1], dtype=D)


def held(x, bits):
    """-> (values [rows, n], exponent bytes [rows, blocks]) of x packed by definition; blocks with NaN or infinity: NaN, 255."""
    rows, n = x.shape
    b = torch.zeros((rows, -(-n // 32) * 32), dtype=D, device=x.device)
    b[:, :n] = x.to(D)
    b = b.view(rows, -1, 32)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], torch.zeros_like(b), b)
    a = b.abs().amax(-1)
    e = torch.full(a.shape, -110, dtype=torch.int64, device=x.device)
    for k in range(-110, 128):
        e = torch.where(a > MAX[bits] * 2.0 ** k, k + 1, e)
    v = b.abs() / torch.exp2(e.to(D))[..., None]
    g = grid(bits).to(x.device)
    hi = torch.searchsorted(g, v).clamp(max=g.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = g[hi] - v, v - g[lo]
    at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    out = torch.sign(b) * g[at] * torch.exp2(e.to(D))[..., None]
    out = torch.where(bad[..., None], torch.full_like(out, math.nan), out)
    return out.view(rows, -1)[:, :n], torch.where(bad, 255, e + 127).to(torch.uint8)


def act(x, kind):
    """-> (act(x), act'(x))"""
    if kind == "gelu":
        cdf = 0.5 * torch.special.erfc(-x / math.sqrt(2.0))
        return x * cdf, cdf + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(1.702 * x)
    return x * s, s * (1 + 1.702 * x * (1 - s))


def stats(t, norm, eps):
    mean = t.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(t[:, :1])
    return mean, 1.0 / torch.sqrt(((t - mean) ** 2).mean(-1, keepdim=True) + eps)


def spread_gate(gate, rows, d):
    g = gate.to(D)
    g = g[:, None].expand(-1, d) if g.dim() == 1 else g
    return g.repeat_interleave(rows // g.shape[0], 0)


def seam_fwd(x, h, post, pre, gate, scale, alpha, norm, eps):
    """-> y in 64 bits and the magnitudes that its rounding errors are relative to."""
    x, h = x.to(D), h.to(D)
    rows, d = x.shape
    p, mag = h, h.abs()
    if post is not None:
        mean, rstd = stats(h, norm, eps)
        p = (h - mean) * rstd * post[0].to(D)
        mag = post[0].to(D).abs() * (rstd * (h.abs() + h.abs().mean(-1, keepdim=True)))
        if post[1] is not None:
            p, mag = p + post[1].to(D), mag + post[1].to(D).abs()
    m = torch.ones((rows, d), dtype=D, device=x.device) if gate is None else spread_gate(gate, rows, d)
    m = m if scale is None else m * scale.to(D)
    y = alpha * x + torch.where(m == 0, torch.zeros_like(p), m * p)
    return y, (alpha * x).abs() + torch.where(m == 0, torch.zeros_like(p), (m * mag).abs())


def seam_norm(y, pre, norm, eps):
    y = y.to(D)
    mean, rstd = stats(y, norm, eps)
    z = (y - mean) * rstd * pre[0].to(D)
    mag = pre[0].to(D).abs() * rstd * (y.abs() + y.abs().mean(-1, keepdim=True))
    if pre[1] is not None:
        z, mag = z + pre[1].to(D), mag + pre[1].to(D).abs()
    return z, mag


def seam_bwd(dy, dz, h, y, post, pre, gate, scale, alpha, norm, eps):
    """-> {name: (gradient, magnitude of the terms it is summed from)} from the formulas."""
    h = h.to(D)
    rows, d = h.shape
    out = {}
    z0 = torch.zeros((rows, d), dtype=D, device=h.device)
    gy = dy.to(D) if dy is not None else z0
    mag = gy.abs()

    def norm_bwd(dn, dn_mag, t, w):
        mean, rstd = stats(t, norm, eps)
        hat = (t - mean) * rstd
        u, um = dn * w, dn_mag * w.abs()
        hm = (t.abs() + t.abs().mean(-1, keepdim=True)) * rstd  # what hat's own error is relative to
        m1 = u.mean(-1, keepdim=True) if norm == "layer" else 0.0 * u[:, :1]
        m2 = (u * hat).mean(-1, keepdim=True)
        g = rstd * (u - m1 - hat * m2)
        gm = rstd * (um + um.mean(-1, keepdim=True) + hm * (um * hm).mean(-1, keepdim=True))
        return g, gm, ((dn * hat).sum(0), (dn_mag * hm).sum(0)), (dn.sum(0), dn_mag.sum(0)), hat, hm

    if pre is not None:
        g, gm, w, b, _, _ = norm_bwd(dz.to(D), dz.to(D).abs(), y.to(D), pre[0].to(D))
        gy, mag = gy + g, mag + gm
        out["pre_w"] = w
        if pre[1] is not None:
            out["pre_b"] = b
    out["x"] = (alpha * gy, abs(alpha) * mag)
    one = torch.ones((rows, d), dtype=D, device=h.device)
    g = one if gate is None else spread_gate(gate, rows, d)
    s = one if scale is None else scale.to(D) * one
    p, pm = h, h.abs()
    if post is not None:
        mean, rstd = stats(h, norm, eps)
        p = (h - mean) * rstd * post[0].to(D)
        pm = (h.abs() + h.abs().mean(-1, keepdim=True)) * rstd * post[0].to(D).abs()
        if post[1] is not None:
            p, pm = p + post[1].to(D), pm + post[1].to(D).abs()
    dead = lambda t, k: torch.where(k == 0, torch.zeros_like(t), t)  # noqa: E731
    if scale is not None:
        out["scale"] = (dead(g * p * gy, g).sum(0), dead(g.abs() * pm * mag, g).sum(0))
    if gate is not None:
        groups = gate.shape[0]
        t, tm = (s * p * gy).view(groups, -1, d).sum(1), (s.abs() * pm * mag).view(groups, -1, d).sum(1)
        out["gate"] = (t.sum(-1), tm.sum(-1)) if gate.dim() == 1 else (t, tm)
    m = g * s
    dp, dm = m * gy, m.abs() * mag
    if post is None:
        out["h"] = (dp, dm)
    else:
        live = ~(m == 0).all(-1, keepdim=True)
        hz = torch.where(live, h, torch.zeros_like(h))
        gh, gm, w, b, _, _ = norm_bwd(dp, dm, hz, post[0].to(D))
        out["h"], out["post_w"] = (gh, gm), w
        if post[1] is not None:
            out["post_b"] = b
    return out
