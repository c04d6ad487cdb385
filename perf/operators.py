"""What the block-seam and microscaled-number operators are measured on: the cases, their inputs, the plain forms in
elementary torch operations, and their definitions in 64 bits.

Three operators, which one transformer block uses together:

  seam     y = alpha x + gate * scale * Norm_post(h),  z = Norm_pre(y), forward and backward
  act8     a checkpoint in 8 bits (e4m3, blocks of 32 with a power-of-two scale) through an activation, and the weight
           gradient taken from such a checkpoint
  mx       4- and 8-bit microscaled numbers: quantisation, and the product of two packed matrices
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_MAX = {4: 6.0, 8: 448.0}
EPS = 1e-5


def _seam(kind, rows, d, **kw):
    case = dict(kind=kind, rows=rows, d=d, norm="layer", post=True, pre=True, gate="none", groups=1, scale=True, x="fp32",
                h="bf16", alpha=1.0)
    case.update(kw)
    return case


def listed():
    return [
        # one image through a block of the patch-32 tower: 50 tokens, a residual scale per channel, the next block's norm
        dict(_seam("seam_fwd", 50, 768, post=False), name="seam_fwd_image"),
        # 64 images of the patch-14 tower (257 tokens) with norms on both sides of the block and stochastic depth per image
        dict(_seam("seam_fwd", 64 * 257, 1024, gate="group", groups=64), name="seam_fwd_large"),
        # training the patch-16 tower (197 tokens) on 64 images, every gradient
        dict(_seam("seam_bwd", 64 * 197, 768, gate="group", groups=64), name="seam_bwd_batch"),
        # 31 captions of 77 tokens, an odd width, a bf16 stream, root-mean-square norms and a gate per caption and channel
        dict(_seam("seam_bwd", 31 * 77, 509, norm="rms", gate="channel", groups=31, x="bf16", alpha=0.75), name="seam_bwd_odd"),
        # one caption's MLP activation (text tower width 512, MLP 2048): latency
        dict(kind="act8", rows=77, n=2048, act="quick_gelu", name="act8_caption"),
        # the MLP activation of a 32-image step of the patch-14 tower, there and back
        dict(kind="act8", rows=32 * 257, n=4096, act="gelu", name="act8_large"),
        # out_proj's weight gradient of a 32-image step of the patch-32 tower
        dict(kind="wgrad8", rows=32 * 50, n=768, k=768, name="wgrad8_step"),
        # c_fc's weight gradient of a 64-image step of the patch-14 tower
        dict(kind="wgrad8", rows=64 * 257, n=4096, k=1024, name="wgrad8_large"),
        # a tower's MLP weight into 4 bits, and the values that it then stands for
        dict(kind="quant", rows=4096, k=1024, bits=4, x="fp32", name="quant4_weight"),
        # one row against a 4-bit weight: latency and the weight's bytes
        dict(kind="matmul", rows=1, n=4096, k=1024, abits=4, bbits=4, bias=True, name="product_row"),
        # 107 captions, 8-bit rows, 4-bit weights, a contraction length that ends inside a block
        dict(kind="matmul", rows=107 * 77, n=2048, k=1000, abits=8, bbits=4, bias=True, name="product_mixed"),
        # c_proj of a 64-image forward of the patch-14 tower with both operands in 4 bits
        dict(kind="matmul", rows=64 * 257, n=1024, k=4096, abits=4, bbits=4, bias=True, name="product_large"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["seam_fwd", "seam_bwd", "act8", "wgrad8", "quant", "matmul"])
    if kind.startswith("seam"):
        gate = rng.choice(["none", "group", "channel", "row"])
        d = _log(rng, 32, 4096)
        d = d if rng.random() < 0.4 else max(32, d // 8 * 8)
        groups = rng.randint(1, 64)
        per = _log(rng, 1, min(257, 64 * 257 * 1024 // (d * groups)))
        return _seam(kind, groups * per, d, norm=rng.choice(["layer", "rms"]), post=rng.random() < 0.6, pre=rng.random() < 0.85,
                     gate=gate, groups=groups * per if gate == "row" else groups if gate != "none" else 1, scale=rng.random() < 0.7,
                     x=rng.choice(["fp32", "fp32", "bf16"]), h=rng.choice(["bf16", "bf16", "fp32"]), alpha=rng.choice([1.0, 0.5, 1.25]))
    if kind == "act8":
        return dict(kind=kind, rows=_log(rng, 1, 8224), n=_log(rng, 33, 4096), act=rng.choice(["gelu", "quick_gelu"]))
    if kind == "wgrad8":
        return dict(kind=kind, rows=_log(rng, 1, 16448), n=_log(rng, 32, 4096), k=_log(rng, 32, 1024))
    if kind == "quant":
        return dict(kind=kind, rows=_log(rng, 1, 4096), k=_log(rng, 1, 4096), bits=rng.choice([4, 8]), x=rng.choice(["fp32", "bf16"]))
    return dict(kind=kind, rows=_log(rng, 1, 16448), n=_log(rng, 32, 1024), k=_log(rng, 32, 4096), abits=rng.choice([4, 4, 8]),
                bbits=rng.choice([4, 4, 8]), bias=rng.random() < 0.5)


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)


def _spread(g, rows, n, dtype=torch.float32):
    """Activations as a tower has them: a few columns much larger than the others."""
    wide = torch.exp(torch.randn((1, n), generator=g, device="cuda") * 0.7)
    return (torch.randn((rows, n), generator=g, device="cuda") * wide).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, s = case, dict(case=case)
    kind = c["kind"]
    if kind.startswith("seam"):
        rows, d, bwd = c["rows"], c["d"], kind == "seam_bwd"
        s["x"] = _normal(g, rows, d, scale=1.3, mean=0.2, dtype=_DT[c["x"]])
        s["h"] = _spread(g, rows, d, _DT[c["h"]])
        bias = c["norm"] == "layer"
        for name in ("post", "pre"):
            w, b = _normal(g, d, scale=0.2, mean=1.0), _normal(g, d, scale=0.1)
            s[name] = (w, b if bias else None) if c[name] else None
        s["scale"] = _normal(g, d, scale=0.1, mean=0.3) if c["scale"] else None
        s["gate"] = None
        if c["gate"] == "group" or c["gate"] == "row":  # stochastic depth: dropped (0) or scaled up
            keep = (torch.rand((c["groups"],), generator=g, device="cuda") < 0.9).float() / 0.9
            s["gate"] = keep
        elif c["gate"] == "channel":
            s["gate"] = _normal(g, c["groups"], d, scale=0.5, mean=0.5)
        if bwd:
            s["dy"] = _normal(g, rows, d, dtype=_DT[c["x"]])
            s["dz"] = _normal(g, rows, d, dtype=torch.bfloat16) if c["pre"] else None
            # what the forward left: the stream, and the statistics of both norms
            y, _, stats = _seam_fwd(s, torch.float32)
            s["y"], s["stats"] = y.to(s["x"].dtype), stats
    elif kind == "act8":
        s["f"] = _spread(g, c["rows"], c["n"], torch.bfloat16)
        s["dg"] = _normal(g, c["rows"], c["n"], dtype=torch.bfloat16)
    elif kind == "wgrad8":
        s["dy"] = _normal(g, c["rows"], c["n"], dtype=torch.bfloat16)
        s["x8"] = _packed(_spread(g, c["rows"], c["k"]), 8)
    elif kind == "quant":
        s["x"] = _spread(g, c["rows"], c["k"], _DT[c["x"]])
    else:
        s["a"] = _packed(_spread(g, c["rows"], c["k"]), c["abits"])
        s["b"] = _packed(_normal(g, c["n"], c["k"], scale=c["k"] ** -0.5), c["bbits"])
        s["bias"] = _normal(g, c["n"], scale=0.1) if c["bias"] else None
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------------
def _blocks(x):
    """[rows, n] -> [rows, ceil(n / 32), 32], zeros behind the last column."""
    rows, n = x.shape
    pad = -n % 32
    return torch.nn.functional.pad(x, (0, pad)).view(rows, (n + pad) // 32, 32)


def _exponents(blocks, bits):
    """The exponent of the smallest power of two (2^-110 at least) that brings a block's largest magnitude under the format's."""
    m, e = torch.frexp(blocks.abs().amax(-1))
    top = 3 if bits == 4 else 9  # 6 = 0.75 2^3, 448 = 0.875 2^9
    e = e.to(torch.int32) - top + (m > (0.75 if bits == 4 else 0.875)).to(torch.int32)
    return torch.where(m == 0, -110, e.clamp(min=-110))


def _round_to(v, bits):
    """Round to nearest, ties to even, on the format's grid (v within its range)."""
    low, mant = (0, 1) if bits == 4 else (-6, 3)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e.to(torch.int32) - 1).clamp(min=low) - mant)
    return torch.round(v / step) * step


def _quantized(x, bits):
    """-> the blocks' values on the format's grid, and their exponents."""
    b = _blocks(x.float())
    e = _exponents(b, bits)
    return _round_to(torch.ldexp(b, -e[..., None]), bits), e


def _held(x, bits):
    """The values that x stands for once it is packed."""
    v, e = _quantized(x, bits)
    return torch.ldexp(v, e[..., None]).view(x.shape[0], -1)[:, :x.shape[1]]


def _packed(x, bits):
    """The packed form: (codes, scale bytes, columns, bits).  Codes: a byte each, or two to a byte, the even column low."""
    rows, n = x.shape
    v, e = _quantized(x, bits)
    v = v.reshape(rows, -1)
    if bits == 8:
        codes = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
        codes = torch.bucketize(v.abs(), grid).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
        codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return codes.contiguous(), (e + 127).to(torch.uint8).contiguous(), n, bits


def _values(packed):
    """The values that a packed matrix stands for, in 32 bits."""
    codes, scale, n, bits = packed
    if bits == 8:
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        grid = torch.cat([grid, -grid])
        v = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).view(codes.shape[0], -1)
    v = torch.ldexp(v.view(codes.shape[0], -1, 32), (scale.to(torch.int32) - 127)[..., None])
    return v.view(codes.shape[0], -1)[:, :n]


def _norm(t, wb, kind):
    mean = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[:, :1])
    rstd = 1.0 / torch.sqrt(((t - mean) ** 2).mean(-1, keepdim=True) + EPS)
    n = (t - mean) * rstd * wb[0]
    return (n + wb[1] if wb[1] is not None else n), mean, rstd


def _gate(s, dt):
    """The gate spread over rows: [rows, 1 or d]."""
    c = s["case"]
    if s["gate"] is None:
        return torch.ones((1, 1), dtype=dt, device="cuda")
    g = s["gate"].to(dt)
    g = g[:, None] if g.dim() == 1 else g
    return g.repeat_interleave(c["rows"] // c["groups"], 0)


def _seam_fwd(s, dt):
    c = s["case"]
    x, p = s["x"].to(dt), s["h"].to(dt)
    st = torch.zeros((4, c["rows"]), dtype=dt, device="cuda")
    if s["post"] is not None:
        p, m, r = _norm(p, s["post"], c["norm"])
        st[0], st[1] = m[:, 0], r[:, 0]
    mul = _gate(s, dt)
    if s["scale"] is not None:
        mul = mul * s["scale"].to(dt)
    y = c["alpha"] * x + mul * p
    z = None
    if s["pre"] is not None:
        # the norm reads the stream as it is kept
        z, m, r = _norm(y.to(s["x"].dtype).to(dt), s["pre"], c["norm"])
        st[2], st[3] = m[:, 0], r[:, 0]
    return y, z, st


def _norm_bwd(dn, t, w, mean, rstd, kind):
    """-> dt, dw, db of n = (t - mean) rstd w + b."""
    hat = (t - mean[:, None]) * rstd[:, None]
    u = dn * w
    dt = u - hat * (u * hat).mean(-1, keepdim=True)
    if kind == "layer":
        dt = dt - u.mean(-1, keepdim=True)
    return dt * rstd[:, None], (dn * hat).sum(0), dn.sum(0)


def _seam_bwd(s):
    c = s["case"]
    f = torch.float32
    layer = c["norm"] == "layer"
    st, out = s["stats"], {}
    gy = s["dy"].to(f)
    if s["pre"] is not None:
        dt, out["pre_w"], db = _norm_bwd(s["dz"].to(f), s["y"].to(f), s["pre"][0], st[2], st[3], c["norm"])
        gy = gy + dt
        if layer:
            out["pre_b"] = db
    h = s["h"].to(f)
    p = h
    if s["post"] is not None:
        p = (h - st[0][:, None]) * st[1][:, None] * s["post"][0]
        p = p + s["post"][1] if layer else p
    gate = _gate(s, f)
    mul = gate
    t = p * gy
    if s["scale"] is not None:
        mul = gate * s["scale"]
        out["scale"] = (gate * t).sum(0)
        t = t * s["scale"]
    if s["gate"] is not None:
        t = t.view(c["groups"], -1, c["d"]).sum(1)
        out["gate"] = t.sum(-1) if s["gate"].dim() == 1 else t
    dh = mul * gy
    if s["post"] is not None:
        dh, out["post_w"], db = _norm_bwd(dh, h, s["post"][0], st[0], st[1], c["norm"])
        if layer:
            out["post_b"] = db
    out["x"], out["h"] = (c["alpha"] * gy).to(s["x"].dtype), dh.to(s["h"].dtype)
    return out


def _erf_gelu(x):
    cdf = 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5)))
    return x * cdf, cdf + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))


def _quick_gelu(x):
    sg = 1.0 / (1.0 + torch.exp(-1.702 * x))
    return x * sg, sg * (1.0 + 1.702 * x * (1.0 - sg))


def _plain(s):
    c = s["case"]
    kind = c["kind"]
    bf = torch.bfloat16
    if kind == "seam_fwd":
        y, z, _ = _seam_fwd(s, torch.float32)
        return dict(y=y.to(s["x"].dtype), z=z.to(bf) if z is not None else None)
    if kind == "seam_bwd":
        return _seam_bwd(s)
    if kind == "act8":
        act = _erf_gelu if c["act"] == "gelu" else _quick_gelu
        g = act(s["f"].float())[0].to(bf)
        again, slope = act(_held(s["f"], 8))
        return dict(g=g, df=(s["dg"].float() * slope).to(bf), again=again.to(bf))
    if kind == "wgrad8":
        dy = s["dy"].float()
        return dict(dw=dy.t() @ _values(s["x8"]), db=dy.sum(0))
    if kind == "quant":
        return dict(held=_held(s["x"], c["bits"]))
    out = _values(s["a"]) @ _values(s["b"]).t()
    return dict(c=(out + s["bias"] if s["bias"] is not None else out).to(bf))


def run(state):
    if not own:
        return _plain(state)
    from swat_amd import mx, ops
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "seam_fwd":
        r = ops.residual_norm_fwd(s["x"], s["h"], post=s["post"], pre=s["pre"], gate=s["gate"], scale=s["scale"], alpha=c["alpha"],
                                  norm=c["norm"], eps=EPS)
        return dict(y=r.y, z=r.z)
    if kind == "seam_bwd":
        return ops.residual_norm_bwd(s["dy"], s["dz"], s["h"], s["y"], s["stats"], post=s["post"], pre=s["pre"], gate=s["gate"],
                                     scale=s["scale"], alpha=c["alpha"], norm=c["norm"])
    if kind == "act8":
        g, f8 = mx.act_fwd(s["f"], c["act"])
        df, again = mx.act_bwd(s["dg"], f8, c["act"])
        return dict(g=g, df=df, again=again)
    if kind == "wgrad8":
        dw, db = mx.linear_wgrad(s["dy"], mx.MX(*s["x8"]), want_bias=True)
        return dict(dw=dw, db=db)
    if kind == "quant":
        return dict(held=mx.dequantize(mx.quantize(s["x"], c["bits"]), torch.float32))
    return dict(c=mx.matmul(mx.MX(*s["a"]), mx.MX(*s["b"]), bias=s["bias"]))


# ---- the least that a pass moves and computes -------------------------------------------------------------------------------------
def work(case):
    c, kind = case, case["kind"]
    size = {"bf16": 2, "fp32": 4}
    if kind.startswith("seam"):
        rows, d, x, h = c["rows"], c["d"], size[c["x"]], size[c["h"]]
        pre, vectors = bool(c["pre"]), 4 * d * (2 * c["post"] + 2 * c["pre"] + c["scale"])
        gate = {"none": 0, "group": 4 * c["groups"], "row": 4 * c["groups"], "channel": 4 * c["groups"] * d}[c["gate"]]
        if kind == "seam_fwd":
            return dict(bytes=rows * d * (2 * x + h + 2 * pre) + vectors + gate, flops=rows * d * (3 + 8 * c["post"] + 8 * pre))
        return dict(bytes=rows * d * (2 * x + 2 * h + (2 + x) * pre) + 16 * rows + 2 * (vectors + gate),
                    flops=rows * d * (8 + 14 * c["post"] + 14 * pre))
    packed = lambda rows, n, bits: rows * ((n + 31) // 32) * (32 * bits // 8 + 1)  # noqa: E731
    if kind == "act8":  # f, dg in; g, df and the recomputed activation out; the checkpoint is written and read
        return dict(bytes=10 * c["rows"] * c["n"] + 2 * packed(c["rows"], c["n"], 8), flops=40 * c["rows"] * c["n"])
    if kind == "wgrad8":
        return dict(bytes=2 * c["rows"] * c["n"] + packed(c["rows"], c["k"], 8) + 4 * c["n"] * (c["k"] + 1),
                    flops=2 * c["rows"] * c["n"] * c["k"])
    if kind == "quant":  # read, packed, read packed, written as values
        return dict(bytes=c["rows"] * c["k"] * (size[c["x"]] + 4) + 2 * packed(c["rows"], c["k"], c["bits"]), flops=6 * c["rows"] * c["k"])
    return dict(bytes=packed(c["rows"], c["k"], c["abits"]) + packed(c["n"], c["k"], c["bbits"]) + 2 * c["rows"] * c["n"] + 4 * c["n"] * c["bias"],
                flops=2 * c["rows"] * c["n"] * c["k"])


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------
def _exact_held(x, bits):
    """Each block by its definition: search the scale by powers of two, the nearest grid value by distance (even code on a tie)."""
    x = x.double()
    rows, n = x.shape
    b = torch.zeros((rows, -(-n // 32) * 32), dtype=torch.float64, device=x.device)
    b[:, :n] = x
    b = b.view(rows, -1, 32)
    a = b.abs().max(-1).values
    e = torch.full(a.shape, -110.0, dtype=torch.float64, device=x.device)
    for k in range(-110, 128):
        e = torch.where(a > _MAX[bits] * 2.0 ** k, float(k + 1), e)
    s = torch.exp2(e)[..., None]
    if bits == 4:
        grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        grid = [(m / 8.0) * 2.0 ** -6 for m in range(8)] + [(1 + m / 8.0) * 2.0 ** k for k in range(-6, 9) for m in range(8)][:-1]
    grid = torch.tensor(grid, dtype=torch.float64, device=x.device)
    v = b.abs() / s
    hi = torch.searchsorted(grid, v).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - v, v - grid[lo]
    at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (torch.sign(b) * grid[at] * s).view(rows, -1)[:, :n]


def _exact_norm(t, wb, kind):
    d = t.shape[-1]
    mean = t.sum(-1) / d if kind == "layer" else t.new_zeros(t.shape[0])
    hat = (t - mean[:, None]) / torch.sqrt(((t - mean[:, None]) ** 2).sum(-1) / d + EPS)[:, None]
    out = hat * wb[0].double()
    return out if wb[1] is None else out + wb[1].double()


def exact(case, seed):
    s, c = prepare(case, seed), case
    kind = c["kind"]
    D = torch.float64
    if kind == "seam_fwd":
        rows, d = c["rows"], c["d"]
        p = s["h"].to(D) if s["post"] is None else _exact_norm(s["h"].to(D), s["post"], c["norm"])
        if s["scale"] is not None:
            p = p * s["scale"].to(D)
        if s["gate"] is not None:
            p = (p.view(c["groups"], -1, d) * s["gate"].to(D).view(c["groups"], 1, -1)).view(rows, d)
        y = s["x"].to(D) * c["alpha"] + p
        z = None if s["pre"] is None else _exact_norm(y.to(s["x"].dtype).to(D), s["pre"], c["norm"])
        return dict(y=y, z=z)
    if kind == "seam_bwd":
        # differentiated by torch in 64 bits: two functions that meet in the stream as it was kept
        leaf = lambda t: None if t is None else t.to(D).requires_grad_()  # noqa: E731
        post = None if s["post"] is None else tuple(leaf(t) for t in s["post"])
        pre = None if s["pre"] is None else tuple(leaf(t) for t in s["pre"])
        x, h, scale, gate = (leaf(s[k]) for k in ("x", "h", "scale", "gate"))
        with torch.enable_grad():
            gy = s["dy"].to(D)
            named = {}
            if pre is not None:
                y = leaf(s["y"])
                _exact_norm(y, pre, c["norm"]).backward(s["dz"].to(D))
                gy = gy + y.grad
                named.update(pre_w=pre[0].grad, pre_b=None if pre[1] is None else pre[1].grad)
            p = h if post is None else _exact_norm(h, post, c["norm"])
            p = p if scale is None else p * scale
            p = p if gate is None else (p.view(c["groups"], -1, c["d"]) * gate.view(c["groups"], 1, -1)).view(p.shape)
            (c["alpha"] * x + p).backward(gy)
        named.update(x=x.grad, h=h.grad, scale=None if scale is None else scale.grad, gate=None if gate is None else gate.grad)
        if post is not None:
            named.update(post_w=post[0].grad, post_b=None if post[1] is None else post[1].grad)
        return {k: v for k, v in named.items() if v is not None}
    if kind == "act8":
        def act(t):
            if c["act"] == "gelu":
                return 0.5 * t * torch.special.erfc(-t / math.sqrt(2.0))
            return t * torch.sigmoid(1.702 * t)

        f = _exact_held(s["f"], 8).requires_grad_()
        with torch.enable_grad():
            again = act(f)
            again.backward(s["dg"].to(D))
        return dict(g=act(s["f"].to(D)), df=f.grad, again=again.detach())
    if kind == "wgrad8":
        dy = s["dy"].to(D)
        return dict(dw=dy.t() @ _exact_values(s["x8"]), db=dy.sum(0))
    if kind == "quant":
        return dict(held=_exact_held(s["x"], c["bits"]))
    out = _exact_values(s["a"]) @ _exact_values(s["b"]).t()
    return dict(c=out if s["bias"] is None else out + s["bias"].to(D))


def _exact_values(packed):
    """Decoded field by field: sign, exponent, mantissa."""
    codes, scale, n, bits = packed
    q = codes.to(torch.int64)
    if bits == 4:
        q = torch.stack([q % 16, q // 16], -1).reshape(q.shape[0], -1)
    mant, width, bias = (2, 2, 1) if bits == 4 else (8, 4, 7)
    sign = torch.where(q // (mant << width) == 1, -1.0, 1.0).double()
    ex, fr = (q // mant) % (1 << width), (q % mant).double() / mant
    v = sign * torch.where(ex == 0, fr * 2.0 ** (1 - bias), (1.0 + fr) * torch.exp2((ex - bias).double()))
    return (v.view(q.shape[0], -1, 32) * torch.exp2(scale.double() - 127.0)[..., None]).view(q.shape[0], -1)[:, :n]
