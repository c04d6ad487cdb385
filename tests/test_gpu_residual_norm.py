"""GPU: the seam between two sublayers (ops.residual_norm_fwd / _bwd) against its formulas in 64 bits.

Tolerances.  A row's sums run over at most 16 values in a lane, 6 lane exchanges and 8 waves: 30 additions, each off by half a
step (2^-24) of the running sum, which the sum of magnitudes bounds; the mean, the deviation, the root, the division and the few
products behind them add under 30 more.  Outputs: 64 x 2^-24 of the magnitudes that enter plus half a step of the output's type;
gradients through two norms twice that.  Column sums: the rows of a team (up to 7 here), 8 teams, 16 workgroups to a thread and 16 of those: at most 47
additions over terms off by 64 x 2^-24 themselves: 256 x 2^-24 of the sum of magnitudes."""
import pytest
import torch

from helpers import mx_formulas as F

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-5
ULP = 2.0 ** -24


def rnd(*shape, seed, scale=1.0, mean=0.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype).cuda()


def near(got, ref, mag, steps, what):
    got, half = got.double(), F.HALF[got.dtype] if got.dtype != F32 else 0.0
    tol = steps * ULP * mag + half * ref.abs() + 1e-30
    over = (got - ref).abs() / tol
    assert torch.isfinite(got).all() and over.max().item() <= 1.0, f"{what}: {over.max().item():.3g} of the tolerance"


def make(rows, d, norm, post, pre, gate, groups, scale, xt, ht, seed=0, bias=True):
    t = dict(x=rnd(rows, d, seed=seed + 1, mean=0.3, dtype=xt), h=rnd(rows, d, seed=seed + 2, scale=2.0, dtype=ht), norm=norm)
    for k, name in enumerate(("post", "pre")):
        on = (post, pre)[k]
        t[name] = (rnd(d, seed=seed + 3 + k, scale=0.2, mean=1.0), rnd(d, seed=seed + 5 + k, scale=0.1) if bias and norm == "layer" else None) if on else None
    t["scale"] = rnd(d, seed=seed + 7, scale=0.3) if scale else None
    t["gate"] = None
    if gate == "group":
        t["gate"] = rnd(groups, seed=seed + 8)
        t["gate"][0] = 0.0
    elif gate == "channel":
        t["gate"] = rnd(groups, d, seed=seed + 8)
        t["gate"][-1, 0] = 0.0
    return t


CASES = [  # rows, d, norm, post, pre, gate, groups, scale, x, h
    (1, 1, "rms", True, True, "none", 1, True, F32, F32),
    (1, 4, "layer", True, True, "group", 1, True, F32, BF),
    (3, 31, "layer", False, True, "none", 1, True, BF, BF),
    (50, 768, "layer", False, True, "none", 1, True, F32, BF),
    (257, 1024, "layer", True, True, "group", 257, True, F32, BF),
    (7 * 33, 509, "rms", True, True, "channel", 7, True, BF, BF),
    (64, 260, "layer", True, False, "group", 16, False, F32, F32),
    (5 * 11, 1028, "rms", True, True, "channel", 5, False, F32, BF),
    (36, 1030, "layer", True, True, "channel", 36, True, BF, F32),
    (30, 4096, "layer", True, True, "group", 3, True, F32, BF),
    (10, 4100, "layer", True, True, "channel", 2, True, F32, BF),
    (9, 8191, "rms", True, True, "group", 3, True, BF, BF),
    (4, 8192, "layer", True, True, "group", 2, True, F32, F32),
    (2100, 256, "layer", False, False, "group", 10, True, F32, BF),
    (12608, 96, "layer", True, True, "group", 64, True, F32, BF),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(str(v).replace("torch.", "") for v in c))
@pytest.mark.parametrize("strided", [False, True])
def test_forward_and_backward(case, strided):
    from swat_amd import mx, ops
    t = make(*case)
    rows, d = t["x"].shape
    if strided:  # rows inside a wider buffer, at an offset that leaves no 16-byte alignment
        for k in ("x", "h"):
            wide = torch.full((rows, d + 5), float("nan"), dtype=t[k].dtype, device="cuda")
            wide[:, 3:3 + d] = t[k]
            t[k] = wide[:, 3:3 + d]
    alpha, norm = 0.75, t["norm"]
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"], alpha=alpha, norm=norm)
    r = ops.residual_norm_fwd(t["x"], t["h"], eps=EPS, pack=t["pre"] is not None, **kw)
    y, mag = F.seam_fwd(t["x"], t["h"], t["post"], t["pre"], t["gate"], t["scale"], alpha, norm, EPS)
    assert r.y.dtype == t["x"].dtype
    near(r.y, y, mag, 64, "y")
    if t["pre"] is None:
        assert r.z is None and r.z8 is None
    else:
        z, zmag = F.seam_norm(r.y, t["pre"], norm, EPS)
        near(r.z, z, zmag, 64, "z")
        again = mx.quantize(r.z, 8)  # the packed z is the z beside it, packed
        assert torch.equal(again.codes, r.z8.codes) and torch.equal(again.scale, r.z8.scale)
        rf = ops.residual_norm_fwd(t["x"], t["h"], eps=EPS, z_dtype=F32, **kw)
        near(rf.z, z, zmag, 64, "z in fp32")
        assert torch.equal(rf.y, r.y) and rf.z8 is None

    dy, dz = rnd(rows, d, seed=20, dtype=t["x"].dtype), rnd(rows, d, seed=21, dtype=BF) if t["pre"] is not None else None
    for with_dy in (True, False) if dz is not None else (True,):
        got = ops.residual_norm_bwd(dy if with_dy else None, dz, t["h"], r.y, r.stats, **kw)
        want = F.seam_bwd(dy if with_dy else None, dz, t["h"], r.y, t["post"], t["pre"], t["gate"], t["scale"], alpha, norm, EPS)
        assert set(got) == set(want)
        for k, (ref, m) in want.items():
            assert got[k].shape == ref.shape
            near(got[k], ref, m, 128 if k in ("x", "h") else 256, k)
        twice = ops.residual_norm_bwd(dy if with_dy else None, dz, t["h"], r.y, r.stats, **kw)
        assert all(torch.equal(got[k], twice[k]) for k in got), "the order of the sums is fixed"


def test_gradients_against_differences():
    """d loss / d (scale, gate, post bias) along a direction, by central differences in 64 bits of the formula."""
    from swat_amd import ops
    t = make(24, 64, "layer", True, True, "channel", 3, True, F32, F32, seed=40)
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"], alpha=1.0, norm="layer")
    r = ops.residual_norm_fwd(t["x"], t["h"], eps=EPS, z_dtype=F32, **kw)
    dy, dz = rnd(24, 64, seed=50), rnd(24, 64, seed=51)
    got = ops.residual_norm_bwd(dy, dz, t["h"], r.y, r.stats, **kw)

    def loss(v):
        y, _ = F.seam_fwd(v["x"], v["h"], v["post"], v["pre"], v["gate"], v["scale"], 1.0, "layer", EPS)
        z, _ = F.seam_norm(y, v["pre"], "layer", EPS)
        return (y * dy.double()).sum() + (z * dz.double()).sum()

    base = {k: tuple(a.double() for a in v) if isinstance(v, tuple) else v.double() if isinstance(v, torch.Tensor) else v for k, v in t.items()}
    for name, key, at in (("x", "x", None), ("h", "h", None), ("scale", "scale", None), ("gate", "gate", None), ("post_w", "post", 0),
                          ("post_b", "post", 1), ("pre_w", "pre", 0), ("pre_b", "pre", 1)):
        val = base[key] if at is None else base[key][at]
        u = torch.randn(val.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64).cuda()
        step = 1e-5
        ends = []
        for sign in (1, -1):
            v = dict(base)
            new = val + sign * step * u
            v[key] = new if at is None else tuple(new if i == at else base[key][i] for i in range(2))
            ends.append(loss(v))
        diff = ((ends[0] - ends[1]) / (2 * step)).item()
        dot = (got[name].double() * u).sum().item()
        size = (got[name].double() * u).norm().item()
        # differences: step^2 of the third derivative and rounding / step, both under 1e-7 of the terms; the kernel: 2^-24 x 256
        assert abs(diff - dot) <= 3e-5 * size + 1e-6, (name, diff, dot)


def test_a_dropped_branch_may_hold_anything():
    from swat_amd import ops
    t = make(12, 96, "layer", True, True, "group", 6, True, F32, BF, seed=60)
    t["gate"] = torch.tensor([0.0, 1.0, 0.0, 1.25, 1.0, 0.0], device="cuda")
    clean = t["h"].clone()
    for rows, v in ((0, float("nan")), (4, float("inf")), (5, 3e38), (11, float("-inf"))):
        t["h"][rows] = v
        clean[rows] = 0
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"], norm="layer")
    a, b = (ops.residual_norm_fwd(t["x"], h, **kw) for h in (t["h"], clean))
    assert torch.equal(a.y, b.y) and torch.equal(a.z, b.z)
    dropped = torch.tensor([0, 1, 4, 5, 10, 11], device="cuda")
    assert torch.equal(a.y[dropped], t["x"][dropped])
    dy, dz = rnd(12, 96, seed=61), rnd(12, 96, seed=62, dtype=BF)
    g, w = ops.residual_norm_bwd(dy, dz, t["h"], a.y, a.stats, **kw), ops.residual_norm_bwd(dy, dz, clean, b.y, b.stats, **kw)
    for k in g:
        if k != "gate":  # (the gate's own gradient is what its branch holds)
            assert torch.equal(g[k], w[k]), k
    assert not g["h"][dropped].any()
    live = torch.tensor([1, 3, 4], device="cuda")
    assert torch.equal(g["gate"][live], w["gate"][live])


@pytest.mark.parametrize("gate", ["group", "channel"])
def test_channels_scaled_by_zero_may_hold_anything(gate):
    """Without a norm after the sublayer: those channels enter neither the stream nor any gradient."""
    from swat_amd import ops
    t = make(12, 96, "layer", False, True, gate, 6, True, F32, BF, seed=65)
    t["scale"][[0, 40, 95]] = 0.0
    clean = t["h"].clone()
    for c, v in ((0, float("nan")), (40, float("inf")), (95, float("-inf"))):
        t["h"][:, c] = v
        clean[:, c] = 0
    kw = dict(pre=t["pre"], gate=t["gate"], scale=t["scale"])
    a, b = (ops.residual_norm_fwd(t["x"], h, **kw) for h in (t["h"], clean))
    assert torch.equal(a.y, b.y) and torch.equal(a.z, b.z)
    dy, dz = rnd(12, 96, seed=66), rnd(12, 96, seed=67, dtype=BF)
    g, w = ops.residual_norm_bwd(dy, dz, t["h"], a.y, a.stats, **kw), ops.residual_norm_bwd(dy, dz, clean, b.y, b.stats, **kw)
    for k in g:
        if k != "scale":  # (the scale's own gradient is what its channel holds)
            assert torch.equal(g[k], w[k]), k
    live = t["scale"] != 0
    assert torch.equal(g["scale"][live], w["scale"][live])


def test_no_rows():
    from swat_amd import ops
    t = make(0, 40, "layer", True, True, "none", 1, True, F32, BF)
    t["gate"] = rnd(3, 40, seed=1)
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"])
    r = ops.residual_norm_fwd(t["x"], t["h"], pack=True, **kw)
    assert r.y.shape == r.z.shape == (0, 40) and r.z8.shape == (0, 40)
    g = ops.residual_norm_bwd(r.y, r.z, t["h"], r.y, r.stats, **kw)
    for k in ("post_w", "post_b", "scale", "pre_w", "pre_b", "gate"):
        assert not g[k].any(), k


def test_rows_past_two_to_the_31_elements():
    """Offsets are 64 bits wide: the last rows of a bf16 stream of 2^31 + elements."""
    from swat_amd import ops
    d, rows = 8192, 2 ** 18 + 3
    x = torch.zeros((rows, d), dtype=BF, device="cuda")
    x[-3:] = rnd(3, d, seed=9, dtype=BF)
    w = (rnd(d, seed=10, mean=1.0), None)
    r = ops.residual_norm_fwd(x, x, pre=w, norm="rms")
    want, mag = F.seam_fwd(x[-3:], x[-3:], None, w, None, None, 1.0, "rms", EPS)
    near(r.y[-3:], want, mag, 64, "y")
    z, zm = F.seam_norm(r.y[-3:], w, "rms", EPS)
    near(r.z[-3:], z, zm, 64, "z")
    assert not r.y[:8].any() and not r.z[rows // 2].any()


@pytest.mark.parametrize("rows,d", [(2 ** 26 + 37, 2), (2 ** 24 + 5, 1028)])
def test_rows_past_one_dimension_of_a_launch(rows, d):
    """A wave (four, past 1024 columns) to a row: more than 2^32 threads."""
    from swat_amd import ops
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 170 << 30:
        pytest.skip("needs 170 GB")
    x = torch.zeros((rows, d), dtype=BF, device="cuda")
    x[:3] = rnd(3, d, seed=8, dtype=BF)
    x[-9:] = rnd(9, d, seed=9, dtype=BF)
    w = (rnd(d, seed=10, mean=1.0), None)
    r = ops.residual_norm_fwd(x, x, pre=w)
    for a, b in ((0, 3), (rows - 9, rows)):
        want = ops.residual_norm_fwd(x[a:b], x[a:b], pre=w)
        assert torch.equal(r.y[a:b], want.y) and torch.equal(r.z[a:b], want.z) and torch.equal(r.stats[2:, a:b], want.stats[2:]) and want.y.any()
    assert not r.y[3:-9:40961].any() and not r.z[3:-9:40961].any()


def test_a_captured_pass_replays():
    from swat_amd import ops
    t = make(31 * 7, 512, "layer", True, True, "group", 31, True, F32, BF, seed=70)
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"])
    dy, dz = rnd(217, 512, seed=71), rnd(217, 512, seed=72, dtype=BF)

    def both():
        r = ops.residual_norm_fwd(t["x"], t["h"], pack=True, **kw)
        return r, ops.residual_norm_bwd(dy, dz, t["h"], r.y, r.stats, **kw)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, g = both()
    for k in range(4):
        t["x"].copy_(rnd(217, 512, seed=80 + k))
        t["h"].copy_(rnd(217, 512, seed=90 + k, dtype=BF))
        graph.replay()
        er, eg = both()  # the program's own work between the replays
        torch.cuda.synchronize()
        assert torch.equal(r.y, er.y) and torch.equal(r.z, er.z) and torch.equal(r.z8.codes, er.z8.codes) and torch.equal(r.z8.scale, er.z8.scale)
        assert all(torch.equal(g[n], eg[n]) for n in g)


def test_on_another_stream():
    from swat_amd import ops
    t = make(300, 768, "layer", True, True, "group", 10, True, F32, BF, seed=100)
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"])
    want = ops.residual_norm_fwd(t["x"], t["h"], **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.residual_norm_fwd(t["x"], t["h"], **kw)
    s.synchronize()
    assert torch.equal(got.y, want.y) and torch.equal(got.z, want.z)


def test_refusals():
    from swat_amd import _lib, ops
    x, h, w = rnd(8, 16, seed=1), rnd(8, 16, seed=2), rnd(16, seed=3)
    for kw in (dict(gate=rnd(3, seed=1)), dict(gate=rnd(2, 15, seed=1)), dict(scale=rnd(15, seed=1)), dict(post=(w.bfloat16(), None)),
               dict(pre=(w, w[:8])), dict(norm="batch"), dict(pack=True), dict(z_dtype=torch.float16), dict(post=(None, w))):
        with pytest.raises(_lib.SwatHipError):
            ops.residual_norm_fwd(x, h, **kw)
    for bad in (h[:, :8], h[:4], h.half(), h.t(), h[:1].expand(8, 16), rnd(8, 32, seed=4)[:, ::2]):
        with pytest.raises(_lib.SwatHipError):
            ops.residual_norm_fwd(x, bad)
    r = ops.residual_norm_fwd(x, h, pre=(w, None))
    for args in ((None, None, h, r.y, r.stats, {}), (x, None, h, r.y, r.stats, dict(pre=(w, None))), (x, x, h, r.y, r.stats, {}),
                 (x, x, h, None, r.stats, dict(pre=(w, None))), (x.bfloat16(), x, h, r.y, r.stats, dict(pre=(w, None))),
                 (x, x, h, r.y, r.stats[:2], dict(pre=(w, None))), (x[:4], x, h, r.y, r.stats, dict(pre=(w, None)))):
        with pytest.raises(_lib.SwatHipError):
            ops.residual_norm_bwd(*args[:5], **args[5])
