"""GPU: microscaled matrices (swat_amd/mx.py) against their definition in 64 bits.

Tolerances.  Packing and unpacking: none (equal).  Activations in bf16: half a step of the type (2^-8) plus 2^-18 |x| for the
exponential, the reciprocal and erf, each good to a few steps of fp32.  Products: operands are exact, products of two bf16 (e4m3, e2m1)
numbers are exact in fp32, so only the additions count: at most one half step (2^-24) of the running sum for each of n terms, which
n 2^-24 of the sum of magnitudes bounds; and because the errors of many additions do not all point one way, the error's norm is
held to 2e-6 of the result's as well (fp32 outputs).

Products with an 8-bit operand come out in bf16 only: the matrix instruction adds eight neighbouring columns' products after dropping what
lies more than 13 binary places below the largest of them, so each product may lose 2^-13 of its eight's largest, which the product of
the operands' largest magnitudes in those eight columns bounds (e2m1 by e2m1: products are multiples of 1/4 up to 36, nothing is lost)."""
import pytest
import torch

from helpers import mx_formulas as F

pytestmark = pytest.mark.gpu
BF, F32, D = torch.bfloat16, torch.float32, torch.float64
ULP = 2.0 ** -24


def rnd(*shape, seed, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def spread(rows, n, seed, dtype=F32):
    """Values over many binary orders, every block another scale."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, n, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, n), generator=g).float())
    return (x * torch.exp2(torch.randint(-20, 20, (rows, -(-n // 32)), generator=g).float()).repeat_interleave(32, 1)[:, :n]).to(dtype).cuda()


def same(got, want):
    got, want = got.double(), want.double()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~torch.isnan(got)], want[~torch.isnan(want)])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 100), (77, 512), (64, 1000), (257, 1024), (9, 4100)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_pack_and_unpack(bits, rows, n, dtype):
    from swat_amd import mx
    for x in (spread(rows, n, 1, dtype), spread(rows, n + 3, 2, dtype)[:, 1:n + 1]):
        want, byte = F.held(x, bits)
        m = mx.quantize(x, bits)
        assert m.shape == (rows, n) and torch.equal(m.scale, byte)
        for out in (BF, F32):
            assert same(mx.dequantize(m, out), want)
        # the columns behind the last one are zeros
        pad = mx.dequantize(mx.MX(m.codes, m.scale, m.scale.shape[1] * 32, bits), F32)[:, n:]
        assert not pad.any()


@pytest.mark.parametrize("bits", [4, 8])
def test_every_rounding_case(bits):
    """The grid, the midpoints (ties to even) and their neighbours on both sides, at the largest, smallest and ordinary scales."""
    from swat_amd import mx
    g = F.grid(bits)
    mid = (g[1:] + g[:-1]) / 2
    v = torch.cat([g, mid, torch.nextafter(mid.float(), torch.tensor(0.0)).double(), torch.nextafter(mid.float(), torch.tensor(1e9)).double()])
    for e in (-110, -60, 0, 30, 119 if bits == 8 else 125):
        rows = torch.zeros((v.numel() * 2, 32), dtype=D)
        rows[:, 0] = torch.cat([v, -v])
        rows[:, 17] = F.MAX[bits]
        x = (rows * 2.0 ** e).float().cuda()
        want, byte = F.held(x, bits)
        m = mx.quantize(x, bits)
        assert torch.equal(m.scale, byte) and same(mx.dequantize(m, F32), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_extremes(bits):
    from swat_amd import mx
    x = torch.zeros((8, 96), device="cuda")
    x[1, 5], x[2, 40], x[3, 95] = float("nan"), float("inf"), float("-inf")
    x[4], x[5] = torch.finfo(F32).max, 1e-45
    x[6, ::3] = 2.0 ** -118
    x[7] = torch.exp2(-torch.arange(96).float()).cuda()
    want, byte = F.held(x, bits)
    m = mx.quantize(x, bits)
    # the largest float32 rounds up to 4 x 2^126 (256 x 2^120) = 2^128, which float32 itself does not have: infinity, as its own rounding
    # to bfloat16 gives
    assert torch.equal(m.scale, byte) and (want[4] == 2.0 ** 128).all() and same(mx.dequantize(m, F32), want.float())
    assert torch.isnan(mx.dequantize(m)[1, :32]).all() and not mx.dequantize(m)[1, 32:].any()


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 40), (77, 2048), (33, 1003), (130, 4096)])
@pytest.mark.parametrize("act", ["gelu", "quick_gelu"])
def test_activation_with_checkpoint(rows, n, act):
    from swat_amd import mx
    for k, f in enumerate((rnd(rows, n, seed=3, scale=3.0, dtype=BF), rnd(rows, n + 9, seed=4, scale=3.0, dtype=BF)[:, 4:4 + n])):
        dg = rnd(rows, n + k, seed=5, dtype=BF)[:, :n]
        g, m = mx.act_fwd(f, act)
        plain = mx.quantize(f, 8)
        assert torch.equal(m.codes, plain.codes) and torch.equal(m.scale, plain.scale)
        ref, _ = F.act(f.double(), act)
        assert ((g.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * f.double().abs()).all()
        df, again = mx.act_bwd(dg, m, act)
        held, _ = F.held(f, 8)
        ref, slope = F.act(held, act)
        assert ((again.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * held.abs()).all()
        want = dg.double() * slope
        assert ((df.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * (1 + held.abs()) * dg.double().abs()).all()
        df2, none = mx.act_bwd(dg, m, act, want_act=False)
        assert none is None and torch.equal(df, df2)


def test_activation_slope_against_differences():
    from swat_amd import mx
    f = torch.linspace(-6, 6, 32 * 64).view(64, 32).bfloat16().cuda()
    one = torch.ones_like(f)
    for act in ("gelu", "quick_gelu"):
        _, m = mx.act_fwd(f, act)
        held, _ = F.held(f, 8)
        df, _ = mx.act_bwd(one, m, act)
        step = 1e-6
        diff = (F.act(held + step, act)[0] - F.act(held - step, act)[0]) / (2 * step)
        assert ((df.double() - diff).abs() <= 2.0 ** -8 * diff.abs() + 1e-4).all()  # 2^-18 x 7, and 1e-6 of the differences


@pytest.mark.parametrize("act", ["gelu", "quick_gelu"])
def test_activation_of_the_largest_numbers(act):
    """Far out the activation is x or 0 and its slope 1 or 0, also where x times a constant passes the type's end."""
    from swat_amd import mx
    big = torch.finfo(BF).max
    f = torch.tensor([[big, 2.5e38, 1e38, 1e19, 1e4] + [0.0] * 27, [-big, -2.5e38, -1e38, -1e19, -1e4] + [0.0] * 27], device="cuda").to(BF)
    g, m = mx.act_fwd(f, act)
    assert torch.equal(g[0], f[0]) and not g[1].any()
    for v in (big, 1e19, 1e4):   # (a block to each: small numbers next to the largest are zeros in it)
        f = torch.tensor([[v] * 3, [-v] * 3], device="cuda").to(BF)
        _, m = mx.act_fwd(f, act)
        held = mx.dequantize(m)
        df, again = mx.act_bwd(torch.ones_like(f), m, act)
        assert torch.equal(again[0], held[0]) and not again[1].any()
        assert (df[0] == 1).all() and not df[1].any()


def small(got, want, mag, terms, what):
    got = got.double()
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() / (terms * ULP * mag + 1e-30)).max().item()
    assert over <= 1.0, f"{what}: {over:.3g} of the tolerance"
    if want.norm() > 0:
        rel = ((got - want).norm() / mag.norm()).item()
        assert rel <= 2e-6, f"{what}: {rel:.3g}"


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 40, 33), (63, 128, 128), (64, 768, 768), (65, 130, 100), (200, 33, 1000), (1600, 768, 768),
                                      (1601, 257, 96), (5000, 64, 64), (8224, 512, 1024), (16448, 129, 40), (777, 2048, 513)])
def test_weight_gradient(rows, n, k):
    from swat_amd import mx
    x = spread(rows, k, 6) if rows < 100 else rnd(rows, k, seed=6)
    m = mx.quantize(x, 8)
    held = mx.dequantize(m, F32).double()
    for dy in (rnd(rows, n, seed=7, dtype=BF), rnd(rows, n + 5, seed=8, dtype=BF)[:, 2:n + 2]):
        dw, db = mx.linear_wgrad(dy, m, want_bias=True)
        d = dy.double()
        # (fp32 matmuls would do for the magnitudes; rows + 64: the partial sums of a split are joined by further additions)
        small(dw, d.t() @ held, d.abs().t() @ held.abs(), rows + 64, "dW")
        small(db, d.sum(0), d.abs().sum(0), rows + 64, "db")
        out = torch.full((n, k), float("nan"), device="cuda")
        assert mx.linear_wgrad(dy, m, out=out) is out and torch.equal(out, dw)


@pytest.mark.parametrize("rows,n,k", [(640, 65, 64), (833, 129, 100), (961, 64, 33), (1025, 255, 257), (1600, 769, 500), (2000, 63, 1000), (3201, 1000, 130)])
def test_weight_gradient_of_few_tiles(rows, n, k):
    """Two groups of waves share the rows: odd widths, an odd number of row tiles, a last tile of one row."""
    test_weight_gradient(rows, n, k)


@pytest.mark.parametrize("rows,n,k", [(5000, 1, 1), (20000, 3, 1), (6980, 32, 35), (12745, 161, 61), (4052, 187, 701), (1738, 1917, 34), (9000, 5, 129)])
def test_weight_gradient_of_many_parts(rows, n, k):
    """Planes of any size and alignment are joined: fewer than four elements, a last four that overlaps the one before."""
    test_weight_gradient(rows, n, k)


def test_weight_gradient_leaves_what_is_not_its_own():
    """Rows of dY and columns behind a view are not read into the sums, outputs behind dW are left as they were."""
    from swat_amd import mx
    wide = torch.full((100, 48), float("nan"), dtype=BF, device="cuda")
    wide[:, 8:40] = rnd(100, 32, seed=1, dtype=BF)
    m = mx.quantize(rnd(100, 70, seed=2), 8)
    room = torch.full((33 * 70,), 7.0, device="cuda")
    out = room[:32 * 70].view(32, 70)
    mx.linear_wgrad(wide[:, 8:40], m, out=out)
    assert (room[32 * 70:] == 7.0).all()
    small(out, wide[:, 8:40].double().t() @ mx.dequantize(m, F32).double(),
          wide[:, 8:40].double().abs().t() @ mx.dequantize(m, F32).double().abs(), 164, "dW")


def test_weight_gradient_of_no_rows_and_of_nan():
    from swat_amd import mx
    dw, db = mx.linear_wgrad(rnd(0, 24, seed=1, dtype=BF), mx.quantize(rnd(0, 50, seed=2), 8), want_bias=True)
    assert dw.shape == (24, 50) and not dw.any() and not db.any()
    x = rnd(70, 96, seed=3)
    x[11, 40] = float("inf")
    dw = mx.linear_wgrad(rnd(70, 24, seed=4, dtype=BF), mx.quantize(x, 8))
    assert torch.isnan(dw[:, 32:64]).all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(dw[:, 64:]).all()


@pytest.mark.parametrize("abits,bbits", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 4096, 1024), (2, 17, 33), (7, 300, 1000), (16, 64, 96), (17, 130, 160), (33, 1028, 2080), (64, 512, 512), (65, 512, 128),
                                   (100, 72, 200), (129, 127, 64), (257, 770, 513), (1600, 768, 768), (513, 2048, 1000), (300, 1024, 4096), (4200, 260, 96)])
def test_product(abits, bbits, M, N, K):
    from swat_amd import mx
    a, b = mx.quantize(spread(M, K, 10), abits), mx.quantize(rnd(N, K, seed=11, scale=K ** -0.5), bbits)
    A, B = mx.dequantize(a, F32).double(), mx.dequantize(b, F32).double()
    bias = rnd(N, seed=12)
    want, mag = A @ B.t(), A.abs() @ B.abs().t()
    if abits == bbits == 4:
        small(mx.matmul(a, b, out_dtype=F32), want, mag, K + 8, "C")
        small(mx.matmul(a, b, bias=bias, out_dtype=F32), want + bias.double(), mag + bias.double().abs(), K + 8, "C + bias")
    drop = eights(A) @ eights(B).t() * 8 * 2.0 ** -13 if abits + bbits > 8 else 0.0
    for with_bias in (bias, None):
        ref = want if with_bias is None else want + bias.double()
        got = mx.matmul(a, b, bias=with_bias).double()
        tol = 2.0 ** -8 * ref.abs() + (K + 8) * ULP * (mag + bias.double().abs()) + drop
        assert ((got - ref).abs() <= tol).all(), ((got - ref).abs() / tol).max().item()
        # and the norm, which the output's rounding alone sets: 2^-8 at most, and half of that in the mean
        assert (got - ref).norm() <= 2.0 ** -8 * ref.norm()


@pytest.mark.parametrize("abits,bbits", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("M,N,K", [(5000, 4100, 130), (4136, 8192, 300), (5130, 3000, 480), (8224, 1024, 520), (3000, 3001, 700)])
def test_product_of_every_tile_size(abits, bbits, M, N, K):
    """Sizes that the kernel cuts into 64, 128 and 256 wide tiles, some with their last rows in a launch of their own."""
    test_product(abits, bbits, M, N, K)


def eights(x):
    """The largest magnitude of every eight neighbouring columns."""
    return torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % 8)).view(x.shape[0], -1, 8).amax(-1)


def test_product_carries_nan_and_nothing_else():
    from swat_amd import mx
    for bits in (4, 8):
        for M in (3, 40, 200):
            x, w = rnd(M, 300, seed=1), rnd(90, 300, seed=2)
            x[2, 299], w[70, 3] = float("nan"), float("inf")
            c = mx.matmul(mx.quantize(x, bits), mx.quantize(w, bits))
            bad = torch.zeros((M, 90), dtype=torch.bool, device="cuda")
            bad[2], bad[:, 70] = True, True
            assert torch.equal(torch.isnan(c), bad) and torch.isfinite(c[~bad]).all()


def test_product_of_large_and_small_scales():
    """2^120 x 2^-100: the scales meet inside the product without passing infinity or zero."""
    from swat_amd import mx
    x, w = rnd(40, 128, seed=1) * 2.0 ** 120, rnd(48, 128, seed=2) * 2.0 ** -100
    a, b = mx.quantize(x, 4), mx.quantize(w, 4)
    A, B = mx.dequantize(a, F32).double(), mx.dequantize(b, F32).double()
    small(mx.matmul(a, b, out_dtype=F32), A @ B.t(), A.abs() @ B.abs().t(), 136, "C")


def test_no_rows_or_columns():
    from swat_amd import mx
    a, b = mx.quantize(rnd(0, 64, seed=1), 4), mx.quantize(rnd(5, 64, seed=2), 8)
    assert mx.matmul(a, b).shape == (0, 5) and mx.matmul(b, a).shape == (5, 0) and mx.dequantize(a).shape == (0, 64)
    g, m = mx.act_fwd(rnd(0, 8, seed=1, dtype=BF))
    assert g.shape == (0, 8) and mx.act_bwd(g, m)[0].shape == (0, 8)


def test_packing_past_two_to_the_31_elements():
    """Offsets are 64 bits wide."""
    from swat_amd import mx
    rows, n = 2 ** 20 + 5, 2080
    x = torch.zeros((rows, n), dtype=BF, device="cuda")
    x[-5:] = rnd(5, n, seed=3, dtype=BF)
    m = mx.quantize(x, 8)
    want, byte = F.held(x[-5:], 8)
    assert torch.equal(m.scale[-5:], byte) and not m.codes[:-5].any()
    assert same(mx.dequantize(mx.MX(m.codes[-9:], m.scale[-9:], n, 8))[-5:], want)
    out = mx.dequantize(m)
    assert same(out[-5:], want) and not out[rows // 2].any()
    del out, x
    w = mx.quantize(rnd(4, n, seed=4), 4)
    c = mx.matmul(m, w)
    A, B = want, mx.dequantize(w, F32).double()
    ref = A @ B.t()
    assert ((c[-5:].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (n + 8) * ULP * (A.abs() @ B.abs().t()) + eights(A) @ eights(B).t() * 2.0 ** -10).all()
    assert not c[:-5].any()


def test_packing_past_one_dimension_of_a_launch():
    """2^35 elements are 2^32 threads: one more row than a launch holds along its first dimension."""
    from swat_amd import mx
    rows, n = 2 ** 20 + 3, 2 ** 15
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 170 << 30:
        pytest.skip("needs 170 GB")
    x = torch.zeros((rows, n), dtype=BF, device="cuda")
    x[0] = rnd(n, seed=2, dtype=BF)
    x[-5:] = rnd(5, n, seed=3, dtype=BF)
    m = mx.quantize(x, 4)
    for a, b in ((0, 1), (rows - 5, rows)):
        want = mx.quantize(x[a:b], 4)
        assert torch.equal(m.codes[a:b], want.codes) and torch.equal(m.scale[a:b], want.scale)
    assert not m.codes[1:-5:4099].any()
    held = mx.dequantize(mx.MX(m.codes[-5:], m.scale[-5:], n, 4))
    out = mx.dequantize(m)
    assert torch.equal(out[-5:], held) and not out[1:-5:4099].any()


@pytest.mark.parametrize("abits,bbits", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("M,N,K", [(100003, 3, 32), (3, 100003, 32), (5, 9000, 96), (70, 3, 160)])
def test_product_of_few_scale_bytes(abits, bbits, M, N, K):
    """An operand of under 16 blocks, the other long."""
    test_product(abits, bbits, M, N, K)


def test_a_block_trained_with_checkpoints():
    """The operators together, as a block uses them: the seam's packed z is the MLP's input checkpoint and an operand of a 4-bit product; the
    pre-activation is kept in 8 bits; the backward pass reads the checkpoints.  Captured, replayed, and against 64 bits."""
    from swat_amd import mx, ops
    rows, d, n = 5 * 50, 256, 1024
    x, h = rnd(rows, d, seed=1), rnd(rows, d, seed=2, dtype=BF)
    w1, w2 = rnd(n, d, seed=3, scale=d ** -0.5, dtype=BF), rnd(d, n, seed=4, scale=n ** -0.5, dtype=BF)
    pre, scale, gate = (rnd(d, seed=5, scale=0.1) + 1, rnd(d, seed=6, scale=0.1)), rnd(d, seed=7, scale=0.3), torch.tensor([1.25, 0.0, 1.25, 1.25, 1.25]).cuda()
    dout, frozen = rnd(rows, d, seed=8, dtype=BF), mx.quantize(rnd(n, d, seed=9, scale=d ** -0.5), 4)

    def step():
        r = ops.residual_norm_fwd(x, h, pre=pre, gate=gate, scale=scale, pack=True)
        side = mx.matmul(r.z8, frozen)
        f = ops.linear_fwd(r.z, w1)
        g, f8 = mx.act_fwd(f, "gelu")
        out = ops.linear_fwd(g, w2)
        dg = ops.linear_dgrad(dout, w2)
        df, again = mx.act_bwd(dg, f8, "gelu")
        dw2 = ops.linear_wgrad(dout, again)
        dz = ops.linear_dgrad(df, w1)
        dw1, db1 = mx.linear_wgrad(df, r.z8, want_bias=True)
        grads = ops.residual_norm_bwd(None, dz, h, r.y, r.stats, pre=pre, gate=gate, scale=scale)
        return dict(y=r.y, z=r.z, side=side, f=f, g=g, out=out, dg=dg, df=df, again=again, dw2=dw2, dz=dz, dw1=dw1, db1=db1,
                    z8=mx.dequantize(r.z8, F32), f8=mx.dequantize(f8, F32), **{"grad_" + k: v for k, v in grads.items()})

    v = step()
    z8 = F.held(v["z"], 8)[0]
    assert same(v["z8"], z8) and same(v["f8"], F.held(v["f"], 8)[0])
    fz = mx.dequantize(frozen, F32).double()
    want = z8 @ fz.t()
    tol = 2.0 ** -8 * want.abs() + (d + 8) * ULP * (z8.abs() @ fz.abs().t()) + eights(z8) @ eights(fz).t() * 2.0 ** -10
    assert ((v["side"].double() - want).abs() <= tol).all()
    df = v["df"].double()
    small(v["dw1"], df.t() @ z8, df.abs().t() @ z8.abs(), rows + 64, "dW1")
    small(v["db1"], df.sum(0), df.abs().sum(0), rows + 64, "db1")
    ref, slope = F.act(v["f8"].double(), "gelu")
    assert ((df - v["dg"].double() * slope).abs() <= 2.0 ** -8 * (v["dg"].double() * slope).abs() + 2.0 ** -16 * v["dg"].double().abs()).all()
    grads = F.seam_bwd(None, v["dz"], h, v["y"], None, pre, gate, scale, 1.0, "layer", 1e-5)
    for k, (g, m) in grads.items():
        got = v["grad_" + k].double()
        half = 2.0 ** -8 if v["grad_" + k].dtype == BF else 0.0
        assert ((got - g).abs() <= 256 * ULP * m + half * g.abs() + 1e-30).all(), k

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for k in range(3):
        x.copy_(rnd(rows, d, seed=30 + k))
        dout.copy_(rnd(rows, d, seed=40 + k, dtype=BF))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for name in kept:
            assert torch.equal(kept[name], eager[name]), name


def test_two_streams_at_once():
    """Workspaces are a call's own: two calls that overlap do not share them."""
    from swat_amd import mx
    sets = [(rnd(1600, 320, seed=s, dtype=BF), mx.quantize(rnd(1600, 256, seed=s + 1), 8)) for s in (1, 5)]
    want = [mx.linear_wgrad(dy, m) for dy, m in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mx.linear_wgrad(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in (0, 1) for g in got[i])


def test_refusals():
    from swat_amd import _lib, mx
    x = rnd(8, 64, seed=1)
    m4, m8 = mx.quantize(x, 4), mx.quantize(x, 8)
    for f in (lambda: mx.quantize(x, 6), lambda: mx.quantize(x.half()), lambda: mx.quantize(x.t()), lambda: mx.quantize(x[:, :0]), lambda: mx.quantize(x[0]),
              lambda: mx.quantize(x[:1].expand(8, 64)), lambda: mx.dequantize(m8, torch.float16), lambda: mx.dequantize(x),
              lambda: mx.dequantize(mx.MX(m8.codes, m8.scale, 65, 8)), lambda: mx.dequantize(mx.MX(m8.codes, m8.scale[:4], 64, 8)),
              lambda: mx.dequantize(mx.MX(m8.codes, m8.scale, 64, 4)), lambda: mx.act_fwd(x), lambda: mx.act_fwd(x.bfloat16(), "relu"),
              lambda: mx.act_bwd(x.bfloat16(), m4), lambda: mx.act_bwd(x[:4].bfloat16(), m8), lambda: mx.act_bwd(x[:, :32].bfloat16(), m8),
              lambda: mx.linear_wgrad(x, m8), lambda: mx.linear_wgrad(x.bfloat16(), m4), lambda: mx.linear_wgrad(x[:4].bfloat16(), m8),
              lambda: mx.linear_wgrad(x.bfloat16(), m8, out=torch.empty(64, 63, device="cuda")),
              lambda: mx.matmul(m8, mx.quantize(x[:, :32])), lambda: mx.matmul(m8, m4, bias=rnd(7, seed=1)), lambda: mx.matmul(m8, m4, out_dtype=torch.float16),
              lambda: mx.matmul(x, m4), lambda: mx.matmul(m8, m4, out_dtype=F32), lambda: mx.matmul(m8, m8, out_dtype=F32)):
        with pytest.raises(_lib.SwatHipError):
            f()
