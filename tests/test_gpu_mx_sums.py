"""GPU: the sums of the packed products, held to what additions in 32 bits leave of the RESULT, and calls at every alignment.

n additions of random terms, each off by at most half a step (2^-24) of a running sum that grows like the root of the number of terms so
far: the errors add up to 2^-24 x sqrt(1 + 2 + .. + n) = 2^-24 n / sqrt 2 of one term's size, or 2^-24 sqrt(n / 2) of the root of the sum of squares
of the products.  Held: 2^-24 sqrt(n) of it in the norm over all elements, 16 times that in a single one (a factor of 16 sqrt 2 over
the standard deviation).  One operand rounded to 13 places would miss the norm at every size here."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, D = torch.bfloat16, torch.float32, torch.float64
ULP = 2.0 ** -24


def rnd(*shape, seed, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def held_to(got, a, b, what, bias=None):
    """got against a^T b for a [terms, n], b [terms, k] in 64 bits."""
    terms = a.shape[0]
    want, rss = a.t() @ b, ((a * a).t() @ (b * b)).sqrt()
    if bias is not None:
        want, rss = want + bias, (rss * rss + bias * bias).sqrt()
    err, unit = (got.double() - want).abs(), ULP * terms ** 0.5 * rss
    assert torch.isfinite(got).all(), what
    rel = (err.norm() / unit.norm()).item()
    assert rel <= 1.0, f"{what}: norm {rel:.3g} of the tolerance"
    worst = (err / (16 * unit + ULP * want.abs() + 1e-30)).max().item()
    assert worst <= 1.0, f"{what}: an element {worst:.3g} of the tolerance"


@pytest.mark.parametrize("rows,n,k", [(64, 96, 96), (512, 200, 160), (1600, 768, 768), (4100, 130, 70), (16448, 256, 512), (16448, 1024, 1024)])
def test_weight_gradient_sums(rows, n, k):
    from swat_amd import mx
    m = mx.quantize(rnd(rows, k, seed=1), 8)
    dy = rnd(rows, n, seed=2, dtype=BF)
    dw, db = mx.linear_wgrad(dy, m, want_bias=True)
    held_to(dw, dy.double(), mx.dequantize(m, F32).double(), "dW")
    held_to(db[:, None], dy.double(), torch.ones((rows, 1), dtype=D, device="cuda"), "db")


@pytest.mark.parametrize("M,N,K", [(7, 300, 1024), (64, 512, 4096), (300, 400, 512), (1600, 768, 768), (4096, 1024, 4096), (8200, 2000, 1000)])
def test_product_sums(M, N, K):
    from swat_amd import mx
    a, b, bias = mx.quantize(rnd(M, K, seed=3), 4), mx.quantize(rnd(N, K, seed=4), 4), rnd(N, seed=5)
    A, B = mx.dequantize(a, F32).double(), mx.dequantize(b, F32).double()
    held_to(mx.matmul(a, b, out_dtype=F32), A.t(), B.t(), "C")
    held_to(mx.matmul(a, b, bias=bias, out_dtype=F32), A.t(), B.t(), "C + bias", bias.double()[None].expand(M, N))


@pytest.mark.parametrize("abits,bbits", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("M,N,K", [(47, 600, 1000), (1600, 768, 768), (8239, 1024, 1000)])
def test_a_product_repeats_itself(abits, bbits, M, N, K):
    from swat_amd import mx
    a, b, bias = mx.quantize(rnd(M, K, seed=6), abits), mx.quantize(rnd(N, K, seed=7), bbits), rnd(N, seed=8)
    first = mx.matmul(a, b, bias=bias)
    for _ in range(4):
        mx.matmul(b, a)
        assert torch.equal(mx.matmul(a, b, bias=bias), first)


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 7])
@pytest.mark.parametrize("rows", [1, 63, 64, 65, 127, 1601])
def test_weight_gradient_of_dy_on_any_element(offset, rows):
    """The base, the row stride and the width odd or even, each; NaN around what belongs to dY."""
    from swat_amd import mx
    k = 70
    m = mx.quantize(rnd(rows, k, seed=9), 8)
    x = mx.dequantize(m, F32).double()
    for n in (1, 2, 33, 64, 127, 200):
        for gap in (0, 1, 2, 5):
            ld = n + gap
            flat = torch.full((offset + rows * ld + 8,), float("nan"), dtype=BF, device="cuda")
            dy = torch.as_strided(flat, (rows, n), (ld, 1), offset)
            dy.copy_(rnd(rows, n, seed=10 + n, dtype=BF))
            dw, db = mx.linear_wgrad(dy, m, want_bias=True)
            d = dy.double()
            # (any rounding to nearest: each addition at most half a step of the running sum, the sum of magnitudes at most)
            assert ((dw.double() - d.t() @ x).abs() <= (rows + 64) * ULP * (d.abs().t() @ x.abs()) + 1e-30).all(), (n, gap)
            assert ((db.double() - d.sum(0)).abs() <= (rows + 64) * ULP * d.abs().sum(0) + 1e-30).all(), (n, gap)


@pytest.mark.parametrize("abits,bbits", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("M", [40, 2000])
def test_large_products_that_cancel_leave_the_small_one(abits, bbits, M):
    """+L, -L and s in a row, by ones: what is left is s, up to half a step of L for each of the three additions and, where s shares its eight
    columns with L and an operand has 8 bits, what the instruction drops there (2^-13 of L)."""
    from swat_amd import mx
    K, N = 512, 48
    g = torch.Generator().manual_seed(11)
    x = torch.zeros(M, K, dtype=D)
    at = torch.stack([torch.randperm(K, generator=g)[:3] for _ in range(M)])
    L = torch.full((M,), 6 * 2.0 ** 12 if abits == 4 else 448.0, dtype=D)
    s = torch.exp2(torch.randint(-6, 8, (M,), generator=g).double()) * (4.0 if abits == 4 else 2.0 ** -2)
    row = torch.arange(M)
    if abits == 4:   # s in a block of its own: 4 bits hold no two numbers that far apart
        at[:, 2] = torch.where((at[:, 2] // 32 == at[:, 0] // 32) | (at[:, 2] // 32 == at[:, 1] // 32), -1, at[:, 2])
        for m in torch.nonzero(at[:, 2] < 0)[:, 0].tolist():
            free = [c for c in range(K) if c // 32 not in (int(at[m, 0]) // 32, int(at[m, 1]) // 32)]
            at[m, 2] = free[int(torch.randint(len(free), (1,), generator=g))]
    x[row, at[:, 0]], x[row, at[:, 1]], x[row, at[:, 2]] = L, -L, s
    a, b = mx.quantize(x.float().cuda(), abits), mx.quantize(torch.ones(N, K, device="cuda"), bbits)
    assert torch.equal(mx.dequantize(a, F32).cpu().double(), x)
    shared = (at[:, 2] // 8 == at[:, 0] // 8) | (at[:, 2] // 8 == at[:, 1] // 8)
    tol = 3 * ULP * L + torch.where(shared & (abits + bbits > 8), 2.0 ** -13 * L, 0 * L)
    out = F32 if abits == bbits == 4 else BF
    got = mx.matmul(a, b, out_dtype=out).double().cpu()
    tol = (tol + (2.0 ** -8 * s if out == BF else 0))[:, None]
    over = ((got - s[:, None]).abs() / tol).max().item()
    assert over <= 1.0, f"{over:.3g} of the tolerance"


@pytest.mark.parametrize("M,N,K", [(47, 600, 1000), (1600, 768, 768)])
@pytest.mark.parametrize("abits,bbits", [(8, 4), (8, 8)])
def test_sums_in_32_bits_are_to_be_had(abits, bbits, M, N, K):
    """Unpacking is exact, so a linear layer on the unpacked matrices adds the same products in 32 bits."""
    from swat_amd import mx, ops
    a, b, bias = mx.quantize(rnd(M, K, seed=12), abits), mx.quantize(rnd(N, K, seed=13), bbits), rnd(N, seed=14)
    A, B = mx.dequantize(a), mx.dequantize(b)
    got = ops.linear_fwd(A, B, bias).double()
    A, B = A.double(), B.double()
    want = A @ B.t() + bias.double()
    unit = ULP * K ** 0.5 * ((A * A) @ (B * B).t() + bias.double() ** 2).sqrt()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 16 * unit).all()
    near = mx.matmul(a, b, bias=bias).double()
    assert (near - want).norm() <= (1 + 2.0 ** -8) * (got - want).norm()   # (and what the packed product drops does not show beside bfloat16)
