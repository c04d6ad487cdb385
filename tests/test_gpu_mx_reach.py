"""GPU: packed products and weight gradients whose offsets pass 2^31, rows cut out of a packed matrix, and a matrix by itself."""
import pytest
import torch

from helpers import mx_formulas as F

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
ULP = 2.0 ** -24


def rnd(*shape, seed, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def eights(x):
    return torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % 8)).view(x.shape[0], -(-x.shape[1] // 8), 8).amax(-1)


def test_weight_gradient_past_two_to_the_31_elements():
    """Rows of zeros but for some at both ends and in the middle: only those enter dW."""
    from swat_amd import mx
    rows, n, k = 2 ** 21 + 37, 1040, 1030
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    at = torch.tensor([0, 63, 64, rows // 2, rows - 65, rows - 2, rows - 1], device="cuda")
    dy, x = rnd(7, n, seed=1, dtype=BF), rnd(7, k, seed=2, dtype=BF)
    dY = torch.zeros((rows, n), dtype=BF, device="cuda").index_copy_(0, at, dy)
    m = mx.quantize(torch.zeros((rows, k), dtype=BF, device="cuda").index_copy_(0, at, x), 8)
    dw, db = mx.linear_wgrad(dY, m, want_bias=True)
    held, d = F.held(x, 8)[0], dy.double()
    assert ((dw.double() - d.t() @ held).abs() <= 16 * ULP * (d.abs().t() @ held.abs())).all()   # (7 terms; zeros add nothing)
    assert ((db.double() - d.sum(0)).abs() <= 16 * ULP * d.abs().sum(0)).all()


@pytest.mark.parametrize("abits,bbits,out", [(4, 4, F32), (8, 4, BF)])
def test_product_past_two_to_the_31_elements(abits, bbits, out):
    from swat_amd import mx
    M, N, K = 70001, 40003, 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    a, b = mx.quantize(rnd(M, K, seed=3), abits), mx.quantize(rnd(N, K, seed=4), bbits)
    c = mx.matmul(a, b, out_dtype=out)
    A, B = mx.dequantize(a, F32).double(), mx.dequantize(b, F32).double()
    for rows in (slice(0, 40), slice(35000, 35040), slice(M - 40, M)):
        want, mag = A[rows] @ B.t(), A[rows].abs() @ B.abs().t()
        tol = (K + 8) * ULP * mag + (2.0 ** -8 * want.abs() + eights(A[rows]) @ eights(B).t() * 2.0 ** -10 if out == BF else 0.0)
        assert ((c[rows].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_cut_out_of_a_matrix(bits):
    """At odd rows the scales start on any byte."""
    from swat_amd import mx
    for n in (33, 520, 1000):
        m, w = mx.quantize(rnd(700, n, seed=5), bits), mx.quantize(rnd(130, n, seed=6), 4)
        whole = mx.matmul(m, w)
        for a, b in ((1, 2), (3, 70), (5, 262), (699, 700), (7, 7)):
            cut = mx.MX(m.codes[a:b], m.scale[a:b], n, bits)
            assert torch.equal(mx.dequantize(cut), mx.dequantize(m)[a:b])
            got, A, B = mx.matmul(cut, w).double(), mx.dequantize(cut).double(), mx.dequantize(w).double()
            tol = 2.0 ** -7 * whole[a:b].double().abs() + (n + 8) * ULP * 2 * (A.abs() @ B.abs().t()) + eights(A) @ eights(B).t() * 2.0 ** -9
            assert ((got - whole[a:b].double()).abs() <= tol).all()   # (another tile, another order of the sums; both rounded to bfloat16, each by half a step)
            if bits == 8 and b > a:
                dy = rnd(b - a, 40, seed=7, dtype=BF)
                d = dy.double()
                assert ((mx.linear_wgrad(dy, cut).double() - d.t() @ A).abs() <= (b - a + 64) * ULP * (d.abs().t() @ A.abs())).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,K", [(5, 40), (300, 520), (1000, 768)])
def test_a_matrix_by_itself(bits, M, K):
    from swat_amd import mx
    m = mx.quantize(rnd(M, K, seed=8), bits)
    A = mx.dequantize(m).double()
    got, want = mx.matmul(m, m).double(), A @ A.t()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (K + 8) * ULP * (A.abs() @ A.abs().t()) + eights(A) @ eights(A).t() * 2.0 ** -10).all()
