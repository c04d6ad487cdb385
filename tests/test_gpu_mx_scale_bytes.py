"""GPU: matrices put together from codes and scale bytes by hand, with every byte the format has: 2^(byte - 127), 0 to 254.

Packing never writes a byte under 17 (2^-110: every held value is a normal bfloat16 number); under it a value is rounded where it is
unpacked to bfloat16 (its own steps end at 2^-133) and exact everywhere else."""
import pytest
import torch

from helpers import mx_formulas as F

pytestmark = pytest.mark.gpu
BF, F32, D = torch.bfloat16, torch.float32, torch.float64
ULP = 2.0 ** -24


def by_hand(byte, bits, rows=48, blocks=3, seed=1):
    """-> an MX matrix of random codes (no NaN) under one scale byte, and its values in 64 bits."""
    from swat_amd import mx
    g = torch.Generator().manual_seed(seed + byte)
    n = 32 * blocks
    q = torch.randint(0, 256 if bits == 8 else 16, (rows, n), generator=g)
    if bits == 8:
        q = torch.where(q % 128 == 127, q - 1, q)
        codes = q
    else:
        codes = q[:, 0::2] | (q[:, 1::2] << 4)
    half = 1 << (bits - 1)
    v = torch.where(q >= half, -1.0, 1.0).to(D) * F.grid(bits)[q % half] * 2.0 ** (byte - 127)
    return mx.MX(codes.to(torch.uint8).cuda(), torch.full((rows, blocks), byte, dtype=torch.uint8, device="cuda"), n, bits), v.cuda()


@pytest.mark.parametrize("bits", [4, 8])
def test_unpacking_of_every_scale_byte(bits):
    from swat_amd import mx
    for byte in range(255):
        m, v = by_hand(byte, bits)
        assert torch.equal(mx.dequantize(m, F32), v.float()), byte
        assert torch.equal(mx.dequantize(m, BF), v.float().bfloat16()), byte


@pytest.mark.parametrize("byte", list(range(18)) + [127, 200])
def test_what_reads_a_matrix_made_by_hand(byte):
    from swat_amd import mx
    m8, v8 = by_hand(byte, 8)
    m4, v4 = by_hand(byte, 4)
    low = 2.0 ** -134 if byte < 17 else 0.0   # half a step of the smallest bfloat16 numbers
    dg = torch.full((48, 96), 2.0, device="cuda").to(BF)
    df, again = mx.act_bwd(dg, m8, "gelu")
    value, slope = F.act(v8, "gelu")
    assert ((again.double() - value).abs() <= 2.0 ** -8 * value.abs() + 2.0 ** -18 * v8.abs() + low).all()
    assert ((df.double() - 2 * slope).abs() <= 2.0 ** -8 * (2 * slope).abs() + 2.0 ** -17 * (1 + v8.abs())).all()
    up = 2.0 ** (100 if byte < 100 else -100)   # (the products are ordinary numbers again)
    g = torch.Generator().manual_seed(7)
    dy = (torch.randn(48, 40, generator=g) * up).to(BF).cuda()
    dw = mx.linear_wgrad(dy, m8)
    d = dy.double()
    tol = (48 + 64) * ULP * (d.abs().t() @ v8.abs()) + low * d.abs().sum(0)[:, None]
    assert ((dw.double() - d.t() @ v8).abs() <= tol).all()
    w = mx.quantize((torch.randn(24, 96, generator=g) * up).cuda(), 4)
    W = mx.dequantize(w, F32).double()
    want, mag = v4 @ W.t(), v4.abs() @ W.abs().t()
    assert ((mx.matmul(m4, w, out_dtype=F32).double() - want).abs() <= 104 * ULP * mag).all()
    want = v8 @ W.t()
    top = lambda t: t.abs().view(t.shape[0], -1, 8).amax(-1)  # noqa: E731
    tol = 2.0 ** -8 * want.abs() + 104 * ULP * (v8.abs() @ W.abs().t()) + top(v8) @ top(W).t() * 2.0 ** -10
    assert ((mx.matmul(m8, w).double() - want).abs() <= tol).all()
