"""CPU: what the block-seam and microscaled entry points refuse before anything is launched, and the host-side formulas of the tests."""
import ctypes

import pytest
import torch

from helpers import mx_formulas as F


@pytest.fixture(scope="module")
def lib():
    import os
    from swat_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


P = 4096  # an address that is never read: every call below is refused first


def refused(lib, rc, word):
    assert rc < 0
    assert word in lib.swat_last_error().decode(), lib.swat_last_error()


def test_c_entries_refuse(lib):
    refused(lib, lib.swat_mx_quantize(P, 64, 0, 6, P, P, 4, 64, None), "bits")
    refused(lib, lib.swat_mx_quantize(P, 63, 0, 8, P, P, 4, 64, None), "stride")
    refused(lib, lib.swat_mx_quantize(P, 64, 0, 8, P + 8, P, 4, 64, None), "16 bytes")
    refused(lib, lib.swat_mx_quantize(None, 64, 0, 8, P, P, 4, 64, None), "needed")
    refused(lib, lib.swat_mx_quantize(P, 64, 0, 8, P, P, -1, 64, None), "rows")
    refused(lib, lib.swat_mx_quantize(P, 64, 0, 8, P, P, 4, 0, None), "columns")
    refused(lib, lib.swat_mx_quantize(P, 1 << 20, 0, 8, P, P, 1 << 40, 1 << 20, None), "launch")
    refused(lib, lib.swat_mx_dequantize(P, P, 5, P, 1, 4, 64, None), "bits")
    refused(lib, lib.swat_mx_act_fwd(P, 64, 0, P, P, P, 4, 64, None), "activation")
    refused(lib, lib.swat_mx_act_bwd(P, 64, P, P, 3, P, None, 4, 64, None), "activation")
    refused(lib, lib.swat_mx_linear_wgrad(P, 63, P, P, P, None, 4, 64, 32, None, 0, None), "stride")
    refused(lib, lib.swat_mx_linear_wgrad(P, 64, P + 4, P, P, None, 4, 64, 32, None, 0, None), "16 bytes")
    refused(lib, lib.swat_mx_linear_wgrad(P, 64, P, P, None, None, 4, 64, 32, None, 0, None), "needed")
    refused(lib, lib.swat_mx_matmul(P, P, 4, P, P, 5, None, P, 1, 4, 4, 64, None), "bits")
    refused(lib, lib.swat_mx_matmul(P, P, 4, P + 1, P, 4, None, P, 1, 4, 4, 64, None), "16 bytes")
    refused(lib, lib.swat_mx_matmul(P, P, 4, P, P, 4, None, P, 1, 4, 4, 0, None), "4 x 4")
    refused(lib, lib.swat_mx_matmul(P, P, 8, P, P, 4, None, P, 0, 4, 4, 64, None), "output type")
    refused(lib, lib.swat_mx_matmul(P, P, 4, P, P, 4, None, P, 1, 1, (1 << 30) + 1, 64, None), "1 x 10737")
    refused(lib, lib.swat_mx_matmul(P, P, 4, P, P, 4, None, P, 1, 1, 1 << 30, 32, None), "launch")
    refused(lib, lib.swat_mx_matmul(P, P, 4, P, P, 4, None, P, 1, 1 << 30, 1 << 30, 64, None), "launch")
    refused(lib, lib.swat_mx_linear_wgrad(P, 1 << 20, P, P, P, None, 64, 1 << 20, 1 << 20, None, 0, None), "launch")
    z = ctypes.c_void_p(None)
    refused(lib, lib.swat_residual_norm_fwd(P, 16, 0, P, 16, 0, z, z, P, 1 << 25, 0, z, z, z, 1.0, 0, 1e-5, P, z, 1, z, z, z, 1 << 26, 16, None), "launch")
    refused(lib, lib.swat_residual_norm_fwd(P, 16, 0, P, 16, 0, z, z, z, 0, 0, z, z, z, 1.0, 0, 1e-5, P, z, 1, z, z, z, 4, 8193, None), "8192")
    refused(lib, lib.swat_residual_norm_fwd(P, 16, 0, P, 16, 0, z, z, P, 3, 0, z, z, z, 1.0, 0, 1e-5, P, z, 1, z, z, z, 4, 16, None), "gates")
    refused(lib, lib.swat_residual_norm_fwd(P, 15, 0, P, 16, 0, z, z, z, 0, 0, z, z, z, 1.0, 0, 1e-5, P, z, 1, z, z, z, 4, 16, None), "strides")
    refused(lib, lib.swat_residual_norm_fwd(P, 16, 0, P, 16, 0, z, z, z, 0, 0, z, z, z, 1.0, 0, 1e-5, P, P, 1, z, z, z, 4, 16, None), "norm after")
    refused(lib, lib.swat_residual_norm_fwd(P, 16, 0, P, 16, 0, z, P, z, 0, 0, z, z, z, 1.0, 0, 1e-5, P, z, 1, z, z, z, 4, 16, None), "bias")
    args = lambda ws, n: (P, 16, z, 16, 1, P, 16, 0, P, 16, 0, z, z, z, z, 0, 0, z, z, z, 1.0, 0, P, P, z, z, z, z, z, z, ws, n, 4, 16, None)  # noqa: E731
    refused(lib, lib.swat_residual_norm_bwd(*args(P, 16)), "workspace")
    assert lib.swat_residual_norm_bwd_workspace_bytes(4, 9000, 0, 0) < 0
    assert lib.swat_residual_norm_bwd_workspace_bytes(0, 16, 0, 0) >= 0


def test_calls_without_a_gpu_are_refused():
    from swat_amd import _lib, mx, ops
    x = torch.zeros(4, 32)
    m = mx.MX(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 32, 8)
    for f in (lambda: mx.quantize(x), lambda: mx.dequantize(m), lambda: mx.act_fwd(x.bfloat16()), lambda: mx.act_bwd(x.bfloat16(), m),
              lambda: mx.linear_wgrad(x.bfloat16(), m), lambda: mx.matmul(m, m), lambda: ops.residual_norm_fwd(x, x),
              lambda: ops.residual_norm_bwd(x, None, x, None, torch.zeros(4, 4))):
        with pytest.raises(_lib.SwatHipError):
            f()


def test_more_columns_than_a_matrix_has_are_refused():
    from swat_amd import _lib, mx
    part = torch.zeros(1, 1, dtype=torch.uint8)
    for cols in (0, (1 << 24) + 1, (1 << 32) + 1):   # (the last would pass as 1 in 32 bits)
        with pytest.raises(_lib.SwatHipError, match="columns is wanted"):
            mx.dequantize(mx.MX(part, part, cols, 8))


def test_the_formats_of_the_formulas():
    """The grids are those of torch's own 8-bit type and of the sixteen 4-bit codes; ties go to the even code."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(F.grid(8), codes)
    x = torch.tensor([[6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] + [0.0] * 24])
    assert F.held(x, 4)[0][0, :8].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    v = torch.linspace(-448, 448, 4001).view(1, -1)
    v = torch.nn.functional.pad(v, (0, 31)).view(-1, 32)
    v[:, 31] = 448.0
    assert torch.equal(F.held(v, 8)[0].float(), v.to(torch.float8_e4m3fn).float())
