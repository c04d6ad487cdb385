"""GPU: arguments of the wrong kind are refused as SwatHipError, like those of a wrong shape or type."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_residual_norm():
    from swat_amd import _lib, ops
    x, w = torch.randn(8, 16, device="cuda"), torch.ones(16, device="cuda")
    r = ops.residual_norm_fwd(x, x, pre=(w, None))
    for kw in (dict(gate=0.5), dict(gate=[1.0]), dict(pre=w), dict(post=w), dict(pre=(w,)), dict(pre=(w, None, None)), dict(post=5), dict(scale=2.0)):
        with pytest.raises(_lib.SwatHipError):
            ops.residual_norm_fwd(x, x, **kw)
        kw.setdefault("pre", (w, None))
        with pytest.raises(_lib.SwatHipError):
            ops.residual_norm_bwd(x, x, x, r.y, r.stats, **kw)
    for args in ((None, x, None, r.y, r.stats), (x, x, x, r.y, None), (x, x, x, 1.0, r.stats), ([1.0], x, x, r.y, r.stats)):
        with pytest.raises(_lib.SwatHipError):
            ops.residual_norm_bwd(*args, pre=(w, None))
    two = torch.ones(2, device="cuda")   # (a weight of two columns unpacks like a pair)
    with pytest.raises(_lib.SwatHipError):
        ops.residual_norm_fwd(x[:, :2], x[:, :2], pre=two)


def test_mx():
    from swat_amd import _lib, mx
    x = torch.randn(8, 32, device="cuda")
    m = mx.quantize(x)
    for f in (lambda: mx.quantize(None), lambda: mx.quantize(x, "8"), lambda: mx.dequantize(mx.MX(None, m.scale, 32, 8)),
              lambda: mx.dequantize(mx.MX(m.codes, None, 32, 8)), lambda: mx.dequantize(mx.MX(m.codes[0, 0], m.scale, 32, 8)),
              lambda: mx.dequantize(mx.MX(m.codes, m.scale, "32", 8)), lambda: mx.act_fwd(x.bfloat16(), ["gelu"]), lambda: mx.matmul(m, None),
              lambda: mx.matmul(m, m, bias=1.0), lambda: mx.linear_wgrad(x.bfloat16(), m, out=3), lambda: mx.linear_wgrad(None, m)):
        with pytest.raises(_lib.SwatHipError):
            f()
