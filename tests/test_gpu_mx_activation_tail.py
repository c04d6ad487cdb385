"""GPU: GELU and QuickGELU where their value is small against x, relative to the value itself.

Tolerance: half a step of bfloat16 (2^-8 of the value) and 2^-14 of it for the arithmetic: the exponent of the density, up to 72 x 1.45 = 104
in powers of two, is off by its rounding (2^-24 x 104 x ln 2 = 2^-17.8), the tail's polynomial by 2^-20, and some twenty operations by 2^-23 each:
2^-17 together, eight times under that.  The slope's two terms cancel to no less than a 64th of their magnitudes below -3 (1 / x^2 of it), which
2^-14 x their sum covers."""
import math

import pytest
import torch

from helpers import mx_formulas as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def every(lo, hi):
    """Every bfloat16 number of [lo, hi], a block of 32 to each (which packs without a rounding of the others)."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    v = bits.view(BF)
    return v[torch.isfinite(v) & (v >= lo) & (v <= hi)].cuda()


def near(got, want, scale, what):
    over = ((got.double() - want).abs() / (2.0 ** -8 * want.abs() + 2.0 ** -14 * scale)).max().item()
    assert over <= 1.0, f"{what}: {over:.3g} of the tolerance"


@pytest.mark.parametrize("act", ["gelu", "quick_gelu"])
def test_the_tail_is_relative_to_itself(act):
    from swat_amd import mx
    x = every(-12.0, -0.5)
    f = torch.zeros((x.numel(), 32), dtype=BF, device="cuda")
    f[:, 3] = x
    g, m = mx.act_fwd(f, act)
    value, _ = F.act(x.double(), act)
    near(g[:, 3], value, value.abs(), "value")
    assert (g[:, 3] < 0).all() and not g[:, :3].any()
    held = mx.dequantize(m)[:, 3].double()
    df, again = mx.act_bwd(torch.ones_like(f), m, act)
    value, slope = F.act(held, act)
    near(again[:, 3], value, value.abs(), "value again")
    terms = (value / held + held.abs() * torch.exp(-0.5 * held ** 2) / math.sqrt(2 * math.pi)) if act == "gelu" else torch.sigmoid(1.702 * held) * (1 + 1.702 * held.abs())
    near(df[:, 3], slope, terms, "slope")
