"""GPU: the seam's backward with every tensor a view, at the narrowest widths, with a bias behind a root-mean-square norm, and past 2^31
elements.  Tolerances: those of test_gpu_residual_norm.py (7 rows to a team at most)."""
import pytest
import torch

from helpers import mx_formulas as F
from test_gpu_residual_norm import BF, EPS, F32, make, near, rnd

pytestmark = pytest.mark.gpu


def view(t, left, right):
    """The same values as columns of a wider matrix of NaN."""
    wide = torch.full((t.shape[0], t.shape[1] + left + right), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, left:left + t.shape[1]] = t
    return wide[:, left:left + t.shape[1]]


@pytest.mark.parametrize("gate", ["none", "group", "channel"])
@pytest.mark.parametrize("norm,bias", [("layer", True), ("rms", True), ("rms", False)])
@pytest.mark.parametrize("x,h,dz", [(F32, BF, BF), (BF, BF, BF), (F32, F32, F32)])
@pytest.mark.parametrize("rows,d", [(21, 2), (21, 3), (21, 5), (2400, 6), (21, 7), (300, 33), (27, 767), (27, 1027), (12, 2049)])
def test_views_and_narrow_rows(rows, d, x, h, dz, norm, bias, gate):
    from swat_amd import ops
    t = make(rows, d, norm, True, True, gate, 3, True, x, h, seed=500)
    if bias and norm == "rms":
        t["post"], t["pre"] = ((t[k][0], rnd(d, seed=507 + i, scale=0.1)) for i, k in enumerate(("post", "pre")))
    t["x"], t["h"] = view(t["x"], 1, 2), view(t["h"], 3, 1)
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"], alpha=-1.25, norm=norm)
    r = ops.residual_norm_fwd(t["x"], t["h"], eps=EPS, z_dtype=dz, **kw)
    y, mag = F.seam_fwd(t["x"], t["h"], t["post"], t["pre"], t["gate"], t["scale"], -1.25, norm, EPS)
    near(r.y, y, mag, 64, "y")
    z, zmag = F.seam_norm(r.y, t["pre"], norm, EPS)
    near(r.z, z, zmag, 64, "z")
    dy, g, yv = view(rnd(rows, d, seed=520, dtype=x), 2, 3), view(rnd(rows, d, seed=521, dtype=dz), 1, 0), view(r.y, 5, 2)
    got = ops.residual_norm_bwd(dy, g, t["h"], yv, r.stats, **kw)
    want = F.seam_bwd(dy, g, t["h"], r.y, t["post"], t["pre"], t["gate"], t["scale"], -1.25, norm, EPS)
    assert set(got) == set(want)
    for k, (ref, m) in want.items():
        near(got[k], ref, m, 128 if k in ("x", "h") else 256, k)


@pytest.mark.parametrize("gate", ["group", "channel"])
def test_backward_past_two_to_the_31_elements(gate):
    """Rows of zeros, and at both ends and in the middle three that are not: their gradients, and sums that only they enter."""
    from swat_amd import ops
    d, rows, groups = 8192, 2 ** 18 + 6, 2
    at = [0, 1, 2, rows // 2 - 1, rows // 2, rows // 2 + 1, rows - 3, rows - 2, rows - 1]
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    full = lambda t: torch.zeros((rows, d), dtype=BF, device="cuda").index_copy_(0, torch.tensor(at, device="cuda"), t)  # noqa: E731
    h, dy, dz = (rnd(9, d, seed=530 + i, dtype=BF) for i in range(3))
    pre, scale = (rnd(d, seed=540, mean=1.0, scale=0.1), rnd(d, seed=541, scale=0.1)), rnd(d, seed=542)
    gates = rnd(groups, seed=543) if gate == "group" else rnd(groups, d, seed=543)
    H = full(h)
    r = ops.residual_norm_fwd(H, H, pre=pre, scale=scale, gate=gates)
    got = ops.residual_norm_bwd(full(dy), full(dz), H, r.y, r.stats, pre=pre, scale=scale, gate=gates)
    # the nine rows by themselves, each with its group's gate: 5 of the first group (rows / 2 and beyond are the second's), 4 of the other
    own = torch.cat([gates[:1].expand(4, *gates.shape[1:]), gates[1:].expand(5, *gates.shape[1:])]).contiguous()
    want = F.seam_bwd(dy, dz, h, r.y[at], None, pre, own, scale, 1.0, "layer", EPS)
    near(got["x"][at], *want["x"], 128, "x")
    near(got["h"][at], *want["h"], 128, "h")
    assert not got["x"][3:rows // 2 - 1:977].any() and not got["h"][rows // 2 + 2:-3:977].any()
    # (additions of zeros are exact: the rows' order and nine additions are what is left)
    for k in ("scale", "pre_w", "pre_b"):
        near(got[k], *want[k], 256, k)
    ref, m = (torch.stack([t[:4].sum(0), t[4:].sum(0)]) for t in want["gate"])
    near(got["gate"], ref, m, 256, "gate")
