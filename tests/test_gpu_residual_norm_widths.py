"""GPU: the seam's backward at the towers' widths with shared gates and every combination of types, and what a channel scaled by zero
receives behind a norm.  Tolerances: those of test_gpu_residual_norm.py (at most 7 rows to a team here, 47 additions to a column)."""
import pytest
import torch

from helpers import mx_formulas as F
from test_gpu_residual_norm import BF, EPS, F32, make, near, rnd

pytestmark = pytest.mark.gpu


def check(t, rows, d, dz_type, with_dy=True):
    from swat_amd import ops
    kw = dict(post=t["post"], pre=t["pre"], gate=t["gate"], scale=t["scale"], alpha=0.75, norm=t["norm"])
    r = ops.residual_norm_fwd(t["x"], t["h"], eps=EPS, z_dtype=dz_type, **kw)
    y, mag = F.seam_fwd(t["x"], t["h"], t["post"], t["pre"], t["gate"], t["scale"], 0.75, t["norm"], EPS)
    near(r.y, y, mag, 64, "y")
    z, zmag = F.seam_norm(r.y, t["pre"], t["norm"], EPS)
    near(r.z, z, zmag, 64, "z")
    dy, dz = rnd(rows, d, seed=20, dtype=t["x"].dtype) if with_dy else None, rnd(rows, d, seed=21, dtype=dz_type)
    got = ops.residual_norm_bwd(dy, dz, t["h"], r.y, r.stats, **kw)
    want = F.seam_bwd(dy, dz, t["h"], r.y, t["post"], t["pre"], t["gate"], t["scale"], 0.75, t["norm"], EPS)
    assert set(got) == set(want)
    for k, (ref, m) in want.items():
        near(got[k], ref, m, 128 if k in ("x", "h") else 256, k)
    twice = ops.residual_norm_bwd(dy, dz, t["h"], r.y, r.stats, **kw)
    assert all(torch.equal(got[k], twice[k]) for k in got)
    return got, want


@pytest.mark.parametrize("gate,groups", [("group", 12), ("channel", 12), ("channel", 600), ("group", 1), ("channel", 1), ("none", 1)])
@pytest.mark.parametrize("rows,d", [(600, 512), (600, 768), (600, 1024), (600, 1280), (600, 2048), (600, 2304)])
def test_gates_at_the_widths_of_towers(rows, d, gate, groups):
    t = make(rows, d, "layer", True, True, gate, groups, True, F32, BF, seed=200)
    if gate == "group" and groups == 1:
        t["gate"].fill_(0.7)
    check(t, rows, d, BF)


@pytest.mark.parametrize("gate", ["none", "group", "channel"])
@pytest.mark.parametrize("x,h,dz", [(F32, F32, F32), (F32, BF, F32), (F32, F32, BF), (BF, BF, F32), (BF, F32, BF), (BF, F32, F32), (BF, BF, BF)])
@pytest.mark.parametrize("rows,d", [(3 * 701, 509), (3 * 701, 768), (420, 1024), (420, 4096)])
def test_every_combination_of_types(rows, d, x, h, dz, gate):
    """Teams of several rows, a last one that is shorter."""
    check(make(rows, d, "layer", True, True, gate, 3, True, x, h, seed=300), rows, d, dz, with_dy=gate != "group")


@pytest.mark.parametrize("d", [96, 768, 1030])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["none", "channel"])
def test_a_channel_scaled_by_zero_behind_a_norm(d, norm, gate):
    """It takes no part in y, but it has its share in the mean and the deviation of its row: its gradient is that of the formula, not zero; a
    row that is dropped whole has none."""
    rows = 24
    t = make(rows, d, norm, True, True, gate, 4, True, F32, BF, seed=400)
    t["scale"][[0, 40, d - 1]] = 0.0
    if gate == "channel":
        t["gate"][1] = 0.0        # rows 6 .. 11
    got, want = check(t, rows, d, BF)
    dead = got["h"][:, [0, 40, d - 1]]
    live = torch.ones(rows, dtype=torch.bool, device="cuda")
    if gate == "channel":
        live[6:12] = False
    assert (dead[live] != 0).all() and (want["h"][0][:, [0, 40, d - 1]][live] != 0).all()
    assert not got["h"][~live].any()
    assert torch.equal(got["post_w"][[0, 40, d - 1]], torch.zeros(3, device="cuda"))
