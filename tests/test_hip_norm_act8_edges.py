"""-m gpu: layer norm and 8-bit activation checkpoints at the ends of their ranges: magnitudes, heights past a launch's rows, launch plans and
offsets that tests/test_hip_norm_act8.py does not reach.  Bounds: tests/norm_act8_ref.py."""
import pytest
import torch

from tests.gpu_util import DEV
from tests.norm_act8_ref import Norm64, inside
from tests.test_hip_norm_act8 import EPS, ops, params, rand

pytestmark = pytest.mark.gpu


# ---- magnitudes -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("scale", [1e20, 1e27, 3e37])
@pytest.mark.parametrize("D", [3, 33, 100, 256, 1419, 2048, 5397, 16384])
def test_layer_norm_of_rows_whose_squares_pass_fp32(D, scale, t):
    """finite rows have finite statistics, whatever their magnitude: squares overflow from 1.8e19 on, sums from 3.4e38 / D on (the
    statistics' relative bounds do not depend on the scale: Norm64's hold); rows beside them keep their bits"""
    M = 6
    small = rand((M, D), D, t).to(DEV)
    x = (rand((M, D), D, leaky=False) * scale).to(t).to(DEV)
    x[::2] = small[::2]
    w, b = (p.to(DEV) for p in params(D, D))
    y, mean, rstd, kept = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    plain = ops().layer_norm_fwd_raw(small, w, b, EPS, checkpoint="e4m3")
    for a, c in zip((y, mean, rstd, kept.codes), (plain[0], plain[1], plain[2], plain[3].codes)):
        assert torch.equal(a[::2], c[::2])
    ref = Norm64(x, w, b, EPS)
    inside(y, ref.y, ref.y_bound(t), "y")
    inside(mean, ref.mean[:, 0], ref.d_mean[:, 0], "mean")
    inside(rstd, ref.rstd[:, 0], (ref.d_rstd * ref.rstd)[:, 0], "rstd")
    g = rand((M, D), D + 1, t, 0.1, leaky=False).to(DEV)
    dx, dw, db = ops().layer_norm_bwd_raw(g, x, w, mean, rstd)
    ref.backward(g)
    inside(dx, ref.dx, ref.dx_bound(t), "dx")
    inside(dw, ref.dw, ref.d_dw, "dweight")
    inside(db, ref.db, ref.d_db, "dbias")


@pytest.mark.parametrize("D", [5, 96, 2048, 5397])
def test_layer_norm_of_large_constant_rows_and_bad_ones(D):
    x = rand((6, D), 8).to(DEV)
    x[1], x[2] = 3.1e25, -2.9e38
    x[3, D // 2], x[4, 0], x[5, D - 1] = float("nan"), float("inf"), -float("inf")
    w, b = (p.to(DEV) for p in params(D, 8))
    y, mean, rstd, _ = ops().layer_norm_fwd_raw(x, w, b, EPS)
    for r in (1, 2):
        assert torch.equal(y[r], b) and torch.equal(mean[r], x[r, 0]) and bool(rstd[r].isfinite())   # a constant row: h = 0
    for r in (3, 4, 5):
        assert bool(y[r].isnan().all()) and bool(mean[r].isnan()) and bool(rstd[r].isnan())
    assert bool(y[0].isfinite().all())
