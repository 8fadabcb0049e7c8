"""-m gpu: layer norm (forward, backward, column sums) and 8-bit activation checkpoints (pack, unpack, LeakyReLU', weight gradient) against
64-bit restatements (tests/norm_act8_ref.py), at the widths, heights, types, strides and values where they can go wrong."""
import numpy as np
import pytest
import torch

from tests.gpu_util import DEV
from tests.norm_act8_ref import SLOPE, TYPES, U, Norm64, half_step, inside, kept64, weight_grad

pytestmark = pytest.mark.gpu

EPS = 1e-5


def ops():
    from pivotcvae_amd import ops as o
    return o


def rand(shape, seed, t=torch.float32, scale=1.0, leaky=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale
    return (torch.where(x > 0, x, SLOPE * x) if leaky else x).to(t)


def params(D, seed):
    g = torch.Generator().manual_seed(seed + 77)
    return 1 + 0.2 * torch.randn(D, generator=g), 0.3 * torch.randn(D, generator=g)


WIDTHS = [1, 2, 7, 31, 32, 33, 64, 100, 128, 255, 256, 257, 512, 513, 1000, 1024, 1419, 2048, 2051, 4096, 5397, 8192, 8200, 16384]


# ---- layer norm ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", WIDTHS)
def test_layer_norm_forward_and_backward(D, t):
    M = 37 if D <= 2051 else 5
    x, g = rand((M, D), D, t).to(DEV), rand((M, D), D + 1, t, 0.1, leaky=False).to(DEV)
    w, b = (p.to(DEV) for p in params(D, D))
    y, mean, rstd, none = ops().layer_norm_fwd_raw(x, w, b, EPS)
    assert none is None and y.dtype == t and mean.dtype == rstd.dtype == torch.float32
    ref = Norm64(x, w, b, EPS)
    inside(y, ref.y, ref.y_bound(t), "y")
    inside(mean, ref.mean[:, 0], ref.d_mean[:, 0], "mean")
    inside(rstd, ref.rstd[:, 0], (ref.d_rstd * ref.rstd)[:, 0], "rstd")
    dx, dw, db = ops().layer_norm_bwd_raw(g, x, w, mean, rstd)
    ref.backward(g)
    inside(dx, ref.dx, ref.dx_bound(t), "dx")
    inside(dw, ref.dw, ref.d_dw, "dweight")
    inside(db, ref.db, ref.d_db, "dbias")


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 31, 257, 2049, 5000])
@pytest.mark.parametrize("D", [48, 256, 1500])
def test_layer_norm_heights(M, D):
    """one row to several rounds of the launch, batches that end inside a workgroup"""
    x, g = rand((M, D), M).to(DEV), rand((M, D), M + 1, scale=0.1, leaky=False).to(DEV)
    w, b = (p.to(DEV) for p in params(D, M))
    y, mean, rstd, kept = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    ref = Norm64(x, w, b, EPS)
    inside(y, ref.y, ref.y_bound(torch.float32), "y")
    q = kept64(x)
    assert torch.equal(kept.unpack().double().cpu(), q)
    for src, arg in ((None, x), (q, kept)):
        for leaky in (False, True):
            dx, dw, db = ops().layer_norm_bwd_raw(g, arg, w, mean, rstd, leaky=leaky)
            ref.backward(g, src, leaky)
            inside(dx, ref.dx, ref.dx_bound(torch.float32), "dx")
            inside(dw, ref.dw, ref.d_dw, "dweight")
            inside(db, ref.db, ref.d_db, "dbias")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [1, 30, 96, 256, 1419, 4097])
def test_layer_norm_from_its_checkpoint(D, t):
    M = 19
    x, g = rand((M, D), D + 5, t, 3.0).to(DEV), rand((M, D), D + 6, t, 0.1, leaky=False).to(DEV)
    w, b = (p.to(DEV) for p in params(D, D))
    y, mean, rstd, kept = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    plain = ops().layer_norm_fwd_raw(x, w, b, EPS)
    assert torch.equal(y, plain[0]) and torch.equal(mean, plain[1]) and torch.equal(rstd, plain[2])   # keeping changes nothing
    packed = ops().act8_pack(x)
    assert torch.equal(kept.codes, packed.codes)
    nb = -(-D // 32)
    rows = [sc.view(-1, nb, 8).transpose(1, 2).reshape(-1, nb)[:M] for sc in (kept.scales, packed.scales)]
    assert torch.equal(*rows)
    q = kept64(x)
    ref = Norm64(x, w, b, EPS).backward(g, q, leaky=True)
    dx, dw, db = ops().layer_norm_bwd_raw(g, kept, w, mean, rstd, leaky=True)
    inside(dx, ref.dx, ref.dx_bound(t), "dx")
    inside(dw, ref.dw, ref.d_dw, "dweight")
    inside(db, ref.db, ref.d_db, "dbias")


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_layer_norm_strides_windows_and_leading_dimensions(t):
    """column windows at odd offsets of wider buffers, transposed and broadcast operands, [.., D] shapes; what lies beside stays"""
    big = rand((23, 301), 3, t).to(DEV)
    w, b = (p.to(DEV) for p in params(100, 1))
    for x in (big[:, 1:101], big[::2, 7:107], big[:, 3:203:2][:, :100], big.t()[:100, :20].t(), big[4:5, 5:105].expand(6, 100)):
        y, mean, rstd, kept = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
        want = ops().layer_norm_fwd_raw(x.contiguous(), w, b, EPS, checkpoint="e4m3")
        assert torch.equal(y, want[0]) and torch.equal(kept.codes, want[3].codes)
        g = rand(tuple(x.shape), 9, t, leaky=False).to(DEV)
        wide = torch.zeros(x.shape[0], 150, dtype=t, device=DEV)
        wide[:, 13:113] = g
        for a, c in zip(ops().layer_norm_bwd_raw(wide[:, 13:113], x, w, mean, rstd), ops().layer_norm_bwd_raw(g, x.contiguous(), w, mean, rstd)):
            assert torch.equal(a, c)
    x3 = rand((2, 3, 5, 64), 4, t).to(DEV)
    y3, mean3, rstd3, kept3 = ops().layer_norm_fwd_raw(x3, checkpoint="e4m3")
    y2 = ops().layer_norm_fwd_raw(x3.reshape(30, 64))[0]
    assert y3.shape == x3.shape and torch.equal(y3.reshape(30, 64), y2) and kept3.unpack().shape == x3.shape
    one = ops().layer_norm_fwd_raw(x3[0, 0, 0])[0]
    assert one.shape == (64,) and torch.equal(one, y2[0])


def test_layer_norm_without_parameters_and_accumulating():
    x, g = rand((70, 200), 1).to(DEV), rand((70, 200), 2, leaky=False).to(DEV)
    w, b = (p.to(DEV) for p in params(200, 2))
    for ww, bb in ((None, None), (w, None), (None, b)):
        y, mean, rstd, _ = ops().layer_norm_fwd_raw(x, ww, bb, EPS)
        ref = Norm64(x, ww, bb, EPS).backward(g)
        inside(y, ref.y, ref.y_bound(torch.float32), "y")
        dx, dw, db = ops().layer_norm_bwd_raw(g, x, ww, mean, rstd)
        inside(dx, ref.dx, ref.dx_bound(torch.float32), "dx")
    dw0, db0 = torch.full_like(dw, 2.0), torch.full_like(db, -3.0)
    out = ops().layer_norm_bwd_raw(g, x, None, mean, rstd, dw0, db0)
    assert out[1] is dw0 and torch.equal(dw0, 2.0 + dw) and torch.equal(db0, -3.0 + db)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,D", [(1, 40), (30, 5), (301, 256), (4099, 99), (700, 2048), (300, 5397)])
def test_layer_norm_backward_over_its_own_gradient(M, D, t):
    """the C entry point with dx in g's memory"""
    from pivotcvae_amd import _hip
    x, g = rand((M, D), 1, t).to(DEV), rand((M, D), 2, t, 0.1, leaky=False).to(DEV)
    w, _ = (p.to(DEV) for p in params(D, 1))
    _, mean, rstd, _ = ops().layer_norm_fwd_raw(x, w)
    dx, dw, db = ops().layer_norm_bwd_raw(g, x, w, mean, rstd)
    L, k = _hip.lib(), _hip.ROW_TYPES[t]
    n = L.pcvae_layer_norm_bwd_ws_bytes(M, D, k)
    ws, dw2, db2 = torch.empty(n, dtype=torch.uint8, device=DEV), torch.empty_like(dw), torch.empty_like(db)
    _hip.check(L.pcvae_layer_norm_bwd(g.data_ptr(), D, k, M, D, x.data_ptr(), D, None, 0, None, 0, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), 0,
                                      g.data_ptr(), D, dw2.data_ptr(), db2.data_ptr(), 0, ws.data_ptr(), n, _hip.stream()))
    assert torch.equal(g, dx) and torch.equal(dw2, dw) and torch.equal(db2, db)


def test_refusals_on_the_device():
    o = ops()
    x = rand((6, 64), 1).to(DEV)
    y, mean, rstd, ck = o.layer_norm_fwd_raw(x, checkpoint="e4m3")
    for err, call in ((TypeError, lambda: o.layer_norm_fwd_raw(x.double())), (TypeError, lambda: o.layer_norm_fwd_raw(x, x[0].half())),
                      (RuntimeError, lambda: o.layer_norm_fwd_raw(x, x[0, :5].contiguous())), (RuntimeError, lambda: o.layer_norm_fwd_raw(x, eps=-1.0)),
                      (RuntimeError, lambda: o.layer_norm_fwd_raw(torch.zeros(2, 16385, device=DEV))), (RuntimeError, lambda: o.layer_norm_fwd_raw(x[:, :0])),
                      (RuntimeError, lambda: o.layer_norm_fwd_raw(x, mean.cpu())), (RuntimeError, lambda: o.layer_norm_bwd_raw(x[:5], x, None, mean, rstd)),
                      (TypeError, lambda: o.layer_norm_bwd_raw(x.half(), x, None, mean, rstd)), (ValueError, lambda: o.layer_norm_bwd_raw(x, x, None, None, rstd)),
                      (RuntimeError, lambda: o.layer_norm_bwd_raw(x, x, None, mean[:3], rstd)), (ValueError, lambda: o.act8_pack(x[:, :0])),
                      (ValueError, lambda: o.layer_norm_bwd_raw(x, x, None, mean, rstd, dweight=x[0])), (RuntimeError, lambda: o.act8_bwd_weight_raw(x[:5], ck)),
                      (ValueError, lambda: o.act8_bwd_weight_raw(x, ck, dW=torch.zeros(64, 64, device=DEV))),
                      (RuntimeError, lambda: o.act8_bwd_weight_raw(x, ck, torch.zeros(64, 63, device=DEV), torch.zeros(64, device=DEV))),
                      (ValueError, lambda: o.act8_bwd_weight_raw(x, ck, norm=(mean, None, None, None))), (RuntimeError, lambda: o.act8_leaky_bwd_(x[:, :3], ck)),
                      (ValueError, lambda: o.act8_leaky_bwd_(x.t().contiguous().t(), ck)), (TypeError, lambda: o.act8_bwd_weight_raw(x.double(), ck))):
        with pytest.raises(err):
            call()
    a = x.clone().requires_grad_()
    (ga,) = torch.autograd.grad(o.layer_norm(a).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):   # second derivatives
        ga.sum().backward()


def test_layer_norm_of_constant_rows_bad_values_and_no_rows():
    x = rand((6, 96), 8).to(DEV)
    x[1] = 0.0
    x[2] = 7.0
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    w, b = (p.to(DEV) for p in params(96, 8))
    y, mean, rstd, kept = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    for r in (1, 2):
        assert torch.equal(y[r], b)               # a constant row: h = 0
    assert bool(y[3].isnan().all()) and bool(y[4].isnan().all()) and bool(y[[0, 1, 2, 5]].isfinite().all())
    q = kept.unpack()
    assert bool(q[3, 5].isnan()) and bool(q[4, 6].isnan()) and int(q.isnan().sum()) == 2   # the neighbours are kept
    g = torch.ones_like(x)
    dx = ops().layer_norm_bwd_raw(g, x, w, mean, rstd)[0]
    assert bool(dx[3].isnan().all()) and bool(dx[[0, 1, 2, 5]].isfinite().all())
    none = torch.empty(0, 96, device=DEV)
    y, mean, rstd, kept = ops().layer_norm_fwd_raw(none, w, b, EPS, checkpoint="e4m3")
    dx, dw, db = ops().layer_norm_bwd_raw(none, none, w, mean, rstd)
    assert y.shape == dx.shape == (0, 96) and not dw.any() and not db.any()
    dx, dw, db = ops().layer_norm_bwd_raw(none, kept, w, mean, rstd, torch.ones_like(w), torch.ones_like(w))
    assert bool((dw == 1).all()) and bool((db == 1).all())


def test_layer_norm_large_offsets_of_the_mean():
    """rows far from zero: the variance is taken about the mean, not from moments"""
    x = (rand((9, 500), 3, leaky=False) * 1e-2 + 100.0).to(DEV)
    y, mean, rstd, _ = ops().layer_norm_fwd_raw(x)
    ref = Norm64(x, None, None, EPS)
    inside(y, ref.y, ref.y_bound(torch.float32), "y")
    assert float(ref.y_bound(torch.float32).max()) < 0.2 * float(ref.y.abs().max())


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_layer_norm_autograd_against_the_formula_and_differences(checkpoint):
    M, D = 6, 40
    x, t = rand((M, D), 5), rand((M, D), 6, leaky=False)
    w, b = params(D, 5)
    args = [v.to(DEV).requires_grad_() for v in (x, w, b)]
    (ops().layer_norm(*args, EPS, checkpoint) * t.to(DEV)).sum().backward()
    src = kept64(x) if checkpoint else None
    ref = Norm64(x, w, b, EPS).backward(t, src)
    inside(args[0].grad, ref.dx, ref.dx_bound(torch.float32), "dx")
    inside(args[1].grad, ref.dw, ref.d_dw, "dw")
    inside(args[2].grad, ref.db, ref.d_db, "db")
    if checkpoint is None:   # central differences of the 64-bit loss along random directions: (f(+s) - f(-s)) / 2s is off by O(s^2)
        gen = torch.Generator().manual_seed(1)
        for k, v in enumerate((x, w, b)):
            for _ in range(3):
                d = torch.randn(v.shape, generator=gen, dtype=torch.float64)
                s = 1e-4

                def loss(sign):
                    p = [q.double() for q in (x, w, b)]
                    p[k] = p[k] + sign * s * d
                    mu = p[0].mean(1, keepdim=True)
                    c = p[0] - mu
                    return float((((c / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)) * p[1] + p[2]) * t.double()).sum())

                slope = (loss(1) - loss(-1)) / (2 * s)
                got = float((args[k].grad.double().cpu() * d).sum())
                assert abs(slope - got) <= 1e-4 * float((args[k].grad.double().cpu() * d).abs().sum())
    only = x.to(DEV)
    wg = w.to(DEV).requires_grad_()
    ops().layer_norm(only, wg, None).sum().backward()   # an input without a gradient, no bias
    assert only.grad is None and wg.grad is not None


# ---- 8-bit rows -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [1, 3, 31, 32, 33, 64, 100, 127, 129, 256, 1419, 5397])
def test_pack_holds_exactly_the_defined_values(D, t):
    for M, scale in ((1, 1.0), (3, 1e-3), (66, 30.0)):
        x = rand((M, D), D + M, t, scale).to(DEV)
        ck = ops().act8_pack(x)
        assert ck.codes.shape == (M, -(-D // 32) * 32) and not ck.codes[:, D:].any()
        q = kept64(x)
        assert torch.equal(ck.unpack(torch.float32).double().cpu(), q)
        for out in TYPES:
            assert torch.equal(ck.unpack(out).cpu(), q.float().to(out))
        assert torch.equal(ck.unpack(torch.float32).cpu() > 0, x.cpu() > 0)   # LeakyReLU' reads off the codes


def test_pack_of_every_rounding_border_and_extreme():
    """all e4m3 values, the ties between them and their neighbours, at the smallest, ordinary and largest scales; zeros; subnormals"""
    e4 = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (e4[:-1] + e4[1:]) / 2
    pts = torch.cat([e4, mid, torch.nextafter(mid, torch.full_like(mid, 1e9)), torch.nextafter(mid, torch.zeros_like(mid))])
    pts = torch.cat([pts, -pts])
    rows = []
    for e in (-149, -140, -130, -126, -120, -117, -60, 0, 60, 118, 119):
        p = pts.double() * 2.0 ** e
        p = p[p.abs() <= 1.875 * 2.0 ** 127].float()
        p = p[: len(p) // 31 * 31].view(-1, 31)
        lead = torch.full((p.shape[0], 1), 448.0).double() * 2.0 ** e
        rows.append(torch.cat([lead.clamp(max=1.75 * 2.0 ** 127).float(), p], 1))
    x = torch.cat(rows)
    x = torch.cat([x, torch.zeros(1, 32), torch.full((1, 32), -0.0), torch.full((1, 32), 2.0 ** -149), torch.full((1, 32), -2.0 ** -149),
                   torch.full((1, 32), 3.4028234663852886e38), torch.full((1, 32), -3.4028234663852886e38)])
    ck = ops().act8_pack(x.to(DEV))
    got, want = ck.unpack().cpu().double(), kept64(x)
    assert torch.equal(got, want), (got - want).abs().max()
    assert torch.equal(got > 0, x > 0)


def test_pack_keeps_nan_and_infinity_out_of_the_scale():
    x = rand((4, 64), 1).to(DEV)
    want = kept64(x)
    x[0, 3], x[1, 40], x[2, 0] = float("nan"), float("inf"), -float("inf")
    x[3, :32] = float("nan")
    q = ops().act8_pack(x).unpack().cpu().double()
    ref = kept64(x)
    assert torch.equal(q.isnan(), ref.isnan()) and torch.equal(q.nan_to_num(0), ref.nan_to_num(0))
    assert bool((q[0, 32:] == want[0, 32:]).all()) and int(q.isnan().sum()) == 35


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_pack_windows_and_leaky_backward_in_place(t):
    big = rand((21, 500), 2, t).to(DEV)
    for x in (big[:, 1:334], big[::3, 5:130], big.t()[:50], big[3:4, :77].expand(5, 77), big[:0, :40]):
        ck = ops().act8_pack(x)
        assert torch.equal(ck.unpack(torch.float32).double().cpu(), kept64(x.contiguous()))
        wide = rand((x.shape[0], x.shape[1] + 9), 6, t, leaky=False).to(DEV)
        before = wide.clone()
        g = wide[:, 4:4 + x.shape[1]]
        assert ops().act8_leaky_bwd_(g, ck) is g
        want = torch.where(x > 0, before[:, 4:4 + x.shape[1]].float(), SLOPE * before[:, 4:4 + x.shape[1]].float()).to(t)
        assert torch.equal(g, want)
        assert torch.equal(wide[:, :4], before[:, :4]) and torch.equal(wide[:, 4 + x.shape[1]:], before[:, 4 + x.shape[1]:])


# ---- weight gradient --------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 8, 16), (2, 3, 33), (31, 17, 30), (32, 128, 128), (33, 129, 127), (64, 256, 102), (65, 200, 257), (257, 64, 1419), (256, 300, 64),
          (1000, 130, 300), (2500, 256, 256), (5000, 40, 700)]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_weight_gradient(M, N, K, normed, t):
    x, g = rand((M, K), M + K, torch.float32, 2.0).to(DEV), rand((M, N), M + N, t, 0.1, leaky=False).to(DEV)
    ck = ops().act8_pack(x)
    q = kept64(x)
    norm = None
    if normed:
        _, mean, rstd, _ = ops().layer_norm_fwd_raw(x)
        norm = (mean, rstd, *(p.to(DEV) for p in params(K, K)))
    dW, db = ops().act8_bwd_weight_raw(g, ck, norm=norm)
    want, bound, wdb, bdb = weight_grad(g, q, norm)
    inside(dW, want, bound, "dW")
    inside(db, wdb, bdb, "db")
    again = ops().act8_bwd_weight_raw(g, ck, norm=norm)
    assert torch.equal(again[0], dW) and torch.equal(again[1], db)      # the same bits every run
    wide = torch.full((N, K + 5), 0.5, device=DEV)
    acc = wide[:, 2:2 + K]
    b2 = torch.full((N,), 0.25, device=DEV)
    ops().act8_bwd_weight_raw(g, ck, acc, b2, norm=norm)
    assert torch.equal(acc, 0.5 + dW) and torch.equal(b2, 0.25 + db)
    assert bool((wide[:, :2] == 0.5).all()) and bool((wide[:, 2 + K:] == 0.5).all())


def test_weight_gradient_of_gradient_windows_and_no_rows():
    M, N, K = 90, 70, 50
    x = rand((M, K), 1).to(DEV)
    ck = ops().act8_pack(x)
    wide = rand((M, 3 * N), 2, leaky=False).to(DEV)
    for g in (wide[:, 1:1 + N], wide[:, ::3], wide.t()[:N].t(), wide[5:6, :N].expand(M, N)):
        a, c = ops().act8_bwd_weight_raw(g, ck), ops().act8_bwd_weight_raw(g.contiguous(), ck)
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    none = ops().act8_pack(torch.empty(0, K, device=DEV))
    dW, db = ops().act8_bwd_weight_raw(torch.empty(0, N, device=DEV), none)
    assert dW.shape == (N, K) and not dW.any() and not db.any()
    keep = torch.ones(N, K, device=DEV)
    ops().act8_bwd_weight_raw(torch.empty(0, N, device=DEV), none, keep, torch.ones(N, device=DEV))
    assert bool((keep == 1).all())


def test_weight_gradient_of_one_row_is_the_exact_product():
    """one row: every product of an fp32 gradient with a code is rounded once"""
    x, g = rand((1, 300), 5).to(DEV), rand((1, 200), 6, leaky=False).to(DEV)
    dW, db = ops().act8_bwd_weight_raw(g, ops().act8_pack(x))
    want = g.double().cpu().t() @ kept64(x)
    assert float(((dW.double().cpu() - want).abs() / want.abs().clamp(min=1e-30)).max()) <= 3 * U   # three components, added in fp32
    assert torch.equal(db, g[0])


def test_weight_gradient_bad_values_stay_in_their_row_and_column():
    x, g = rand((40, 70), 1).to(DEV), rand((40, 50), 2, leaky=False).to(DEV)
    good = ops().act8_bwd_weight_raw(g, ops().act8_pack(x))[0]
    x[39, 7] = float("nan")
    g2 = g.clone()
    g2[38, 9] = float("nan")
    dW, db = ops().act8_bwd_weight_raw(g2, ops().act8_pack(x))
    bad = torch.zeros(50, 70, dtype=torch.bool)
    bad[9], bad[:, 7] = True, True
    assert torch.equal(dW.isnan().cpu(), bad) and torch.equal(dW[~bad.to(DEV)], good[~bad.to(DEV)])
    assert bool(db[9].isnan()) and int(db.isnan().sum()) == 1


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,N,K,normed", [(8197, 300, 520, False), (8200, 301, 519, True), (16421, 129, 1000, False)])
def test_weight_gradient_in_wide_tiles(M, N, K, normed, t):
    """over 2048 chunks of 32 rows in all tiles: 128 x 256 tiles, several ranges of rows and a ragged last one"""
    assert -(-N // 128) * -(-K // 256) * -(-M // 32) >= 2048
    x, g = rand((M, K), 11, torch.float32, 2.0).to(DEV), rand((M, N), 12, t, 0.1, leaky=False).to(DEV)
    ck = ops().act8_pack(x)
    norm = None
    if normed:
        _, mean, rstd, _ = ops().layer_norm_fwd_raw(x)
        norm = (mean, rstd, *(p.to(DEV) for p in params(K, K)))
    dW, db = ops().act8_bwd_weight_raw(g, ck, norm=norm)
    want, bound, wdb, bdb = weight_grad(g, kept64(x), norm)
    inside(dW, want, bound, "dW")
    inside(db, wdb, bdb, "db")
    assert torch.equal(ops().act8_bwd_weight_raw(g, ck, norm=norm)[0], dW)


def test_rows_behind_offsets_over_32_bits():
    """row strides that take a batch past 2^31 elements, and 2^32 bytes of codes"""
    ld, M, D = 1 << 20, 2100, 40
    base = torch.empty(ld * M, dtype=torch.bfloat16, device=DEV)
    x = base.as_strided((M, D), (ld, 1))
    src = rand((M, D), 3, torch.bfloat16).to(DEV)
    x.copy_(src)
    w, b = (p.to(DEV) for p in params(D, 1))
    y, mean, rstd, ck = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    want = ops().layer_norm_fwd_raw(src, w, b, EPS, checkpoint="e4m3")
    assert torch.equal(y, want[0]) and torch.equal(ck.codes, want[3].codes) and torch.equal(ops().act8_pack(x).codes, ck.codes)
    g = rand((M, D), 4, torch.bfloat16, leaky=False).to(DEV)
    for a, c in zip(ops().layer_norm_bwd_raw(g, x, w, mean, rstd), ops().layer_norm_bwd_raw(g, src, w, mean, rstd)):
        assert torch.equal(a, c)
    x.copy_(g)   # now a gradient with far rows
    for a, c in zip(ops().act8_bwd_weight_raw(x, ck), ops().act8_bwd_weight_raw(g, ck)):
        assert torch.equal(a, c)
    for a, c in zip(ops().layer_norm_bwd_raw(x, src, w, mean, rstd), ops().layer_norm_bwd_raw(g, src, w, mean, rstd)):
        assert torch.equal(a, c)


# ---- streams, graphs, repetition --------------------------------------------------------------------------------------------------------
def _pass(x, g, gz, w, b):
    y, mean, rstd, ck = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    dW, db = ops().act8_bwd_weight_raw(gz, ck, norm=(mean, rstd, w, b))
    return (y, dW, db) + ops().layer_norm_bwd_raw(g, ck, w, mean, rstd, leaky=True) + ops().layer_norm_bwd_raw(g, x, w, mean, rstd) + \
        (ck.unpack(), ops().act8_leaky_bwd_(g.clone(), ck))


def test_captured_replayed_and_on_other_streams():
    M, D, N = 700, 200, 90
    w, b = (p.to(DEV) for p in params(D, 1))
    x, g, gz = rand((M, D), 1).to(DEV), rand((M, D), 2, leaky=False).to(DEV), rand((M, N), 3, leaky=False).to(DEV)
    eager = [t.clone() for t in _pass(x, g, gz, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _pass(x, g, gz, w, b)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(eager, other))
    graphs = []
    for _ in range(2):   # two graphs of the same calls, replayed on two streams at once
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = _pass(x, g, gz, w, b)
        graphs.append((gr, out))
    for k in range(4):
        x.copy_(rand((M, D), 10 + k).to(DEV))
        gz.copy_(rand((M, N), 20 + k, leaky=False).to(DEV))
        for t in graphs[0][1] + graphs[1][1]:
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        want = _pass(x, g, gz, w, b)
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(want, out)), k


# ---- stacks -----------------------------------------------------------------------------------------------------------------------------
def _stack(widths, seed, norms):
    g = torch.Generator().manual_seed(seed)
    layers = [(torch.randn(o, i, generator=g) / i ** 0.5, 0.1 * torch.randn(o, generator=g)) for i, o in zip(widths[:-1], widths[1:])]
    nrm = [(1 + 0.1 * torch.randn(o, generator=g), 0.1 * torch.randn(o, generator=g)) for o in widths[1:]] if norms else None
    return layers, nrm


def _to(dev_pairs):
    return [tuple(t.to(DEV).requires_grad_() for t in p) for p in dev_pairs]


@pytest.mark.parametrize("normed,checkpoint", [(False, "e4m3"), (True, None), (True, "e4m3")])
@pytest.mark.parametrize("shape", ["mlp linear", "mlp activated", "heads"])
def test_stack_with_norms_and_checkpoints(shape, normed, checkpoint):
    """a stack's outputs and every gradient against a 64-bit pass that keeps what the stack keeps.  Activations are taken from the same
    forward kernels run layer by layer (their own bits decide the codes); gradients of a stack of three layers of width <= 60 over 75
    rows in fp32: every value passes at most 8 sums of 75 terms, so 1e-5 of the largest magnitude (160 u) is allowed"""
    o = ops()
    widths, M = [37, 60, 33, 20], 75
    layers, nrm = _stack(widths, 4, normed)
    heads = shape == "heads"
    last_linear = shape == "mlp linear"
    hw, _ = _stack([widths[-1], 9], 8, False)
    hv, _ = _stack([widths[-1], 9], 9, False)
    P = _to(layers)
    NP = _to(nrm if heads else nrm[:-1]) if normed else None
    H = _to(hw + hv) if heads else []
    x = rand((M, widths[0]), 3, leaky=False).to(DEV).requires_grad_()
    if heads:
        outs = o.mlp_heads(x, P, H[0], H[1], norms=NP, checkpoint=checkpoint)
    else:
        outs = (o.mlp(x, P, last_linear, norms=NP, checkpoint=checkpoint),)
    ts = [rand(tuple(t.shape), 30 + i, leaky=False).to(DEV) for i, t in enumerate(outs)]
    sum((t * y).sum() for t, y in zip(ts, outs)).backward()

    # the same forward kernels, layer by layer
    keep, h = [x.detach()], x.detach()
    stats, n = [], len(P)
    for i in range(n):
        hidden = i < n - 1 or heads
        h = o.linear_fwd_raw(h, P[i][0].detach(), P[i][1].detach(), 1 if hidden or not last_linear else 0)
        top = h
        if hidden:
            keep.append(h)
            if normed:
                h, mean, rstd, _ = o.layer_norm_fwd_raw(h, NP[i][0].detach(), NP[i][1].detach())
                stats.append((mean, rstd))
    final = [o.linear_fwd_raw(h, a.detach(), c.detach(), 0) for a, c in H] if heads else [h]
    assert all(torch.equal(a, c) for a, c in zip(outs, final))

    D = lambda t: t.detach().double().cpu()   # noqa: E731
    q = [kept64(k) if checkpoint else D(k) for k in keep]
    inputs = [q[0]]
    for i in range(1, len(q)):
        if normed:
            mu, r = (D(s)[:, None] for s in stats[i - 1])
            inputs.append((q[i] - mu) * r * D(NP[i - 1][0]) + D(NP[i - 1][1]))
        else:
            inputs.append(q[i])

    def close(got, want, what):
        assert float((D(got) - want).abs().max()) <= 1e-5 * max(float(want.abs().max()), 1e-3), what

    def into(i, g):
        if normed:
            mu, r = (D(s)[:, None] for s in stats[i - 1])
            hh = (q[i] - mu) * r
            close(NP[i - 1][0].grad, (g * hh).sum(0), f"norm {i} weight")
            close(NP[i - 1][1].grad, g.sum(0), f"norm {i} bias")
            u = g * D(NP[i - 1][0])
            g = r * (u - u.mean(1, keepdim=True) - hh * (u * hh).mean(1, keepdim=True))
        return g * torch.where(D(keep[i]) > 0, 1.0, SLOPE)

    if heads:
        for (W, b), t in zip(H, ts):
            close(W.grad, D(t).t() @ inputs[n], "head weight")
            close(b.grad, D(t).sum(0), "head bias")
        g = into(n, sum(D(t) @ D(W) for (W, _), t in zip(H, ts)))
    else:
        g = D(ts[0])
        if not last_linear:
            g = g * torch.where(D(top) > 0, 1.0, SLOPE)
    for i in range(n - 1, -1, -1):
        close(P[i][0].grad, g.t() @ inputs[i], f"layer {i} weight")
        close(P[i][1].grad, g.sum(0), f"layer {i} bias")
        g = g @ D(P[i][0])
        if i > 0:
            g = into(i, g)
    close(x.grad, g, "x")


def test_stack_keeps_a_quarter_and_trains_nothing_without_gradients():
    o = ops()
    M, W = 4096, 256
    layers, _ = _stack([W] * 6, 1, False)
    P = _to(layers)
    x = rand((M, W), 1).to(DEV)

    def held(**kw):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = o.mlp(x, P, True, **kw)
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated() - before - y.numel() * 4, y

    full, y0 = held()
    kept, y1 = held(checkpoint="e4m3")
    assert torch.equal(y0, y1)
    assert full >= 4 * M * W * 4                       # (x itself is the caller's)
    assert kept <= 1.05 * 5 * M * W * (1 + 1 / 32)     # five inputs, x among them, at 1 + 1/32 bytes
    with torch.no_grad():
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y2 = o.mlp(x, P, True, checkpoint="e4m3")
        torch.cuda.synchronize()
        assert torch.equal(y2, y0) and torch.cuda.memory_allocated() - before <= y2.numel() * 4 + 512


# ---- models -----------------------------------------------------------------------------------------------------------------------------
S, D, Z, H, HP, NU = 5, 32, 8, 64, 32, 50


def make(variant, N=500, layer_norm=False, seed=0):
    import pivotcvae_amd as pa
    from oracle import pivotcvae_oracle as orc
    from pivotcvae_amd.models.listcvae import UserListCVAEWithPrior
    torch.manual_seed(seed)
    e, u = orc.synthetic_tables(N, NU, D, seed=seed)
    C = S + 1
    doc, usr = torch.nn.Embedding.from_pretrained(e), torch.nn.Embedding.from_pretrained(u)
    enc, prior = [S * D + C + D, H, H], [C + D, HP, HP]
    if variant == "listcvae":
        return UserListCVAEWithPrior(doc, usr, S, D, Z, C, enc, [Z + C + D, H, H, S * D], prior, False, DEV, layer_norm=layer_norm)
    return pa.PIVOTCVAE_MODELS[variant](doc, usr, S, D, Z, C, enc, [Z + C + D, H, H, D], [Z + C + 2 * D, H, H, (S - 1) * D], prior, False, DEV,
                                        layer_norm=layer_norm)


def batch(B, N=500, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, N, (B, S), generator=g).to(DEV), (torch.rand(B, S, generator=g) < 0.5).float().to(DEV),
            torch.randint(0, NU, (B, 1), generator=g).to(DEV), torch.randn(B, Z, generator=g).to(DEV))


@pytest.mark.parametrize("variant", ["pivotcvae_gt_pi", "pivotcvae_sgt_pi", "listcvae"])
def test_checkpointed_model_has_the_same_loss_and_bias_gradients(variant):
    """without norms the 8-bit activations only enter weight gradients: forward, loss, and every gradient that runs along the chain
    (all bias gradients) are what fp32 activations give; weight gradients differ by the codes' rounding, 2^-4 of a value"""
    s, r, u, eps = batch(96)
    res = {}
    for ck in (None, "e4m3"):
        m = make(variant)
        m.FUSED_TRAIN_PATH = False
        m.set_activation_checkpoint(ck)
        loss, rec, kld = m.loss(s, r, u, 0.01, eps=eps)
        loss.backward()
        res[ck] = (loss.detach(), {k: p.grad for k, p in m.named_parameters() if p.grad is not None})
    assert torch.equal(res[None][0], res["e4m3"][0])
    assert res[None][1].keys() == res["e4m3"][1].keys() and len(res[None][1]) > 10
    for k, g in res[None][1].items():
        got = res["e4m3"][1][k]
        if k.endswith("bias"):
            # column sums of the same rows in another order: 96 terms, at most 96 u of the sum of magnitudes; magnitudes <= 100 x the sum
            torch.testing.assert_close(got, g, rtol=1e-4, atol=1e-7, msg=k)
        else:
            assert float((got - g).norm()) <= 2.0 ** -4 * float(g.norm()) * 2, k


@pytest.mark.parametrize("variant", ["pivotcvae_gt_pi", "pivotcvae_spt_pi", "listcvae"])
def test_normed_checkpointed_model_trains_captured_as_eagerly_and_recommends(variant):
    """Trainer steps of a model with norms and 8-bit checkpoints: the captured step follows the eager one bit for bit; then slates"""
    from pivotcvae_amd.train_generative import Trainer
    runs = []
    for graph in (False, True):
        m = make(variant, layer_norm=True)
        m.set_activation_checkpoint("e4m3")
        tr = Trainer(m, lr=1e-3, beta=0.01, capture_graph=graph)
        assert any("norm" in k for k, _ in m.named_parameters())
        before = {k: p.detach().clone() for k, p in m.named_parameters()}
        losses = []
        for i in range(4):
            s, r, u, _ = batch(128, seed=i)
            losses.append(float(tr.step(s, r, u)[0]))
            torch.cuda.synchronize()
        assert not graph or (tr.capture_failed is None and tr._graph is not None)
        assert all(np.isfinite(losses))
        moved = {k for k, p in m.named_parameters() if not torch.equal(p, before[k])}
        assert all(k in moved for k, _ in m.named_parameters() if not k.startswith(("psm", "docEmbed", "userEmbed")))
        items, _ = m.recommend(r, u, return_item=True, eps=torch.zeros(128, Z, device=DEV))
        runs.append((losses, items, [p.detach().clone() for p in m.parameters()]))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])
    assert all(torch.equal(a, c) for a, c in zip(runs[0][2], runs[1][2]))


def test_normed_model_encodes_as_the_definition_and_round_trips():
    import io
    m = make("pivotcvae_gt_pi", layer_norm=True)
    s, r, u, eps = batch(40)
    with torch.no_grad():
        mu, lv = m.sample_encoding(s, r, u)
        x = torch.cat([m.docEmbed.weight[s.reshape(-1)].reshape(40, -1), m.get_condition(r), m.userEmbed.weight[u.reshape(-1)]], 1).double()
        for i in (1, 2):
            lin, nrm = getattr(m, f"enc_{i}"), getattr(m, f"enc_norm_{i}")
            x = torch.nn.functional.leaky_relu(x @ lin.weight.double().t() + lin.bias.double(), SLOPE)
            x = (x - x.mean(1, keepdim=True)) / torch.sqrt(((x - x.mean(1, keepdim=True)) ** 2).mean(1, keepdim=True) + EPS)
            x = x * nrm.weight.double() + nrm.bias.double()
        # three layers of at most 198 terms and two norms in fp32: 1e-5 of the output's scale is 160 u
        for got, head in ((mu, m.encmu), (lv, m.enclogvar)):
            want = x @ head.weight.double().t() + head.bias.double()
            assert float((got.double() - want).abs().max()) <= 1e-5 * float(want.abs().max())
        buf = io.BytesIO()
        torch.save(m, buf)
        buf.seek(0)
        m2 = torch.load(buf, weights_only=False)   # a file this test wrote
        assert m2.layer_norm and torch.equal(m2.sample_encoding(s, r, u)[0], mu)
    assert set(make("pivotcvae_gt_pi").state_dict()) == {k for k in m.state_dict() if "_norm_" not in k}
