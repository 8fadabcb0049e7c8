"""-m gpu: layer norm and 8-bit activation checkpoints at the ends of their ranges: magnitudes, heights past a launch's rows, launch plans and
offsets that tests/test_hip_norm_act8.py does not reach.  Bounds: tests/norm_act8_ref.py."""
import pytest
import torch

from tests.gpu_util import DEV
from tests.norm_act8_ref import SLOPE, TYPES, U, Norm64, inside, kept64, weight_grad
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


# ---- more rows than a launch holds at once ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,D,t", [(1100, 4097, torch.float32), (1100, 5397, torch.float32), (300, 8200, torch.float32), (1100, 16384, torch.float32),
                                   (1100, 5397, torch.bfloat16), (1100, 8192, torch.float16), (300, 8200, torch.bfloat16), (1100, 16384, torch.float16),
                                   (140001, 3, torch.float32), (140001, 30, torch.float32), (140001, 64, torch.bfloat16), (70003, 61, torch.float16)], ids=str)
def test_layer_norm_walks_over_its_rows(M, D, t):
    """workgroups that take several rows (1024 threads a row: over 1024 forward, over 256 backward) or several groups of rows (8 to 16 lanes a row:
    over 131072 / 65536 forward, over 24576 / 12288 backward), from the rows and from their 8-bit form"""
    x, g = rand((M, D), D + 3, t).to(DEV), rand((M, D), D + 4, t, 0.1, leaky=False).to(DEV)
    w, b = (p.to(DEV) for p in params(D, D))
    y, mean, rstd, kept = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    ref = Norm64(x, w, b, EPS)
    inside(y, ref.y, ref.y_bound(t), "y")
    inside(mean, ref.mean[:, 0], ref.d_mean[:, 0], "mean")
    inside(rstd, ref.rstd[:, 0], (ref.d_rstd * ref.rstd)[:, 0], "rstd")
    assert torch.equal(ops().layer_norm_fwd_raw(x, w, b, EPS)[0], y)
    q = kept64(x)
    assert torch.equal(kept.unpack(torch.float32).double().cpu(), q)
    for src, arg in ((None, x), (q, kept)):
        ref.backward(g, src, leaky=True)
        dx, dw, db = ops().layer_norm_bwd_raw(g, arg, w, mean, rstd, leaky=True)
        inside(dx, ref.dx, ref.dx_bound(t), "dx")
        inside(dw, ref.dw, ref.d_dw, "dweight")
        inside(db, ref.db, ref.d_db, "dbias")


@pytest.mark.parametrize("M,D,t", [(7001, 1419, torch.float32), (25001, 1419, torch.bfloat16), (70001, 300, torch.float16)], ids=str)
def test_rows_kernels_walk_over_their_rows(M, D, t):
    """over 2^21 pieces of 16 bytes: lanes of pack, unpack and LeakyReLU' take several, in rows that end inside a piece"""
    assert M * (-(-D // 32) * 32 // (4 if t == torch.float32 else 8)) > 8192 * 256
    x, g = rand((M, D), D + 3, t).to(DEV), rand((M, D), D + 4, t, 0.1, leaky=False).to(DEV)
    ck = ops().act8_pack(x)
    q = kept64(x)
    assert torch.equal(ck.unpack(torch.float32).double().cpu(), q) and torch.equal(ck.unpack().cpu(), q.float().to(t))
    want = torch.where(x > 0, g.float(), SLOPE * g.float()).to(t)
    assert torch.equal(ops().act8_leaky_bwd_(g, ck), want)


# ---- weight gradient: the launch plans ----------------------------------------------------------------------------------------------------
def _weight_case(M, N, K, t, normed, seed=11):
    x, g = rand((M, K), seed, torch.float32, 2.0).to(DEV), rand((M, N), seed + 1, t, 0.1, leaky=False).to(DEV)
    norm = None
    if normed:
        _, mean, rstd, _ = ops().layer_norm_fwd_raw(x)
        norm = (mean, rstd, *(p.to(DEV) for p in params(K, K)))
    return g, ops().act8_pack(x), norm, weight_grad(g, kept64(x), norm)


def _weight_check(g, ck, norm, ref, K):
    want, bound, wdb, bdb = ref
    N = g.shape[1]
    dW, db = ops().act8_bwd_weight_raw(g, ck, norm=norm)
    inside(dW, want, bound, "dW")
    inside(db, wdb, bdb, "db")
    wide, b2 = torch.full((N, K + 5), 0.5, device=DEV), torch.full((N,), 0.25, device=DEV)
    ops().act8_bwd_weight_raw(g, ck, wide[:, 2:2 + K], b2, norm=norm)
    assert torch.equal(wide[:, 2:2 + K], 0.5 + dW) and torch.equal(b2, 0.25 + db)
    assert bool((wide[:, :2] == 0.5).all()) and bool((wide[:, 2 + K:] == 0.5).all())


def _ranges(M, N, K, tile):
    """ranges of rows that a call takes with tiles of 128 x `tile`, from the workspace it asks for (none: one)"""
    from pivotcvae_amd import _hip
    nn, n = -(-N // 128), _hip.lib().pcvae_act8_bwd_weight_ws_bytes(M, N, K) // 4
    per = nn * -(-K // tile) * 128 * tile + nn * 128
    assert n % per == 0
    return max(1, n // per)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("M,N,K", [(100, 4095, 4001), (131, 4096, 4000), (128, 8191, 2047)])
def test_weight_gradient_in_wide_tiles_of_one_range(M, N, K, normed, t):
    """512 tiles of 128 x 256: one range of rows, products stored (and accumulated) without a join, columns that end inside a lane's four"""
    assert -(-N // 128) * -(-K // 256) * -(-M // 32) >= 2048 and _ranges(M, N, K, 256) == 1
    _weight_check(*_weight_case(M, N, K, t, normed), K)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,N,K,tile,normed", [(8197, 300, 520, 256, False), (8200, 301, 519, 256, True), (1200, 1300, 1100, 256, False), (5000, 40, 700, 128, True)])
def test_weight_gradient_accumulates_over_its_join(M, N, K, tile, normed, t):
    assert _ranges(M, N, K, tile) > 1
    _weight_check(*_weight_case(M, N, K, t, normed), K)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M,N,K", [(70000, 1, 200), (5001, 1, 33), (20000, 2, 16), (65553, 8, 16), (65553, 129, 257), (3000, 1, 1)])
def test_weight_gradient_of_narrow_layers_over_long_batches(M, N, K, t):
    """heads and single columns: one or two tiles, as many ranges of rows as the plan gives"""
    _weight_check(*_weight_case(M, N, K, t, False), K)


# ---- offsets --------------------------------------------------------------------------------------------------------------------------------
def test_codes_and_scales_behind_offsets_over_32_bits():
    """the C entry points with code rows 2 MiB and groups of scales 16 MiB apart: both reach past 2^32 bytes, what lies between stays"""
    from pivotcvae_amd import _hip
    L, M, D, N, ldc, lds = _hip.lib(), 2100, 40, 24, 1 << 21, 1 << 24
    groups = -(-M // 8)
    x, g, gz = rand((M, D), 3).to(DEV), rand((M, D), 4, leaky=False).to(DEV), rand((M, N), 5, leaky=False).to(DEV)
    w, b = (p.to(DEV) for p in params(D, 1))
    codes = torch.full((M * ldc,), 0x55, dtype=torch.uint8, device=DEV)
    scales = torch.full((groups * lds,), 0x55, dtype=torch.uint8, device=DEV)
    assert (M - 1) * ldc > 1 << 32 and (groups - 1) * lds > 1 << 32
    far = (codes.data_ptr(), ldc, scales.data_ptr(), lds)
    near = ops().act8_pack(x)

    def held():   # the rows' codes and scale bytes are the packed ones, the bytes behind them untouched
        c, s = codes.view(M, ldc), scales.view(groups, lds)
        rows = [v.view(groups, -1, 8).transpose(1, 2).reshape(groups * 8, -1)[:M] for v in (s[:, :16].contiguous(), near.scales)]
        return torch.equal(c[:, :64], near.codes) and torch.equal(*rows) and bool((c[:, 64:128] == 0x55).all()) and bool((s[:, 16:32] == 0x55).all())

    st = _hip.stream()
    _hip.check(L.pcvae_act8_pack(x.data_ptr(), D, 0, M, D, *far, st))
    assert held()
    y = torch.empty_like(x)
    _hip.check(L.pcvae_act8_unpack(*far, M, D, y.data_ptr(), D, 0, st))
    assert torch.equal(y, near.unpack())
    ga, gb = g.clone(), g.clone()
    _hip.check(L.pcvae_act8_leaky_bwd(ga.data_ptr(), D, 0, *far, M, D, st))
    assert torch.equal(ga, ops().act8_leaky_bwd_(gb, near))
    codes.fill_(0x55)
    scales.fill_(0x55)
    want = ops().layer_norm_fwd_raw(x, w, b, EPS, checkpoint="e4m3")
    mean, rstd = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    _hip.check(L.pcvae_layer_norm_fwd(x.data_ptr(), D, 0, M, D, w.data_ptr(), b.data_ptr(), EPS, y.data_ptr(), D, mean.data_ptr(), rstd.data_ptr(), *far, st))
    assert held() and torch.equal(y, want[0])
    wb = ops().layer_norm_bwd_raw(g, near, w, mean, rstd, leaky=True)
    n = L.pcvae_layer_norm_bwd_ws_bytes(M, D, 0)
    ws, dw, db = torch.empty(n, dtype=torch.uint8, device=DEV), torch.empty(D, device=DEV), torch.empty(D, device=DEV)
    _hip.check(L.pcvae_layer_norm_bwd(g.data_ptr(), D, 0, M, D, None, 0, *far, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), 1, y.data_ptr(), D,
                                      dw.data_ptr(), db.data_ptr(), 0, ws.data_ptr(), n, st))
    assert all(torch.equal(a, c) for a, c in zip((y, dw, db), wb))
    ww = ops().act8_bwd_weight_raw(gz, near, norm=(mean, rstd, w, b))
    n = L.pcvae_act8_bwd_weight_ws_bytes(M, N, D)
    ws, dW, dz = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV), torch.empty(N, D, device=DEV), torch.empty(N, device=DEV)
    _hip.check(L.pcvae_act8_bwd_weight(gz.data_ptr(), N, 0, *far, M, N, D, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), b.data_ptr(), dW.data_ptr(), D,
                                       dz.data_ptr(), 0, ws.data_ptr(), n, st))
    assert torch.equal(dW, ww[0]) and torch.equal(dz, ww[1])


# ---- the largest fp16 values ------------------------------------------------------------------------------------------------------------------
def test_finite_fp16_rows_come_back_finite():
    """65504 is nearest to 65536 among its scale's multiples, an infinity in fp16: fp16 rows are held at 61440 (2^-4 of their value off at
    most, as every code), alone and from the norm's pass; infinities stay NaN"""
    top = torch.arange(0x7a00, 0x7c00, dtype=torch.int16).view(torch.float16)     # 49152 .. 65504
    x = torch.cat([top, -top, rand((1024,), 1, torch.float16), torch.full((32,), 65504.0).half()]).view(-1, 32)
    want = kept64(x.clamp(-61440, 61440))
    ck = ops().act8_pack(x.to(DEV))
    got = ck.unpack().cpu()
    assert got.dtype == torch.float16 and bool(got.isfinite().all()) and torch.equal(got.double(), want)
    assert bool(((got.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -13).all())   # (ordinary rows: blocks below 8)
    assert torch.equal(ops().layer_norm_fwd_raw(x.to(DEV), checkpoint="e4m3")[3].codes, ck.codes)
    assert torch.equal(ops().act8_pack(x.float().to(DEV)).unpack(torch.float32).double().cpu(), kept64(x.float()))   # fp32 rows: as they were
    x[0, 5] = float("inf")
    got = ops().act8_pack(x.to(DEV)).unpack().cpu()
    assert bool(got[0, 5].isnan()) and int(got.isnan().sum()) == 1 and not bool(got.isinf().any())


# ---- shared parameters ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("normed,checkpoint", [(False, None), (True, None), (False, "e4m3"), (True, "e4m3")])
def test_tied_layers_accumulate_into_their_one_gradient(normed, checkpoint):
    """three layers (and two norms) that are the same parameters, gradients accumulated in place: the sum of what each layer gives on its
    own.  Per layer and norm one fp32 addition to what is there (zero, exactly, at first): three layers agree to 2 u of the parts'
    magnitudes per addition, two norms to 2 u in all"""
    W, M = 192, 3000
    w = (rand((W, W), 1, leaky=False) / W ** 0.5).to(DEV)
    x, t = rand((M, W), 3, leaky=False).to(DEV), rand((M, W), 4, leaky=False).to(DEV)
    grads = []
    for tied in (True, False):
        layers = [(w.clone().requires_grad_(), torch.zeros(W, device=DEV).requires_grad_()) for _ in range(1 if tied else 3)]
        norms = [tuple(p.to(DEV).requires_grad_() for p in params(W, 5)) for _ in range(1 if tied else 2)] if normed else None
        for p in [q for pair in layers + (norms or []) for q in pair]:
            p.grad = torch.zeros_like(p)
        each = 3 // len(layers)
        (ops().mlp(x, layers * each, True, norms=norms and norms * (2 // len(norms)), checkpoint=checkpoint) * t).sum().backward()
        grads.append([[p.grad for p in pair] for pair in layers + (norms or [])])
    tied, single = grads
    for k in range(2):
        parts = [single[i][k].double() for i in range(3)]
        assert bool(((tied[0][k].double() - sum(parts)).abs() <= 4 * U * sum(p.abs() for p in parts)).all())
        if normed:
            parts = [single[3 + i][k].double() for i in range(2)]
            assert bool(((tied[1][k].double() - sum(parts)).abs() <= 2 * U * sum(p.abs() for p in parts)).all())


# ---- gradients cleared between the passes -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("how", ["to none", "to zero", "replaced"])
@pytest.mark.parametrize("stack", ["mlp", "mlp normed", "mlp kept", "mlp both", "heads", "heads both", "into"])
def test_gradients_cleared_after_the_forward_pass_arrive_all_the_same(stack, how):
    """output = f(x); optimizer.zero_grad(); output.backward(): the gradient goes to where the parameter holds it by then"""
    o, W, M = ops(), 48, 70
    layers = [((rand((W, W), i, leaky=False) / W ** 0.5).to(DEV).requires_grad_(), torch.zeros(W, device=DEV).requires_grad_()) for i in range(4)]
    norms = [tuple(p.to(DEV).requires_grad_() for p in params(W, 5 + i)) for i in range(2)]
    x, t = rand((M, W), 3, leaky=False).to(DEV), rand((M, W), 4, leaky=False).to(DEV)
    kw = dict(norms=norms if stack.endswith(("normed", "both")) else None, checkpoint="e4m3" if stack.endswith(("kept", "both")) else None)
    if stack.startswith("mlp"):
        f, used = lambda: o.mlp(x, layers[:3], True, **kw), layers[:3]
    elif stack.startswith("heads"):
        f, used = lambda: sum(o.mlp_heads(x, layers[:2], layers[2], layers[3], **kw)), layers
    else:
        f, used = lambda: o.mlp_into(x, layers[:2], torch.zeros(M, W + 8, device=DEV), 8)[:, 8:], layers[:2]
    leaves = [p for pair in used + (norms if kw["norms"] else []) for p in pair]
    (f() * t).sum().backward()
    want = [p.grad.clone() for p in leaves]      # into parameters that held no gradient
    assert all(bool(g.any()) for g in want)
    out = (f() * t).sum()                        # ... and now they do
    old = [p.grad for p in leaves]
    for p in leaves:
        if how == "to zero":
            p.grad.zero_()
        else:
            p.grad = None if how == "to none" else torch.zeros_like(p)
    before = [g.clone() for g in old]
    out.backward()
    assert all(p.grad is not None and torch.equal(p.grad, g) for p, g in zip(leaves, want))
    assert all((p.grad is g) == (how == "to zero") for p, g in zip(leaves, old))
    assert how == "to zero" or all(torch.equal(g, b) for g, b in zip(old, before))       # buffers let go of are left alone
