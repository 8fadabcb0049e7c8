"""CPU: what the layer norm and the 8-bit checkpoints refuse, before any launch - and the 64-bit restatement of the 8-bit rows itself."""
import pytest
import torch

from pivotcvae_amd import _hip, ops
from tests.norm_act8_ref import kept64

P = 1 << 12   # a pointer no call here reaches


def text():
    return _hip.lib().pcvae_last_error().decode()


def fwd(**kw):
    a = dict(x=P, ldx=64, type=0, M=4, D=64, w=None, b=None, eps=1e-5, y=P, ldy=64, mean=None, rstd=None, codes=None, ldc=0, scales=None, lds=0)
    a.update(kw)
    return _hip.lib().pcvae_layer_norm_fwd(*a.values(), None)


def bwd(**kw):
    a = dict(g=P, ldg=64, type=0, M=4, D=64, x=P, ldx=64, codes=None, ldc=0, scales=None, lds=0, w=None, mean=P, rstd=P, leaky=0, dx=P, lddx=64,
             dw=None, db=None, acc=0, ws=P, n=1 << 30)
    a.update(kw)
    return _hip.lib().pcvae_layer_norm_bwd(*a.values(), None)


@pytest.mark.parametrize("kw,say", [(dict(type=3), "type"), (dict(M=-1), "rows"), (dict(D=0), "width"), (dict(D=16385, ldx=16385), "width"),
                                    (dict(x=None), "null"), (dict(y=None), "null"), (dict(ldx=63), "stride"), (dict(ldy=63), "stride"),
                                    (dict(eps=-1.0), "eps"), (dict(codes=P), "together"), (dict(scales=P), "together"),
                                    (dict(codes=P, scales=P, ldc=32, lds=16), "codes"), (dict(codes=P + 8, scales=P, ldc=64, lds=16), "codes"),
                                    (dict(codes=P, scales=P + 4, ldc=64, lds=16), "scales"), (dict(codes=P, scales=P, ldc=64, lds=8), "scales"),
                                    (dict(codes=P, scales=P, ldc=72, lds=16), "codes")])
def test_layer_norm_forward_refuses(kw, say):
    assert fwd(**kw) == -1 and say in text()


@pytest.mark.parametrize("kw,say", [(dict(type=-1), "type"), (dict(D=0), "width"), (dict(g=None), "null"), (dict(dx=None), "null"), (dict(x=None), "either"),
                                    (dict(codes=P, scales=P, ldc=64, lds=16), "either"), (dict(mean=None), "mean"), (dict(rstd=None), "mean"),
                                    (dict(ldg=1), "stride"), (dict(lddx=8), "stride"), (dict(ldx=8), "stride")])
def test_layer_norm_backward_refuses(kw, say):
    assert bwd(**kw) == -1 and say in text()


def test_workspaces_are_checked():
    need = _hip.lib().pcvae_layer_norm_bwd_ws_bytes(4, 64, 0)
    assert need > 0 and bwd(n=need - 1) == -3 and bwd(ws=None) == -3 and "workspace" in text()
    assert _hip.lib().pcvae_layer_norm_bwd_ws_bytes(0, 64, 0) == 0 and _hip.lib().pcvae_layer_norm_bwd_ws_bytes(4, 0, 0) == 0
    need = _hip.lib().pcvae_act8_bwd_weight_ws_bytes(8192, 256, 1419)
    assert need > 0
    a = [P, 256, 0, P, 1440, P, 360, 8192, 256, 1419, None, None, None, None, P, 1419, P, 0]
    assert _hip.lib().pcvae_act8_bwd_weight(*a, P, need - 1, None) == -3 and "workspace" in text()
    assert _hip.lib().pcvae_act8_bwd_weight(*a, None, need, None) == -3


@pytest.mark.parametrize("at,value,say", [(2, 9, "type"), (0, None, "null"), (1, 255, "stride"), (3, None, "null"), (4, 1424, "codes"), (6, 352, "scales"),
                                          (8, 0, "N"), (9, 0, "width"), (10, P, "together"), (12, P, "mean"), (14, None, "dW"), (15, 1418, "stride"),
                                          (7, -1, "rows")])
def test_weight_gradient_refuses(at, value, say):
    a = [P, 256, 0, P, 1440, P, 360, 8192, 256, 1419, None, None, None, None, P, 1419, P, 0]
    a[at] = value
    assert _hip.lib().pcvae_act8_bwd_weight(*a, P, 1 << 40, None) == -1 and say in text()


def test_rows_kernels_refuse():
    L = _hip.lib()
    assert L.pcvae_act8_pack(P, 64, 0, 4, 64, None, 64, P, 16, None) == -1 and "null" in text()
    assert L.pcvae_act8_pack(None, 64, 0, 4, 64, P, 64, P, 16, None) == -1
    assert L.pcvae_act8_pack(P, 60, 0, 4, 64, P, 64, P, 16, None) == -1 and "stride" in text()
    assert L.pcvae_act8_pack(P, 64, 7, 4, 64, P, 64, P, 16, None) == -1 and "type" in text()
    assert L.pcvae_act8_unpack(P, 32, P, 16, 4, 64, P, 64, 0, None) == -1 and "codes" in text()
    assert L.pcvae_act8_leaky_bwd(P, 3, 0, P, 64, P, 16, 4, 64, None) == -1 and "stride" in text()
    assert L.pcvae_act8_pack(None, 0, 0, 0, 64, None, 0, None, 0, None) == 0   # no rows: nothing to do


def test_python_layer_refuses():
    x = torch.zeros(4, 64)
    for call in (lambda: ops.layer_norm(x), lambda: ops.layer_norm_fwd_raw(x), lambda: ops.act8_pack(x), lambda: ops.mlp(x, [(x, x[0])], True, norms=[])):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()
    with pytest.raises(ValueError, match="checkpoint"):
        ops.layer_norm(x, checkpoint="int4")
    with pytest.raises(ValueError, match="checkpoint"):
        ops.mlp(x, [(x, x[0])], True, checkpoint="e5m2")
    with pytest.raises(RuntimeError, match="norms for"):
        ops.mlp(x, [(x, x[0])], True, norms=[(x[0], x[0])])
    with pytest.raises(ValueError, match="weight and a bias"):
        ops.mlp_heads(x, [(x, x[0])], (x, x[0]), (x, x[0]), norms=[(None, None)])
    u8 = torch.zeros(4, 64, dtype=torch.uint8)
    sc = torch.zeros(1, 16, dtype=torch.uint8)
    assert ops.Act8(u8, sc, (4, 64)).nbytes == 4 * 64 + 16 and ops.Act8(u8, sc, (2, 2, 50)).shape == (2, 2, 50)
    with pytest.raises(RuntimeError, match="do not hold"):
        ops.Act8(u8, sc, (4, 65))
    with pytest.raises(TypeError):
        ops.Act8(x, sc, (4, 64))
    with pytest.raises(ValueError, match="width"):
        ops.Act8(u8[:, :0], sc[:, :0], (4, 0))
    with pytest.raises(ValueError, match="contiguous"):
        ops.Act8(torch.zeros(4, 128, dtype=torch.uint8)[:, ::2], sc, (4, 64))


def test_models_validate_the_options():
    from pivotcvae_amd.models.cvae import BaseCVAE
    emb = torch.nn.Embedding(10, 8)
    m = BaseCVAE(emb, None, 5, 4, True, "cpu")
    assert m._stack_options("enc", 2) == {} and m.set_activation_checkpoint("e4m3") is m
    assert m._stack_options("enc", 2) == dict(norms=None, checkpoint="e4m3")
    with pytest.raises(ValueError, match="checkpoint"):
        m.set_activation_checkpoint("fp4")
    n = BaseCVAE(emb, None, 5, 4, True, "cpu", layer_norm=True)
    n._add_norms("enc", [8, 6, 7], 2)
    opts = n._stack_options("enc", 2)
    assert [tuple(w.shape) for w, _ in opts["norms"]] == [(6,), (7,)] and opts["checkpoint"] is None
    with pytest.raises(ValueError, match="layer norm over"):
        n._add_norms("big", [8, 20000], 1)


def test_restated_rows_against_the_type_itself():
    """the restatement rounds as torch's own float8_e4m3fn where the scale is 1, and holds its invariants elsewhere"""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 96, generator=g) * 40
    x[:, ::32] = 448.0     # pins the scale to 1
    q = kept64(x)
    want = x.to(torch.float8_e4m3fn).double()
    want = torch.where((x > 0) & (want == 0), torch.full_like(want, 2.0 ** -9), want)
    assert torch.equal(q, want)
    y = torch.randn(50, 100, generator=g) * torch.exp(3 * torch.randn(50, 1, generator=g))
    q = kept64(y)
    assert torch.equal(q > 0, y > 0)
    top = torch.nn.functional.pad(y.abs().double(), (0, 28)).view(50, 4, 32).amax(2, keepdim=True).expand(50, 4, 32).reshape(50, 128)[:, :100]
    err = (q - y.double()).abs()
    assert bool((err <= torch.maximum(2.0 ** -4 * y.abs().double(), top * 2.0 ** -9 * 2.0 ** -8 * 2)).all())
