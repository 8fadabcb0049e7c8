"""CPU: what the layer norm and the stacks ask of their kernels (recorded in place of the launches)."""
import pytest
import torch

from pivotcvae_amd import ops


@pytest.fixture
def asked(monkeypatch):
    """checkpoint arguments of the forward launches, in order"""
    seen = []

    def record(x, weight=None, bias=None, eps=1e-5, checkpoint=None):
        seen.append(checkpoint)
        ck = ops.Act8.empty(x.shape, x.dtype, x.device) if checkpoint else None
        return x.clone(), x.new_zeros(x.shape[0]), x.new_ones(x.shape[0]), ck

    monkeypatch.setattr(ops, "layer_norm_fwd_raw", record)
    return seen


def test_layer_norm_keeps_its_rows_for_a_backward_pass_alone(asked):
    x, w, b = torch.ones(4, 8), torch.ones(8), torch.zeros(8)
    ops.layer_norm(x, w, b, checkpoint="e4m3")                          # nothing wants a gradient
    with torch.no_grad():
        ops.layer_norm(x.requires_grad_(), w, b, checkpoint="e4m3")
    assert asked == [None, None]
    ops.layer_norm(x, w, b, checkpoint="e4m3")
    ops.layer_norm(x.detach(), w.requires_grad_(), None, checkpoint="e4m3")
    ops.layer_norm(x.detach(), None, b.requires_grad_(), checkpoint="e4m3")
    assert asked[2:] == ["e4m3"] * 3
    with pytest.raises(ValueError, match="checkpoint"):
        with torch.no_grad():
            ops.layer_norm(x, checkpoint="int4")


def test_one_launch_never_accumulates_twice_into_a_buffer(monkeypatch):
    """layers that share a parameter share its gradient buffer: their weight gradients are read-modify-write and go into launches that follow
    each other; others stay in one launch"""
    launches = []

    class Lib:
        def pcvae_linear_group_ws_bytes(self, arr, n):
            return 0

        def pcvae_linear_group(self, arr, n, ws, nbytes, stream):
            launches.append([(d.c, d.aux_out) for d in arr])
            return 0

    monkeypatch.setattr(ops, "lib", lambda: Lib())
    monkeypatch.setattr(ops, "stream", lambda: None)
    monkeypatch.setattr(ops, "ptr", lambda *a: None)
    x, g = torch.ones(4, 8), torch.ones(4, 8)
    W = [torch.zeros(8, 8) for _ in range(3)]
    b = [torch.zeros(8) for _ in range(3)]
    grp = ops.GemmGroup()
    for k, j in ((0, 0), (1, 1), (0, 0), (2, 1), (2, 2)):   # a tied layer; one that shares a bias alone; one that shares a weight alone
        grp.dw(g, x, W[k], b[j])
    grp.launch()
    got = [[(c, d) for c, d in part] for part in launches]
    at = lambda k, j: (W[k].data_ptr(), b[j].data_ptr())   # noqa: E731
    assert got == [[at(0, 0), at(1, 1)], [at(0, 0), at(2, 1)], [at(2, 2)]]


@pytest.mark.parametrize("call", ["mlp", "mlp normed", "mlp kept", "heads", "heads kept", "relu", "into"])
@pytest.mark.parametrize("W,b,err,say", [(torch.zeros(8, 16)[:, ::2], torch.zeros(8), ValueError, "contiguous rows"), (torch.zeros(8, 8).t(), torch.zeros(8), ValueError, "contiguous rows"),
                                         (torch.zeros(8, 8), torch.zeros(16)[::2], ValueError, "contiguous"), (torch.zeros(8, 8), torch.zeros(1).expand(8), ValueError, "contiguous"),
                                         (torch.zeros(8, 8), torch.zeros(7), RuntimeError, "shape"), (torch.zeros(8, 8), torch.zeros(8, 1), RuntimeError, "shape"),
                                         (torch.zeros(8), torch.zeros(8), RuntimeError, "shape")])
def test_stacks_refuse_layers_that_the_kernels_would_misread(call, W, b, err, say):
    """the kernels read weights by rows of unit column stride and one bias per row: anything else is refused before a launch"""
    x, ok = torch.zeros(4, 8), (torch.zeros(8, 8), torch.zeros(8))
    norm = [(torch.ones(8), torch.zeros(8))]
    with pytest.raises(err, match=say):
        {"mlp": lambda: ops.mlp(x, [ok, (W, b)], True),
         "mlp normed": lambda: ops.mlp(x, [(W, b), ok], True, norms=norm),
         "mlp kept": lambda: ops.mlp(x, [ok, (W, b)], True, checkpoint="e4m3"),
         "heads": lambda: ops.mlp_heads(x, [ok], ok, (W, b)),
         "heads kept": lambda: ops.mlp_heads(x, [(W, b)], ok, ok, checkpoint="e4m3"),
         "relu": lambda: ops.mlp_relu(x, [ok, (W, b)]),
         "into": lambda: ops.mlp_into(x, [(W, b)], torch.zeros(4, 16), 8)}[call]()
