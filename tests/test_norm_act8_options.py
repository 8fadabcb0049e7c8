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
