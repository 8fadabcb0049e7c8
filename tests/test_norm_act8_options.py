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
