"""``torch.ops.rwkv_tl.layer_norm_forward``, which has no gradient, says so in a backward pass that reaches it."""

from __future__ import annotations

import pytest
import torch

import rwkv_tl_amd  # noqa: F401

ops = torch.ops.rwkv_tl


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("leaf", [0, 1, 2])
def test_layer_norm_forward_has_no_gradient(which, leaf):
    args = [torch.empty(*s, device="meta") for s in ((6, 8), (8,), (8,))]
    args[leaf].requires_grad_()
    out = ops.layer_norm_forward(*args)[which]
    with pytest.raises(NotImplementedError, match="layer_norm is the differentiable form"):
        out.sum().backward()
    with torch.no_grad():
        assert not ops.layer_norm_forward(*args)[which].requires_grad
