"""Teachers at the edges of ``distill_loss``: rows that a mask leaves nothing of. Against float64 on the CPU
(``oracle.logits_ref``)."""

from __future__ import annotations

import pytest
import torch

import rwkv_tl_amd  # noqa: F401
from oracle import logits_ref as R
from rwkv_tl_amd import kernels as K

pytestmark = pytest.mark.gpu
U = 2.0**-24  # half a step of float32
INF = float("inf")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("V,k", [(40, 5), (8, 8), (9001, 256)])
def test_a_teacher_row_that_a_mask_leaves_nothing_of(cuda, dtype, V, k):
    """top_logits gives it k ids, values of -inf and an lse of -inf: no mass, loss 0 and gradient 0."""
    g = torch.Generator().manual_seed(V)
    t = torch.randn(3, V, generator=g)
    t[1] = -INF
    t[2, 3:] = -INF
    z = torch.randn(3, V, generator=g).to(dtype)
    val, idx, lse = K.top_logits(t.to(cuda), k)
    assert lse[1] == -INF and bool((val[1] == -INF).all())
    loss, grad = K.distill_loss_grad(z.to(cuda), val, idx, lse)
    assert torch.equal(K.distill_loss(z.to(cuda), val, idx, lse), loss)
    assert torch.equal(K.distill_loss_backward(torch.ones(3, device=cuda), z.to(cuda), val, idx, lse, 1.0), grad)
    want = R.distill_loss(z.double(), val.cpu(), idx.cpu(), lse.cpu())
    assert loss[1] == 0 and bool((grad[1] == 0).all())
    # (half steps of P < 1 logarithms of the row and two of its rest, 56 each)
    assert bool(((loss.cpu() - want).abs() <= 112 * U + U * want.abs()).all())
    # whatever the row's logits hold, as in a row without an entry
    z[1] = float("nan")
    again = K.distill_loss_grad(z.to(cuda), val, idx, lse)
    assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    # a finite entry beside an lse of -inf is no distribution
    val[1, 0] = 0.0
    assert K.distill_loss(torch.zeros(3, V, device=cuda), val, idx, lse)[1].isnan()
