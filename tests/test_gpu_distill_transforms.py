"""``torch.ops.rwkv_tl.distill_loss`` under autograd's batching, vmap and checkpointing, the same bits as the kernels called
row by row; and a teacher that requires gradients."""

from __future__ import annotations

import pytest
import torch

import rwkv_tl_amd  # noqa: F401
from rwkv_tl_amd import kernels as K

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:There is a performance drop")]
ops = torch.ops.rwkv_tl


@pytest.fixture
def case(cuda):
    g = torch.Generator().manual_seed(3)
    z, t = torch.randn(4, 1003, generator=g), 3.0 * torch.randn(4, 1003, generator=g)
    val, idx = t.topk(20)
    return tuple(x.to(cuda) for x in (z, val, idx, torch.logsumexp(t / 1.5, -1)))


def _loss(case):
    return lambda x: ops.distill_loss(x, *case[1:], 1.5)


def test_batched_gradients(case):
    """Several gradients of one loss in a call, and what calls that: the rows of the Jacobian."""
    grad = K.distill_loss_grad(*case, temperature=1.5)[1]
    want = torch.zeros(4, 4, 1003, device=grad.device)
    want[torch.arange(4), torch.arange(4)] = grad
    x = case[0].clone().requires_grad_()
    (got,) = torch.autograd.grad(_loss(case)(x), x, torch.eye(4, device=x.device), is_grads_batched=True)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.functional.jacobian(_loss(case), case[0], vectorize=True), want)


def test_vmap(case):
    one = lambda x, v, i, s: ops.distill_loss(x, v, i, s, 1.5)  # noqa: E731
    loss = K.distill_loss(*case, temperature=1.5)
    assert torch.equal(torch.func.vmap(one)(*case), loss)
    assert torch.equal(torch.func.vmap(one, in_dims=(None, 0, 0, 0))(case[0][0], *case[1:]),
                       K.distill_loss(case[0][:1].expand(4, -1), *case[1:], temperature=1.5))


def test_checkpointing(case):
    x = case[0].clone().requires_grad_()
    torch.utils.checkpoint.checkpoint(_loss(case), x, use_reentrant=False).sum().backward()
    assert torch.equal(x.grad, K.distill_loss_grad(*case, temperature=1.5)[1])


def test_transforms_without_a_rule_are_refused(case):
    z = case[0]
    with pytest.raises(RuntimeError, match="setup_context"):  # torch's own refusal, as of its registered operators
        torch.func.grad(lambda x: _loss(case)(x).sum())(z)
    with pytest.raises(NotImplementedError, match="jvp"), torch.autograd.forward_ad.dual_level():
        _loss(case)(torch.autograd.forward_ad.make_dual(z, z))


def test_a_teacher_that_requires_gradients_without_grad_mode(cuda):
    """Evaluation inside no_grad of a teacher whose tensors are part of a graph: nothing asks for their gradient."""
    z = torch.randn(3, 100, generator=torch.Generator().manual_seed(4)).to(cuda)
    t = torch.randn(3, 100, generator=torch.Generator().manual_seed(5)).to(cuda).requires_grad_()
    val, idx = t.topk(7)
    lse = torch.logsumexp(t, -1)
    want = K.distill_loss(z, val.detach(), idx, lse.detach())
    for x in (z, z.clone().requires_grad_()):
        with torch.no_grad():
            assert torch.equal(ops.distill_loss(x, val, idx, lse), want)
        with pytest.raises(ValueError, match="no gradient to the teacher"):
            ops.distill_loss(x, val, idx, lse)
