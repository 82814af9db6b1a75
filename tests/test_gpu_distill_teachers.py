"""Teachers at the edges of ``distill_loss``: rows that a mask leaves nothing of, and log-sum-exps far from 0, against
float64 on the CPU (``oracle.logits_ref``)."""

from __future__ import annotations

import math

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


@pytest.mark.parametrize("other", [float("nan"), INF])
def test_a_teacher_row_of_a_nan_or_an_infinity(cuda, other):
    """top_logits gives it an lse of NaN; its entries may all be -inf (NaN comes behind them)."""
    t = torch.full((2, 300), -INF)
    t[0], t[1, 250] = torch.randn(300, generator=torch.Generator().manual_seed(1)), other
    val, idx, lse = K.top_logits(t.to(cuda), 4)
    assert bool(lse[1].isnan())
    for z in (torch.zeros(2, 300, dtype=torch.float16), torch.randn(2, 300, generator=torch.Generator().manual_seed(2))):
        loss, grad = K.distill_loss_grad(z.to(cuda), val, idx, lse)
        assert torch.equal(K.distill_loss(z.to(cuda), val, idx, lse).isnan(), loss.isnan())
        assert loss.isnan().tolist() == [False, True] and bool(grad[1].isnan().all()) and bool(grad[0].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("T", [1.0, 0.7, 3.0, 1e-20])
@pytest.mark.parametrize("V,k", [(1, 1), (40, 5), (3001, 130)])
def test_a_teacher_row_of_the_lowest_value(cuda, dtype, T, V, k):
    """Without an lse: the softmax of equal entries, however far from 0 they lie."""
    g = torch.Generator().manual_seed(V)
    t = torch.full((2, V), torch.finfo(dtype).min)
    t[1] *= -1.0
    z = (T * torch.randn(2, V, generator=g)).float()
    val, idx, _ = K.top_logits(t.to(dtype).to(cuda), k)
    loss, grad = (x.double().cpu() for x in K.distill_loss_grad(z.to(cuda), val, idx, temperature=T))
    y = torch.log_softmax(z.double() / T, -1)
    want = -math.log(k) - y[:, :k].mean(-1)
    assert bool(((loss - want).abs() <= 112 * U + U * want.abs()).all())
    ref = y.exp()
    size = ref.clone()
    ref[:, :k] -= 1 / k
    size[:, :k] += 1 / k
    assert bool(((grad * T - ref).abs() <= (60 + 3 * 20) * U * size + U * ref.abs() + 2.0**-125 * max(T, 1.0)).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("T", [1.0, 0.7, 1.5, 3.0, 50.0])
def test_a_teacher_row_of_the_lowest_value_with_its_lse(cuda, dtype, T):
    """float16's (-65504) has a log-sum-exp that tells its distribution; bfloat16's and float32's, whose half step is 1e30,
    have not, and such a row has no teacher."""
    g = torch.Generator().manual_seed(5)
    V, k = 50, 7
    t = torch.randn(3, V, generator=g)
    t[1] = torch.finfo(dtype).min
    val, idx, lse = K.top_logits(t.to(dtype).to(cuda), k, temperature=T)
    z = torch.randn(3, V, generator=g)
    loss, grad = K.distill_loss_grad(z.to(cuda), val, idx, lse, temperature=T)
    want = R.distill_loss(z.double(), val.cpu(), idx.cpu(), lse.cpu(), T)
    assert bool(((loss.cpu() - want).abs() <= 112 * U + U * want.abs()).all()) and bool(grad.isfinite().all())
    assert (float(loss[1]) == 0 and bool((grad[1] == 0).all())) == (dtype != torch.float16)
    assert bool((grad[0] != 0).all()) and bool((grad[2] != 0).all())


@pytest.mark.parametrize("at", [100.0, -100.0, 200.3, -1000.7, 60000.0])
def test_a_rounded_log_sum_exp_leaves_no_mass(cuda, at):
    """Teachers whose listed logits are all of their mass, far from 0: what rounding their lse to float32 takes from 1 is
    no rest, however little the student has outside the ids."""
    g = torch.Generator().manual_seed(int(abs(at)))
    N, V, k = 64, 500, 12
    t = (torch.randn(N, k, generator=g) + at).float()
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(N)])
    lse = torch.logsumexp(t.double(), -1)
    lse32 = lse.float()
    assert bool((lse32.double() > lse).any())  # of which P < 1
    z = torch.full((N, V), -80.0)
    z.scatter_(1, idx, torch.randn(N, k, generator=g))
    loss, grad = (x.double().cpu() for x in K.distill_loss_grad(z.to(cuda), t.to(cuda), idx.to(cuda), lse32.to(cuda)))
    p = (t.double() - lse32.double()[:, None]).exp()  # the teacher that the stored lse gives, without a rest
    y = torch.log_softmax(z.double(), -1)
    want = (p * (p.log() - y.gather(1, idx))).sum(-1)
    assert bool(((loss - want).abs() <= 112 * U + U * want.abs()).all())
    ref = (y.exp() * p.sum(-1, keepdim=True)).scatter_add(1, idx, -p)
    # 60 half steps of each term, and 3 of the exponent's size (up to 85)
    size = (y.exp() * p.sum(-1, keepdim=True)).scatter_add(1, idx, p)
    assert bool(((grad - ref).abs() <= (60 + 3 * 90) * U * size + U * ref.abs() + 2.0**-125).all())
    assert torch.allclose(R.distill_loss(z.double(), t, idx, lse32), want, rtol=0, atol=1e-9)


def test_a_rest_just_above_half_a_step_counts(cuda):
    """A teacher's mass outside its ids of twice the cut is held against the student's."""
    z = torch.tensor([[0.0, 0.0, -3.0, -4.0]]).repeat(2, 1)
    val, idx = torch.tensor([[200.0], [10.0]]), torch.zeros(2, 1, dtype=torch.int64)
    lse = torch.tensor([200.0 + 2.0**-16, 10.0 + 2.0**-19])  # half steps of 2^-17 and 2^-21
    want = R.distill_loss(z.double(), val, idx, lse)
    q = torch.softmax(z[0].double(), -1)
    for r in range(2):
        p = math.exp(float(val[r, 0]) - float(lse[r]))
        by_hand = p * math.log(p / float(q[0])) + (1 - p) * math.log((1 - p) / float(q[1:].sum()))
        assert abs(by_hand - float(want[r])) < 1e-10
    loss = K.distill_loss(z.to(cuda), val.to(cuda), idx.to(cuda), lse.to(cuda)).double().cpu()
    assert bool(((loss - want).abs() <= 112 * U + U * want.abs()).all())
    # (without it the first loss would be 1.5e-4 more; the tolerance is 6.7e-6)
    assert abs(float(want[0]) + math.log(float(q[0]))) > 1e-4
