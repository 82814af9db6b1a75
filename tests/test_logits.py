"""Operators between a large and a small model, on the CPU: the float64 oracle
against closed forms, refusals of the C entries and of the Python ones, Meta
shapes. (The kernels themselves: test_gpu_logits.py.)"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import rwkv_tl_amd
from oracle import logits_ref as R
from rwkv_tl_amd import _lib
from rwkv_tl_amd import kernels as K

ops = torch.ops.rwkv_tl


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------


def test_oracle_top_logits_order():
    x = torch.tensor([[0.0, 3.0, float("nan"), 3.0, -torch.inf, -0.0]])
    v, i, lse = R.top_logits(x, 6)
    assert i.tolist() == [[1, 3, 0, 5, 4, 2]]
    assert v[0, :5].tolist() == [3.0, 3.0, 0.0, -0.0, -torch.inf] and lse.isnan().all()


def test_oracle_loss_is_the_kl_when_every_token_is_listed():
    g = torch.Generator().manual_seed(0)
    z, t = torch.randn(4, 9, generator=g).double(), torch.randn(4, 9, generator=g).double()
    idx = torch.stack([torch.randperm(9, generator=g) for _ in range(4)])
    p, y = torch.softmax(t / 2, -1), torch.log_softmax(z / 2, -1)
    want = (p * (p.log() - y)).sum(-1)
    for lse in (None, torch.logsumexp(t / 2, -1)):
        got = R.distill_loss(z, t.gather(1, idx), idx, lse, 2.0)
        assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)


def test_oracle_loss_of_one_entry_is_cross_entropy_and_of_a_rest_two_bins():
    z = torch.tensor([[0.5, -1.0, 2.0, 0.0]]).double()
    y = torch.log_softmax(z, -1)[0]
    one = R.distill_loss(z, torch.tensor([[7.0]]), torch.tensor([[2]]), None)
    assert math.isclose(float(one), -float(y[2]), rel_tol=1e-12)
    p = 0.625  # the teacher's probability of token 2, by lse = 7 - log p
    two = R.distill_loss(z, torch.tensor([[7.0]]), torch.tensor([[2]]), torch.tensor([7.0 - math.log(p)], dtype=torch.float64))
    q = float(y[2].exp())
    assert math.isclose(float(two), p * math.log(p / q) + (1 - p) * math.log((1 - p) / (1 - q)), rel_tol=1e-9)


def test_oracle_gradient_matches_the_formula_and_differences():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(3, 12, generator=g).double().requires_grad_()
    t = torch.randn(3, 12, generator=g).double()
    val, idx = t.topk(4)
    lse = torch.logsumexp(t / 1.5, -1)
    (grad,) = torch.autograd.grad(R.distill_loss(z, val, idx, lse, 1.5).sum(), z)
    q = torch.softmax(z.detach() / 1.5, -1)
    p = (val / 1.5 - lse[:, None]).exp()
    inside = torch.zeros(3, 12, dtype=torch.bool).scatter_(1, idx, True)
    rest = 1 - p.sum(-1, keepdim=True)
    want = torch.where(inside, q, q * (1 - rest / q.masked_fill(inside, 0).sum(-1, keepdim=True)))
    want = want.scatter_add(1, idx, -p) / 1.5
    assert torch.allclose(grad, want, atol=1e-12)
    assert torch.autograd.gradcheck(lambda x: R.distill_loss(x, val, idx, lse, 1.5), z, eps=1e-6, atol=1e-7)


def test_oracle_verification_closed_forms():
    target = torch.tensor([[[0.0, 1.0, 2.0], [3.0, 0.0, 0.0], [0.0, 0.0, 5.0]]]).log()  # p: unnormalised weights
    tok = torch.tensor([[2, 1]])
    # p_0(2) = 2/3 accepted below it, p_1(1) = 0 rejected; the rest of row 1 is token 0
    out, n = R.verify_draft(target, tok, torch.tensor([[0.66, 0.0, 0.5]]), None, 1.0, 0.0)
    assert out.tolist() == [[2, 0, -1]] and n.tolist() == [1]
    out, n = R.verify_draft(target, tok, torch.tensor([[0.67, 0.0, 0.5]]), None, 1.0, 0.0)
    assert out.tolist() == [[1, -1, -1]] and n.tolist() == [0]
    out, n = R.verify_draft(target, torch.tensor([[2, 0]]), torch.tensor([[0.1, 0.9, 0.9]]), None, 1.0, 0.0)
    assert out.tolist() == [[2, 0, 2]] and n.tolist() == [2]
    out, n = R.verify_draft(target, torch.tensor([[2, 0]]), None, None, 0.0, 0.0, torch.tensor([1]))
    assert out.tolist() == [[2, 0, -1]] and n.tolist() == [1]


def test_oracle_verification_draws_the_targets_distribution():
    """Accepting and drawing again, integrated over a grid of both uniforms, gives p itself."""
    g = torch.Generator().manual_seed(2)
    V, n = 5, 60
    target, draft = torch.randn(1, 2, V, generator=g), torch.randn(1, 1, V, generator=g)
    p, q = torch.softmax(target[0, 0].double(), -1), torch.softmax(draft[0, 0].double(), -1)
    mass = torch.zeros(V, dtype=torch.float64)
    for x in range(V):
        for a in range(n):
            for u in range(n) if (a + 0.5) / n * q[x] >= p[x] else range(1):
                got, acc = R.verify_draft(target, torch.tensor([[x]]), torch.tensor([[(a + 0.5) / n, (u + 0.5) / n]]), draft, 1.0, 1.0)
                mass[got[0, 0]] += q[x] / n / (1 if int(acc) else n)
    # each of the two grids misplaces at most one cell of 1 / n per border
    assert (mass - p).abs().max() < 2.0 / n


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

_ONE = ctypes.c_char * 64


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    buf = _ONE()
    p = ctypes.addressof(buf)  # never read: every call is refused on the host
    EINVAL, ESHAPE, EWORKSPACE = 1, 2, 3

    def top(logits=p, dt=0, ld=16, N=1, V=16, k=4, T=1.0, val=p):
        return lib.rwkv7_top_logits(logits, dt, ld, N, V, k, T, val, p, p, None)

    assert top(logits=None) == EINVAL and top(val=None) == EINVAL and top(dt=3) == EINVAL and top(dt=-1) == EINVAL
    for T in (0.0, -1.0, math.nan, math.inf):
        assert top(T=T) == EINVAL
    assert top(N=0) == top(V=0) == top(V=65537, ld=65537) == top(ld=15) == top(k=0) == top(k=17) == ESHAPE
    assert top(V=1000, ld=1000, k=257) == ESHAPE

    def dis(logits=p, dt=0, ld=16, N=1, V=16, vt=0, K=4, T=1.0, loss=p, grad=p, gld=16, idx=p):
        return lib.rwkv7_distill(logits, dt, ld, N, V, p, vt, idx, K, None, T, None, 1.0, loss, grad, gld, None)

    assert dis(logits=None) == dis(idx=None) == dis(loss=None, grad=None) == dis(dt=3) == dis(vt=3) == EINVAL
    for T in (0.0, -1.0, math.nan, math.inf):
        assert dis(T=T) == EINVAL
    assert dis(N=0) == dis(V=0) == dis(V=65537, ld=65537, gld=65537) == dis(ld=15) == dis(K=0) == dis(K=1025) == ESHAPE
    assert dis(gld=15) == ESHAPE

    def ver(target=p, draft=p, dt=0, tok=p, u=p, B=1, K=2, V=16, tr=16, dr=16, T=1.0, Td=1.0, ws=1 << 20, out=p):
        return lib.rwkv7_verify(target, 48, tr, draft, 32, dr, dt, tok, u, None, B, K, V, T, Td, out, p, p, ws, None)

    assert ver(target=None) == ver(tok=None) == ver(u=None) == ver(dt=3) == ver(out=None) == EINVAL
    assert ver(T=math.nan) == ver(Td=math.nan) == ver(T=math.inf) == ver(Td=math.inf) == EINVAL
    assert ver(B=0) == ver(K=-1) == ver(K=64) == ver(V=0) == ver(V=65537, tr=65537) == ver(tr=15) == ver(dr=15) == ESHAPE
    assert ver(B=13108) == ESHAPE  # 13108 (2 2 + 1) rows
    assert ver(ws=16) == EWORKSPACE
    assert lib.rwkv7_verify_workspace_bytes(0, 1, 16) == lib.rwkv7_verify_workspace_bytes(1, 64, 16) == 0


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="ROCm device"):
        K.top_logits(_t(2, 8), 2)
    with pytest.raises(ValueError, match="ROCm device"):
        K.distill_loss(_t(2, 8), _t(2, 3), _t(2, 3, dtype=torch.int64))
    with pytest.raises(ValueError, match="ROCm device"):
        rwkv_tl_amd.verify_draft(_t(1, 3, 8), _t(1, 2, dtype=torch.int64), None)
    with pytest.raises(NotImplementedError):
        ops.top_logits(_t(2, 8), 2)


def test_meta_shapes():
    x = torch.empty(2, 5, 100, dtype=torch.bfloat16, device="meta")
    v, i, lse = ops.top_logits(x, 7, 2.0)
    assert (v.shape, v.dtype, i.shape, i.dtype, lse.shape, lse.dtype) == (
        (2, 5, 7), torch.bfloat16, (2, 5, 7), torch.int64, (2, 5), torch.float32)
    y = x.clone().requires_grad_()
    loss = ops.distill_loss(y, v, i, lse, 2.0)
    assert loss.shape == (2, 5) and loss.dtype == torch.float32
    (g,) = torch.autograd.grad(loss.sum(), y, create_graph=True)
    assert g.shape == x.shape and g.dtype == torch.bfloat16
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(g.float().sum(), y)
    with pytest.raises(ValueError, match="no gradient to the teacher"):
        ops.distill_loss(y, v.clone().requires_grad_(), i, lse, 2.0)
