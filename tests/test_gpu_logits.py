"""The operators between a large and a small model (``rwkv_tl_amd.logits``) on
the GPU, against float64 on the CPU (``oracle.logits_ref``).

Tolerances (u = 2^-24, half a step of float32). An exponential 2^((x - m) kf) with
a = (m - x) / T is off by its argument's three roundings, 3u a, and the
instruction's last place, 2u. In a sum S of them about m that is 3u times the mean
a, which is the entropy less log S, so at most log V < 11.1; the additions of a
thread and a wave add at most 20u. A sum, and its logarithm, are so within 56u =
3.3e-6, and u of the stored value. A loss has P < 1 such logarithms of the row and
at most two for its rest: 112u. A gradient's terms f q and f p: the sum's 56u, the
factor's and the product's roundings and the exponential's 3u a + 2u, 60u + 3u a
with a < -log q, and half a step of the type it is stored in.
"""

from __future__ import annotations

import math

import pytest

import torch

import rwkv_tl_amd  # noqa: F401
from oracle import logits_ref as R
from rwkv_tl_amd import kernels as K
from rwkv_tl_amd import verify_draft

pytestmark = pytest.mark.gpu
ops = torch.ops.rwkv_tl
H, B16, F = torch.float16, torch.bfloat16, torch.float32
U = 2.0**-24
INF, NAN = float("inf"), float("nan")


def _zipf(g, *shape):
    return -1.3 * torch.empty(*shape).exponential_(generator=g).log()


def _gen(*key):
    return torch.Generator().manual_seed(sum((i + 3) * 1009**i * k for i, k in enumerate(key)) % (1 << 40))


def _lse_close(got, want):
    got, stored = got.double().cpu(), want.float()
    want = torch.where(stored.isinf(), stored.double(), want)  # past float32's range
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    assert ((got - want).abs()[fine] <= 56 * U + U * want.abs()[fine]).all()


# ---------------------------------------------------------------------------
# top_logits
# ---------------------------------------------------------------------------


def _ref_top(x, k, T):
    d = x.double().cpu()
    v, i = torch.sort(d, dim=-1, descending=True, stable=True)
    return v[..., :k], i[..., :k], torch.logsumexp(d / T, -1)


def _check_top(x, k, T=1.0, ref=None):
    v, i, lse = K.top_logits(x, k, temperature=T)
    wv, wi, wl = _ref_top(x, k, T) if ref is None else ref
    assert v.dtype == x.dtype and torch.equal(i.cpu(), wi)
    assert torch.equal(v.double().cpu().nan_to_num(nan=1e300, posinf=1e301, neginf=-1e301),
                       wv.nan_to_num(nan=1e300, posinf=1e301, neginf=-1e301))
    _lse_close(lse, wl)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("N,V,k,T", [
    (1, 1, 1, 1.0), (3, 7, 7, 0.5), (2, 8, 8, 1.0), (5, 100, 100, 1.0), (2, 257, 256, 3.0), (4, 1000, 17, 1.0), (2, 2047, 1, 1.0),
    (3, 5001, 64, 0.8), (2, 16384, 200, 1.0), (2, 16385, 256, 1.0), (3, 32769, 100, 2.0), (2, 65535, 128, 1.0),
    (2, 65536, 256, 1.0), (2, 65536, 1, 0.1), (301, 777, 5, 1.0)])
def test_top_logits(cuda, dtype, N, V, k, T):
    _check_top(_zipf(_gen(N, V, k), N, V).to(dtype).to(cuda), k, T)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("V,k", [(9, 9), (3000, 50), (20000, 256), (65536, 100), (65533, 256)])
def test_top_logits_ties(cuda, dtype, V, k):
    g = _gen(V, k, 5)
    x = torch.empty(6, V)
    x[0] = 1.25                                              # all alike
    x[1] = torch.randint(0, 2, (V,), generator=g).float()    # two values
    x[2] = torch.randint(-3, 4, (V,), generator=g).float()
    x[3] = torch.arange(V).float() / V                       # ascending: the last ids win
    x[4] = -x[3]
    x[5] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)  # zeros of both signs are one value
    x = x.to(dtype).to(cuda)
    _check_top(x, k)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("V,k", [(40, 40), (3000, 60)])
def test_top_logits_masks_and_nan(cuda, dtype, V, k):
    g = _gen(V, k, 6)
    x = torch.randn(8, V, generator=g)
    x[0] = -INF                                 # nothing left
    x[1, 5:] = -INF                             # fewer than k left
    x[2, torch.randperm(V, generator=g)[: V - k // 2]] = -INF
    x[3, ::3] = NAN
    x[4] = NAN
    x[5, 7] = INF
    x[6, 1:] = NAN
    x[7, 3:9] = torch.finfo(dtype).min          # a mask of the type's lowest value
    x = x.to(dtype)
    v, i, lse = R.top_logits(x, k)
    lse[5] = NAN                                # a row with +inf: as m + log sum exp(x - m)
    _check_top(x.to(cuda), k, ref=(v, i, lse))


def test_top_logits_layouts(cuda):
    g = _gen(7)
    base = _zipf(g, 9, 2100).to(H).to(cuda)
    _check_top(base[:, 3:2050], 33)                       # rows at odd 16-bit offsets
    _check_top(base[::2, 1:1000], 5)
    _check_top(base.t(), 9)                               # columns apart
    _check_top(base[0, :50].expand(4, 50), 10)            # one row several times
    f = _zipf(g, 4, 3001).to(cuda)
    _check_top(f[:, 1:], 20)
    v, i, lse = K.top_logits(base.view(3, 3, 2100), 4)
    assert v.shape == i.shape == (3, 3, 4) and lse.shape == (3, 3)
    w = K.top_logits(base, 4)
    assert torch.equal(v.view(9, 4), w[0]) and torch.equal(i.view(9, 4), w[1]) and torch.equal(lse.view(9), w[2])
    v, i, lse = K.top_logits(base[0], 4)
    assert v.shape == (4,) and lse.shape == () and torch.equal(i, w[1][0])
    v, i, lse = K.top_logits(base[:0], 4)
    assert v.shape == (0, 4) and i.shape == (0, 4) and lse.shape == (0,)


def test_top_logits_rows_past_2_to_the_31_elements(cuda):
    """Row offsets past 32 bits: the last rows of 2.2e9 half logits."""
    N = 33600
    x = torch.zeros(N, 65536, dtype=H, device=cuda)
    hot = (torch.arange(N, device=cuda) * 7919) % 65536
    x[torch.arange(N, device=cuda), hot] = 3.0
    v, i, _ = K.top_logits(x, 1)
    assert torch.equal(i[:, 0], hot) and bool((v == 3.0).all())
    val, idx = v.contiguous(), i.contiguous()
    loss, grad = K.distill_loss_grad(x, val, idx)
    want = float(torch.logsumexp(torch.cat([torch.zeros(65535), torch.tensor([3.0])]).double(), 0)) - 3.0
    assert (loss.double() - want).abs().max() < 56 * U + U * want
    assert bool((grad[torch.arange(N, device=cuda), hot].double() + (1 - 2.718281828459045 ** -want)).abs().max() < 1e-3)
    assert bool((grad != 0).sum(-1).min() == grad.shape[1])


def test_more_rows_than_a_launch_has(cuda):
    # Rows of the same logits have the same bits. Rows whose 1.0 stands elsewhere add the same
    # three numbers in another order, which is a rounding of a sum in 32 bits: (1 + e) + e and
    # (e + e) + 1, e = 1/exp(1), are half a step apart before they round. They are held to the
    # formula: lse = log(exp(1) + 2), loss = lse - 1 (no rest: the entry alone is the teacher).
    N = (1 << 21) + 5
    x = torch.zeros(N, 3, dtype=H, device=cuda)
    hot = torch.arange(N, device=cuda) % 3
    x[torch.arange(N, device=cuda), hot] = 1.0
    v, i, lse = K.top_logits(x, 1)
    want = math.log(math.exp(1.0) + 2.0)
    assert torch.equal(i[:, 0], hot) and bool((v == 1).all())
    assert torch.equal(lse, lse[hot]) and bool(((lse - want).abs() < 16 * U * want).all())
    loss, grad = K.distill_loss_grad(x, v, i)
    assert torch.equal(loss, loss[hot]) and bool(((loss - (want - 1)).abs() < 56 * U).all())
    assert torch.equal(grad, grad[hot]) and bool((grad != 0).all())


def test_top_logits_refusals(cuda):
    x = torch.zeros(2, 100, dtype=H, device=cuda)
    for bad in (lambda: K.top_logits(x, 0), lambda: K.top_logits(x, 101), lambda: K.top_logits(x, 2.0),
                lambda: K.top_logits(x.double(), 2), lambda: K.top_logits(x.long(), 2),
                lambda: K.top_logits(torch.zeros(1, 1000, device=cuda), 257),
                lambda: K.top_logits(torch.zeros(1, 65537, device=cuda), 2),
                lambda: K.top_logits(x, 2, temperature=0.0), lambda: K.top_logits(x, 2, temperature=NAN),
                lambda: K.top_logits(torch.zeros((), device=cuda), 1), lambda: K.top_logits(x[:, :0], 1)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------
# distill_loss and its gradient
# ---------------------------------------------------------------------------


def _case(g, N, V, k, dtype, T, rest, val_dtype=None):
    """(logits, top_val, top_idx, lse) on the CPU, the logits of `dtype`."""
    t = _zipf(g, N, V)
    z = (t + 0.7 * torch.randn(N, V, generator=g) - 1.5).to(dtype)
    val, idx = t.topk(min(k, V))
    return z, val.to(val_dtype or dtype), idx, torch.logsumexp(t / T, -1) if rest else None


def _check_distill(cuda, z, val, idx, lse, T=1.0, scale=None):
    """Loss, and loss with gradient, against float64 with element-wise tolerances."""
    N, V = z.shape
    dtype = z.dtype
    scale = torch.linspace(0.5, 2.0, max(N, 1))[:N] if scale is None else scale
    up = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    zc, vc, ic, lc = up(z), up(val), up(idx), up(lse)
    loss = K.distill_loss(zc, vc, ic, lc, temperature=T)
    both = K.distill_loss_grad(zc, vc, ic, lc, temperature=T, scale=up(scale))
    back = K.distill_loss_backward(up(scale), zc, vc, ic, lc, T)
    assert torch.equal(both[0].nan_to_num(nan=1e30), loss.nan_to_num(nan=1e30)) and torch.equal(both[1], back)
    assert back.dtype == dtype and back.shape == z.shape
    d = z.double().requires_grad_()
    want = R.distill_loss(d, val, idx, lse, T)
    some = ((idx >= 0) & (idx < V)).any(-1)
    got = loss.double().cpu()
    fine = want.detach().isfinite()
    assert torch.equal(got[~fine], want.detach()[~fine])
    assert ((got - want.detach()).abs()[fine] <= 112 * U + U * want.detach().abs()[fine]).all()
    assert (got[~some] == 0).all()
    (ref,) = torch.autograd.grad((want * scale.double()).sum(), d) if want.requires_grad else (torch.zeros_like(d),)
    # the sizes of the terms: q (P + R), q R / (1 - Q) and p, each times scale / T
    q = torch.softmax(d.detach() / T, -1)
    live = (idx >= 0) & (idx < V)
    if lse is None:
        p = torch.softmax((val.double() / T).masked_fill(~live, -INF), -1).nan_to_num(0.0)
    else:
        p = (val.double() / T - lse.double()[:, None]).exp()
    p = torch.where(live, p, 0.0)
    at = torch.where(live, idx, 0)
    inside = torch.zeros(N, V + 1, dtype=torch.bool).scatter_(1, torch.where(live, idx, V), True)[:, :V]
    rest = (1 - p.sum(-1, keepdim=True)).clamp_min(0) * (~inside).any(-1, keepdim=True) if lse is not None else torch.zeros(N, 1)
    among = torch.softmax((d.detach() / T).masked_fill(inside, -INF), -1).nan_to_num(0.0)  # q / (1 - Q) outside the ids
    size = q * (p.sum(-1, keepdim=True) + rest) + among * rest + torch.zeros_like(q).scatter_add(1, at, p)
    size = size * (scale.double()[:, None] / T)
    tiny = {H: 2.0**-25, B16: 2.0**-133, F: 2.0**-126}[dtype]  # half the lowest step; an exponential below the normals is 0
    tol = (60 - 3 * q.clamp_min(1e-300).log()) * U * size + torch.finfo(dtype).eps / 2 * ref.abs() + tiny + 2.0**-125 * scale.double().abs()[:, None] / T
    err = (back.double().cpu() - ref).abs()
    assert (err <= tol).all(), f"{float((err / tol).max())} of the tolerance"
    assert (back[~some.to(cuda)] == 0).all()


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("N,V,k,T", [
    (1, 1, 1, 1.0), (2, 7, 3, 0.5), (3, 8, 8, 1.0), (4, 100, 1, 1.0), (5, 1000, 64, 2.0), (3, 1001, 65, 1.0), (2, 2000, 1000, 1.0),
    (2, 1024, 1024, 1.0), (3, 16384, 256, 1.0), (2, 16385, 257, 0.7), (2, 20011, 100, 2.0), (2, 32768, 20, 1.0),
    (2, 32771, 600, 1.0), (2, 65535, 64, 1.0), (2, 65536, 1024, 1.5), (2, 65536, 50, 1.0), (130, 999, 30, 1.0)])
def test_distill(cuda, dtype, rest, N, V, k, T):
    _check_distill(cuda, *_case(_gen(N, V, k, rest), N, V, k, dtype, T, rest), T)


@pytest.mark.parametrize("dtype", [H, F], ids=str)
@pytest.mark.parametrize("rest", [False, True])
def test_distill_ragged_rows_and_foreign_ids(cuda, dtype, rest):
    """Rows with fewer entries, with none, ids past the vocabulary, and what stands in their places."""
    g = _gen(11, rest)
    z, val, idx, lse = _case(g, 12, 3003, 70, dtype, 1.0, rest, F)
    keep = torch.tensor([70, 0, 1, 35, 64, 65, 69, 0, 2, 70, 70, 70])
    gone = torch.arange(70) >= keep[:, None]
    idx = torch.where(gone, torch.tensor([-1, 3003, -(2**40), 2**40])[torch.randint(0, 4, (12, 70), generator=g)], idx)
    val = torch.where(gone, torch.tensor([NAN, INF, -INF])[torch.randint(0, 3, (12, 70), generator=g)], val)
    perm = torch.randperm(70, generator=g)  # absent entries anywhere
    idx, val = idx[:, perm].contiguous(), val[:, perm].contiguous()
    z[1] = NAN  # padded rows hold anything
    z[7] = INF
    clean = z.clone()
    clean[1] = clean[7] = 0.0
    _check_distill(cuda, clean, val, idx, lse)
    up = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    a = K.distill_loss_grad(up(z), up(val), up(idx), up(lse))
    b = K.distill_loss_grad(up(clean), up(val), up(idx), up(lse))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [B16, F], ids=str)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("V,k", [(50, 40), (5000, 300)])
def test_distill_same_id_in_several_entries(cuda, dtype, rest, V, k):
    g = _gen(V, k, 12)
    z, val, idx, lse = _case(g, 4, V, k, dtype, 1.0, rest, F)
    twin = torch.randint(0, k, (4, k), generator=g)
    idx = idx.gather(1, twin)
    idx[0, :] = idx[0, 0]  # a row of one id
    val = val.gather(1, twin) - 1.0
    _check_distill(cuda, z, val, idx, lse)
    up = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    runs = [K.distill_loss_grad(up(z), up(val), up(idx), up(lse)) for _ in range(3)]
    assert all(torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1]) for r in runs)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("T", [1.0, 0.04])
@pytest.mark.parametrize("rest", [False, True])
def test_distill_masked_vocabularies(cuda, dtype, T, rest):
    g = _gen(13, rest)
    low = torch.finfo(dtype).min
    z, val, idx, lse = _case(g, 9, 2001, 20, F, T, rest)
    away = torch.ones(2001, dtype=torch.bool)
    away[idx[0]] = False
    z[0, away] = torch.where(torch.rand(int(away.sum()), generator=g) < 0.7, -INF, z[0, away])  # a mask outside the entries
    val[1, 5:] = -INF                                    # the teacher's own mask
    z[1, idx[1, 5:]] = -INF                              # under which the student's -inf costs nothing
    z[2, torch.randint(0, 2001, (900,), generator=g)] = low / 2
    z[2, idx[2]] = 0.0
    z[3] -= 30000.0                                      # far from 0
    z[4] *= 40.0
    z[5] = 0.25                                          # a flat student
    z[6] = low                                           # masks of the type's lowest value: a row of nothing else,
    val[7], idx[7] = val[1], idx[1]
    z[7] = low                                           # and one outside the entries
    z[7, idx[7]] = torch.linspace(-2.0, 2.0, 20)
    z[8] = -low                                          # and of its highest, but for one
    z[8, 77] = -low / 2
    if lse is not None:
        lse[7] = lse[1]
    _check_distill(cuda, z.to(dtype), val, idx, lse, T)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
def test_top_logits_far_from_zero(cuda, dtype):
    g = _gen(41)
    low = torch.finfo(dtype).min
    x = torch.randn(6, 3001, generator=g)
    x[0] = low
    x[1] = -low
    x[1, 5] = -low / 2
    x[2, 100:] = low
    x[3] += 30000.0
    x[4] *= 500.0
    x[5, ::2] = low
    for T in (1.0, 0.02, 50.0):
        _check_top(x.to(dtype).to(cuda), 40, T)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("V", [20003, 65536])
def test_distill_rows_whose_first_logits_say_little(cuda, dtype, V):
    """A wave's sum is about the largest of its first 512 logits: rows that rise by hundreds behind them, whose first ones
    are masked, or the highest by hundreds."""
    g = _gen(43, V)
    z, val, idx, lse = _case(g, 5, V, 20, F, 1.0, True)
    z[0, V // 2:] += 300.0
    z[1, V - 3:] += 90.0
    z[2, :V // 4] = -INF
    z[2, idx[2]] = 0.0
    z[3, :V // 4] += 500.0
    z[4, :V - 100] = torch.finfo(dtype).min
    z[4, idx[4]] = 0.0
    _check_distill(cuda, z.to(dtype), val, idx, lse)
    x = z.clone()
    x[4, ::7] = -INF
    _check_top(x.to(dtype).to(cuda), 30)


def test_distill_infinite_and_nan_rows(cuda):
    z = torch.zeros(6, 40)
    val, idx = torch.zeros(6, 3), torch.tensor([[1, 2, 3]]).repeat(6, 1)
    z[0, 2] = -INF            # the teacher wants what the student rules out
    z[1] = NAN
    z[2, 30] = NAN
    z[3] = -INF
    val[4] = -INF             # without mass
    val[5, 1] = NAN
    loss, grad = (t.cpu() for t in K.distill_loss_grad(z.to(cuda), val.to(cuda), idx.to(cuda)))
    assert loss[0] == INF and loss[1].isnan() and loss[2].isnan() and loss[3].isnan() and loss[4] == 0 and loss[5].isnan()
    want = torch.softmax(z[0], -1)
    want[1:4] -= 1 / 3
    assert torch.allclose(grad[0], want, atol=1e-6)
    assert grad[1:4].isnan().all() and (grad[4] == 0).all() and grad[5].isnan().all()
    # rows that count for nothing
    grad = K.distill_loss_grad(z.to(cuda), val.to(cuda), idx.to(cuda), scale=torch.zeros(6, device=cuda))[1]
    assert (grad == 0).all()
    grad = K.distill_loss_grad(z.to(cuda), val.to(cuda), idx.to(cuda), scale=0.0)[1]
    assert (grad == 0).all()
    # a rest, and nothing of the student outside the ids: infinite, and no gradient to what has no probability
    z = torch.full((1, 40), -INF)
    z[0, 1:4] = 0.0
    loss, grad = K.distill_loss_grad(z.to(cuda), val[:1].to(cuda), idx[:1].to(cuda), torch.tensor([2.0], device=cuda))
    assert loss.item() == INF and (grad[0, 4:] == 0).all() and grad.isfinite().all()


def test_distill_gradient_against_differences(cuda):
    """The kernel's gradient along random directions against central differences of the float64 loss (h = 1e-4: h^2
    times a third derivative below 1 is 1e-8), within the gradient's own tolerance summed over the direction."""
    g = _gen(14)
    z, val, idx, lse = _case(g, 5, 3001, 40, F, 1.5, True)
    grad = K.distill_loss_grad(z.to(cuda), val.to(cuda), idx.to(cuda), lse.to(cuda), temperature=1.5)[1].double().cpu()
    for _ in range(4):
        d = torch.randn(5, 3001, generator=g, dtype=torch.float64)
        h = 1e-4
        diff = (R.distill_loss(z.double() + h * d, val, idx, lse, 1.5) - R.distill_loss(z.double() - h * d, val, idx, lse, 1.5)) / (2 * h)
        # (a gradient's terms are at most |g| + 2 q here, and a < 40: 180u)
        tol = 180 * U * ((grad.abs() + 2 * torch.softmax(z.double() / 1.5, -1)) * d.abs()).sum(-1) + 1e-7
        assert ((grad * d).sum(-1) - diff).abs().le(tol).all()


def test_distill_autograd(cuda):
    g = _gen(15)
    z, val, idx, lse = (t.to(cuda) for t in _case(g, 6, 4001, 30, H, 2.0, True))
    x = z.view(2, 3, 4001).clone().requires_grad_()
    v, i, ls = val.view(2, 3, 30), idx.view(2, 3, 30), lse.view(2, 3)
    loss = ops.distill_loss(x, v, i, ls, 2.0)
    assert loss.shape == (2, 3) and loss.dtype == F
    w = torch.rand(2, 3, generator=g).to(cuda)
    (loss * w).sum().backward()
    assert torch.equal(x.grad.view(6, 4001), K.distill_loss_backward(w.view(6), z, val, idx, lse, 2.0))
    x.grad = None
    ops.distill_loss(x, v, i, ls, 2.0).mean().backward()  # an expanded upstream gradient
    assert torch.equal(x.grad.view(6, 4001), K.distill_loss_grad(z, val, idx, lse, temperature=2.0, scale=1.0 / 6)[1])
    # not the contiguous layout: the gradient of a slice
    y = torch.zeros(6, 4010, dtype=H, device=cuda)
    y[:, 3:4004] = z
    y.requires_grad_()
    ops.distill_loss(y[:, 3:4004], val, idx, lse, 2.0).sum().backward()
    assert torch.equal(y.grad[:, 3:4004], K.distill_loss_grad(z, val, idx, lse, temperature=2.0)[1])
    with pytest.raises(ValueError, match="no gradient to the teacher"):
        ops.distill_loss(x, v.clone().requires_grad_(), i, ls, 2.0)
    (g1,) = torch.autograd.grad(ops.distill_loss(x, v, i, ls, 2.0).sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivative"):
        g1.float().sum().backward()


def test_distill_saved_tensors(cuda):
    """A saved-tensor hook that brings them back elsewhere, an in-place change that autograd refuses, copies of operands
    that are not adjacent, and a graph kept for a second backward."""
    g = _gen(18)
    z, val, idx, lse = (t.to(cuda) for t in _case(g, 4, 2001, 12, B16, 1.0, True))
    want = K.distill_loss_grad(z, val, idx, lse)[1]
    x = z.clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(cuda)):
        loss = ops.distill_loss(x, val, idx, lse).sum()
    loss.backward()
    assert torch.equal(x.grad, want)
    x = z.clone().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        loss = ops.distill_loss(x, val.t().contiguous().t(), idx.t().contiguous().t(), lse).sum()
    loss.backward()
    assert torch.equal(x.grad, want)
    x = z.clone().requires_grad_()
    loss = ops.distill_loss(x, val.t().contiguous().t(), idx, lse).sum()
    loss.backward(retain_graph=True)
    loss.backward()
    assert torch.equal(x.grad, want + want)
    x, v = z.clone().requires_grad_(), val.clone()
    loss = ops.distill_loss(x, v, idx, lse).sum()
    v.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.no_grad():
        assert torch.equal(ops.distill_loss(x, val, idx, lse), K.distill_loss(z, val, idx, lse))
    assert not ops.distill_loss(z, val, idx, lse).requires_grad


def test_distill_compiles(cuda):
    z, val, idx, _ = (None if t is None else t.to(cuda) for t in _case(_gen(16), 4, 1000, 10, F, 1.0, False))

    def step(x):
        return ops.distill_loss(x * 2.0, val, idx).sum()

    x = z.clone().requires_grad_()
    torch.compile(step, backend="aot_eager", fullgraph=True)(x).backward()
    y = z.clone().requires_grad_()
    step(y).backward()
    assert torch.equal(x.grad, y.grad)


def test_distill_layouts_and_empty(cuda):
    g = _gen(17)
    z, val, idx, lse = _case(g, 4, 999, 20, H, 1.0, True)
    wide = torch.zeros(4, 1010, dtype=H)
    wide[:, 5:1004] = z
    a = K.distill_loss_grad(wide.to(cuda)[:, 5:1004], val.to(cuda), idx.to(cuda), lse.to(cuda))
    b = K.distill_loss_grad(z.to(cuda), val.to(cuda), idx.to(cuda), lse.to(cuda))
    c = K.distill_loss_grad(z.to(cuda).t().contiguous().t(), val.to(cuda).t().contiguous().t(), idx.to(cuda), lse.to(cuda))
    for o in (a, c):
        assert torch.equal(o[0], b[0]) and torch.equal(o[1], b[1])
    loss, grad = K.distill_loss_grad(z.to(cuda)[:0], val.to(cuda)[:0], idx.to(cuda)[:0])
    assert loss.shape == (0,) and grad.shape == (0, 999)
    loss, grad = K.distill_loss_grad(z.to(cuda), val.to(cuda)[:, :0], idx.to(cuda)[:, :0])
    assert (loss == 0).all() and (grad == 0).all()


def test_distill_refusals(cuda):
    z, val, idx = torch.zeros(2, 50, device=cuda), torch.zeros(2, 4, device=cuda), torch.zeros(2, 4, dtype=torch.int64, device=cuda)
    lse = torch.zeros(2, device=cuda)
    big = torch.zeros(2, 1025, device=cuda)
    for bad in (lambda: K.distill_loss(z.double(), val, idx), lambda: K.distill_loss(z, val.double(), idx),
                lambda: K.distill_loss(z, val, idx.int()), lambda: K.distill_loss(z, val[:1], idx),
                lambda: K.distill_loss(z, val, idx[:, :3]), lambda: K.distill_loss(z, val, idx, lse[:1]),
                lambda: K.distill_loss(z, val, idx, lse.half()), lambda: K.distill_loss(z, val, idx, temperature=-1.0),
                lambda: K.distill_loss(z, val, idx, temperature=INF), lambda: K.distill_loss(z, big, big.long()),
                lambda: K.distill_loss_grad(z, val, idx, scale=lse[:1]), lambda: K.distill_loss(z, val.cpu(), idx),
                lambda: K.distill_loss(z, val, idx.cpu()), lambda: K.distill_loss(z, val, idx, lse.cpu())):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------
# verify_draft
# ---------------------------------------------------------------------------


def _drafts(g, B, k, V, dtype, Td, noise=0.7):
    target = _zipf(g, B, k + 1, V)
    draft = (target[:, :k] + noise * torch.randn(B, k, V, generator=g)).to(dtype)
    x = draft.float()
    if Td > 0:
        x = x / Td - torch.empty_like(x).exponential_(generator=g).log()
    tok = x.argmax(-1) if k else torch.zeros(B, 0, dtype=torch.int64)
    return target.to(dtype), tok, torch.rand(B, k + 1, generator=g), draft


def _check_verify(cuda, target, tok, u, draft, T, Td, lengths=None):
    up = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    out, n = verify_draft(up(target), up(tok), up(u), up(draft), temperature=T, draft_temperature=Td, lengths=up(lengths))
    want, wn = R.verify_draft(target, tok, u, draft, T, Td, lengths)
    assert torch.equal(n.cpu(), wn) and torch.equal(out.cpu(), want)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("T,Td", [(1.0, 1.0), (0.7, 1.2), (1.0, 0.0), (0.0, 0.0), (3.0, 0.5)])
@pytest.mark.parametrize("B,k,V", [(1, 1, 1), (2, 2, 7), (3, 0, 100), (5, 4, 1000), (2, 63, 130), (3, 3, 8191), (3, 3, 8192), (3, 3, 8193),
                                   (2, 5, 20011), (40, 3, 515), (2, 4, 65535), (3, 7, 65536)])
def test_verify(cuda, dtype, T, Td, B, k, V):
    target, tok, u, draft = _drafts(_gen(B, k, V, int(10 * T), int(10 * Td)), B, k, V, dtype, Td)
    _check_verify(cuda, target, tok, u, draft, T, Td)


@pytest.mark.parametrize("T,Td", [(1.0, 1.0), (1.0, 0.0), (0.0, 0.0)])
def test_verify_ragged_lengths(cuda, T, Td):
    g = _gen(21, int(T), int(Td))
    target, tok, u, draft = _drafts(g, 40, 6, 9001, H, Td, 0.3)
    lengths = torch.arange(40) % 7
    lengths[0], lengths[1] = -5, 100  # clamped
    tok[torch.arange(6) >= lengths.clamp(0, 6)[:, None]] = -7  # what stands behind them is not looked at
    _check_verify(cuda, target, tok, u, draft, T, Td, lengths)


def test_verify_identical_models_accept_everything(cuda):
    g = _gen(22)
    target, tok, u, _ = _drafts(g, 30, 5, 3001, B16, 1.0, 0.0)
    out, n = verify_draft(target.to(cuda), tok.to(cuda), u.to(cuda), target[:, :5].contiguous().to(cuda), temperature=1.0)
    assert (n == 5).all() and torch.equal(out[:, :5].cpu(), tok)
    # even a u of 1, which rejects, leaves no residue of p - q to draw from: p itself
    one = torch.ones_like(u)
    one[:, 5] = u[:, 5]
    _check_verify(cuda, target, tok, one, target[:, :5].contiguous(), 1.0, 1.0)


def test_verify_borders(cuda):
    """u = 0, the largest u below 1, 1, NaN; masked first tokens; nothing left to draw from."""
    V = 9000
    target = torch.full((6, 2, V), -INF)
    target[:, :, 100] = 0.0
    target[:, :, 8999] = 0.0
    target[:, :, 5] = NAN
    draft = target[:, :1].clone()
    draft[:, :, 100] = 3.0
    tok = torch.tensor([[100]] * 6)
    top = 1.0 - 2.0**-24
    u = torch.tensor([[0.0, 0.0], [top, 0.0], [top, top], [top, 1.0], [0.9, NAN], [NAN, 0.5]])
    for Td in (1.0, 0.0):
        _check_verify(cuda, target, tok, u, draft, 1.0, Td)
    out, n = verify_draft(target.to(cuda), tok.to(cuda), u.to(cuda), draft.to(cuda), temperature=1.0)
    assert n[0] == 1 and out[0].tolist() == [100, 100]         # u = 0: the first token with any weight
    assert n[1] == 0 and out[1].tolist() == [8999, -1]         # what the draft had too much of is taken out
    empty = torch.full((3, 2, 50), -INF)
    empty[1] = NAN
    empty[2, 1] = 0.0
    _check_verify(cuda, empty, torch.zeros(3, 1, dtype=torch.int64), torch.full((3, 2), 0.25), None, 1.0, 0.0)
    _check_verify(cuda, empty, torch.zeros(3, 1, dtype=torch.int64), torch.full((3, 2), 0.25), empty[:, :1].clone(), 1.0, 1.0)
    _check_verify(cuda, empty, torch.zeros(3, 1, dtype=torch.int64), None, None, 0.0, 0.0)


def test_verify_infinities_and_foreign_ids(cuda):
    g = _gen(23)
    target, tok, u, draft = _drafts(g, 8, 3, 2000, F, 1.0)
    target[0, 1, 7] = INF
    target[1, 0, 7] = target[1, 0, 9] = INF
    draft[2, 0, 11] = INF
    draft[3, 0] = -INF
    target[4, 0] = torch.finfo(F).min
    tok[5, 0], tok[6, 1], tok[7, 0] = -1, 2000, 2**40
    for T, Td in ((1.0, 1.0), (1.0, 0.0), (0.0, 0.0)):
        _check_verify(cuda, target, tok, u, draft, T, Td)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("T", [1.0, 0.01, 100.0])
def test_verify_far_from_zero(cuda, dtype, T):
    """Rows, and parts of rows, whose exponentials about 0 are past 64 bits on either side."""
    g = _gen(26)
    target, tok, u, draft = _drafts(g, 9, 2, 20003, F, T)
    low = torch.finfo(dtype).min
    target[0] -= 30000.0
    draft[0] += 30000.0
    target[1, :, :9000] = low
    draft[1, :, 9000:] = low
    target[2] *= 700.0
    target[3, :, 5] = -low
    draft[4] = low
    target[5] = low
    target[6, :, 100:] = -INF
    target[7, :, 8192:16384] -= 2000.0
    draft[7, :, :8192] += 1500.0
    target[8, :, 8192:] = NAN
    _check_verify(cuda, target.to(dtype), tok, u, draft.to(dtype), T, T)
    _check_verify(cuda, target.to(dtype), tok, u, None, T, 0.0)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("B,k,V", [(450, 3, 515), (225, 2, 9001), (57, 1, 65535)])
def test_verify_wide_batches(cuda, dtype, B, k, V):
    """As many sequences as take more of a decisive row to a workgroup."""
    for T, Td in ((1.0, 1.0), (0.7, 0.0)):
        _check_verify(cuda, *_drafts(_gen(27, B, int(Td)), B, k, V, dtype, Td, 1.5), T, Td)
    target, tok, u, draft = _drafts(_gen(28, B), 9, k, V, dtype, 1.0)
    low = torch.finfo(dtype).min
    target[0] *= 700.0
    target[1, :, V // 2 :] = low
    draft[2, :, : V // 2] = low
    draft[3] = low
    target[4, :, 3:] = -INF
    target[5] = -INF
    target[6, :, V // 2 :] = NAN
    target[7, :, : V // 3] -= 2000.0
    n = -(-B // 9)
    _check_verify(cuda, *(t.repeat(n, *[1] * (t.ndim - 1)) for t in (target, tok, u, draft)), 1.0, 1.0)


def test_verify_greedy_ties_take_the_lowest_id(cuda):
    target = torch.zeros(3, 3, 20000, dtype=H)
    target[1, :, 9000] = target[1, :, 8000] = target[1, :, 15000] = 1.0
    target[2, :, 12000:] = 2.0
    tok = torch.tensor([[0, 0], [8000, 9000], [12000, 12000]])
    out, n = verify_draft(target.to(cuda), tok.to(cuda), None)
    assert out.tolist() == [[0, 0, 0], [8000, 8000, -1], [12000, 12000, 12000]] and n.tolist() == [2, 1, 2]


def test_verify_layouts(cuda):
    g = _gen(24)
    target, tok, u, draft = _drafts(g, 4, 3, 1003, H, 1.0)
    want = R.verify_draft(target, tok, u, draft, 1.0, 1.0)
    tw = torch.zeros(4, 4, 1010, dtype=H, device=cuda)
    tw[:, :, 2:1005] = target.to(cuda)
    dw = torch.zeros(3, 4, 1003, dtype=H, device=cuda)
    dw.copy_(draft.transpose(0, 1))
    for t, d in ((tw[:, :, 2:1005], dw.transpose(0, 1)), (target.to(cuda).transpose(1, 2).contiguous().transpose(1, 2), draft.to(cuda))):
        out, n = verify_draft(t, tok.to(cuda).t().contiguous().t(), u.to(cuda), d, temperature=1.0)
        assert torch.equal(out.cpu(), want[0]) and torch.equal(n.cpu(), want[1])
    out, n = verify_draft(target[1].to(cuda), tok[1].to(cuda), u[1].to(cuda), draft[1].to(cuda), temperature=1.0,
                          lengths=torch.tensor(3, device=cuda))
    assert out.shape == (4,) and n.shape == () and torch.equal(out.cpu(), want[0][1])
    out, n = verify_draft(target[:0].to(cuda), tok[:0].to(cuda), u[:0].to(cuda), draft[:0].to(cuda), temperature=1.0)
    assert out.shape == (0, 4) and n.shape == (0,)


def test_verify_follows_the_targets_distribution(cuda):
    """60,000 drafts of one token against p: each frequency within 5 standard deviations (12 values; one in 10^5 runs
    would be outside by chance, and the inputs are fixed)."""
    g = _gen(25)
    V, n = 12, 60000
    pt, qd = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p, q = torch.softmax(pt.double() / 0.8, -1), torch.softmax(qd.double() / 1.3, -1)
    tok = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    u = torch.rand(n, 2, generator=g)
    counts = torch.zeros(V, dtype=torch.float64)
    for lo in range(0, n, 20000):
        s = slice(lo, lo + 20000)
        out, _ = verify_draft(pt.to(cuda).expand(20000, 2, V), tok[s].to(cuda), u[s].to(cuda), qd.to(cuda).expand(20000, 1, V),
                              temperature=0.8, draft_temperature=1.3)
        counts += torch.bincount(out[:, 0].cpu(), minlength=V)
    assert ((counts / n - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


def test_verify_refusals(cuda):
    t, x = torch.zeros(2, 4, 50, device=cuda), torch.zeros(2, 3, dtype=torch.int64, device=cuda)
    u, d = torch.zeros(2, 4, device=cuda), torch.zeros(2, 3, 50, device=cuda)
    for bad in (lambda: verify_draft(t, x, None, temperature=1.0), lambda: verify_draft(t.double(), x, u, temperature=1.0),
                lambda: verify_draft(t, x.int(), u, temperature=1.0), lambda: verify_draft(t, x[:, :2], u, temperature=1.0),
                lambda: verify_draft(t, x, u[:, :3], temperature=1.0), lambda: verify_draft(t, x, u.half(), temperature=1.0),
                lambda: verify_draft(t, x, u, d.half(), temperature=1.0), lambda: verify_draft(t, x, u, d[:, :2], temperature=1.0),
                lambda: verify_draft(t, x, u, d, temperature=NAN), lambda: verify_draft(t, x, u, d, temperature=1.0, draft_temperature=NAN),
                lambda: verify_draft(t, x, u, d, temperature=INF), lambda: verify_draft(t[0, 0], x, u, temperature=1.0),
                lambda: verify_draft(t, x, u, lengths=torch.zeros(2, device=cuda)), lambda: verify_draft(t, x.cpu(), u, temperature=1.0),
                lambda: verify_draft(torch.zeros(1, 65, 8, device=cuda), torch.zeros(1, 64, dtype=torch.int64, device=cuda), None),
                lambda: verify_draft(torch.zeros(1, 1, 8, device=cuda).expand(30000, 2, 8),
                                     torch.zeros(30000, 1, dtype=torch.int64, device=cuda), None)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------
# streams, graphs, and a run of them together
# ---------------------------------------------------------------------------


def test_calls_on_a_side_stream_and_two_at_once(cuda):
    g = _gen(31)
    z, val, idx, lse = (t.to(cuda) for t in _case(g, 40, 9001, 30, H, 1.0, True))
    target, tok, u, draft = (t.to(cuda) for t in _drafts(g, 4, 4, 9001, H, 1.0))
    call = lambda: (*K.top_logits(z, 20), *K.distill_loss_grad(z, val, idx, lse), *verify_draft(target, tok, u, draft, temperature=1.0))  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_graph_replays_match_eager(cuda):
    """Forward, backward, top logits and verification captured together; every replay on new inputs against eager."""
    g = _gen(32)
    bufs = [t.to(cuda) for t in _case(g, 33, 5001, 40, B16, 1.0, True)]
    ver = [t.to(cuda) for t in _drafts(g, 3, 4, 5001, B16, 1.0)]
    x = bufs[0].requires_grad_()

    def call():
        loss = ops.distill_loss(x, *bufs[1:], 1.0)
        (grad,) = torch.autograd.grad(loss, x, torch.full_like(loss, 0.25))
        return (*K.top_logits(x.detach(), 50), loss.detach(), grad, *verify_draft(*ver, temperature=0.9))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        h = _gen(33, i)
        for dst, src in zip(bufs + ver, [*_case(h, 33, 5001, 40, B16, 1.0, True), *_drafts(h, 3, 4, 5001, B16, 1.0)]):
            dst.data.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_single_rows_empty_batches_and_broadcast_inputs(cuda):
    """One row without a batch dimension, batches without rows, and gradients to a row that stands for many."""
    g = _gen(34)
    x = torch.randn(3, 2, 777, generator=g).to(B16).to(cuda)
    val, idx, lse = K.top_logits(x, 9)
    v1, i1, l1 = K.top_logits(x[1, 1], 9)
    assert v1.shape == (9,) and l1.shape == () and torch.equal(v1, val[1, 1]) and torch.equal(i1, idx[1, 1]) and torch.equal(l1, lse[1, 1])
    loss = K.distill_loss(x, val, idx, lse)
    one, grad = K.distill_loss_grad(x[1, 1], v1, i1, l1)
    assert loss.shape == (3, 2) and one.shape == () and torch.equal(one, loss[1, 1]) and grad.shape == (777,)
    for shape in ((0, 777), (3, 0, 777)):
        e = torch.empty(shape, device=cuda, requires_grad=True)
        top = K.top_logits(e.detach(), 5)
        assert top[0].shape == top[1].shape == (*shape[:-1], 5) and top[2].shape == shape[:-1]
        ops.distill_loss(e, *top, 1.0).sum().backward()
        assert e.grad.shape == shape
    # six equal rows: their gradients are added by autograd, in f32: five roundings of a sum below 6
    w = torch.randn(777, generator=g).to(cuda).requires_grad_()
    ops.distill_loss(w.expand(3, 2, 777), val, idx, lse).sum().backward()
    rows = K.distill_loss_grad(w.detach().expand(3, 2, 777), val, idx, lse)[1]
    assert bool(((w.grad - rows.double().sum((0, 1))).abs() <= 5 * U * rows.double().abs().sum((0, 1))).all())
    # an entry of one row for all
    assert torch.equal(K.distill_loss(x, val[:1, :1].expand(3, 2, 9), idx[:1, :1].expand(3, 2, 9)),
                       K.distill_loss(x, val[:1, :1].repeat(3, 2, 1), idx[:1, :1].repeat(3, 2, 1)))
    for B in (0, 1):
        t = torch.randn(B, 4, 777, generator=g).to(cuda)
        out, n = verify_draft(t, torch.zeros(B, 3, dtype=torch.int64, device=cuda), torch.rand(B, 4, device=cuda), t[:, :3], temperature=1.0)
        assert out.shape == (B, 4) and n.shape == (B,)
    t = torch.randn(1, 777, generator=g)
    u, tok = torch.rand(5, 4, generator=g), torch.randint(0, 777, (5, 3), generator=g)
    out, n = verify_draft(t.to(cuda).expand(5, 4, 777), tok.to(cuda), u.to(cuda), t.to(cuda).expand(5, 3, 777), temperature=1.0)
    want, wn = R.verify_draft(t.expand(5, 4, 777).contiguous(), tok, u, t.expand(5, 3, 777).contiguous(), 1.0, 1.0)
    assert torch.equal(out.cpu(), want) and torch.equal(n.cpu(), wn)
