"""The ends and the norms of a training step, on the CPU: the float64 oracle against
closed forms and differences, refusals of the C entries and of the Python ones, Meta
shapes. (The kernels themselves: test_gpu_training.py, test_gpu_token_logprobs.py.)"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import rwkv_tl_amd  # noqa: F401
from oracle import training_ref as R
from rwkv_tl_amd import _lib
from rwkv_tl_amd import kernels as K

ops = torch.ops.rwkv_tl
INF, NAN = math.inf, math.nan


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------


def test_oracle_embedding():
    w = torch.arange(12.0).reshape(4, 3)
    t = torch.tensor([[2, -1], [2, 4]])
    assert R.embed(w, t, 0.5).tolist() == [[[3, 3.5, 4], [0, 0, 0]], [[3, 3.5, 4], [0, 0, 0]]]
    g = torch.arange(12.0).reshape(2, 2, 3)
    assert R.embed_grad(g, t, 4, 2.0).tolist() == [[0, 0, 0], [0, 0, 0], [12, 16, 20], [0, 0, 0]]
    # the gradient is the lookup's transpose: <embed(w), g> = <w, embed_grad(g)>
    left, right = (R.embed(w, t, 3.0) * g).sum(), (w * R.embed_grad(g, t, 4, 3.0)).sum()
    assert math.isclose(float(left), float(right), rel_tol=1e-14)


def test_oracle_layer_norm():
    x = torch.tensor([[1.0, 3.0], [5.0, 5.0]]).double()
    one, zero = torch.ones(2).double(), torch.zeros(2).double()
    y, mean, rstd = R.layer_norm(x, one, zero, 1e-30)
    assert mean.tolist() == [2.0, 5.0] and math.isclose(rstd[0], 1.0) and y[0].tolist() == pytest.approx([-1.0, 1.0])
    assert y[1].tolist() == [0.0, 0.0] and math.isclose(rstd[1], 1e15)
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = (torch.randn(*s, generator=g).double() for s in ((5, 7), (7,), (7,), (5, 7)))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    assert torch.autograd.gradcheck(lambda *a: R.layer_norm(*a)[0], leaves, eps=1e-6, atol=1e-7)
    want = torch.autograd.grad(R.layer_norm(x, w, b)[0], leaves, dy)
    for got, ref in zip(R.layer_norm_grad(dy, x.detach(), w.detach()), want):
        assert torch.allclose(got, ref, rtol=1e-12, atol=1e-13)


def test_oracle_token_logprobs():
    z = torch.tensor([[0.0, math.log(3.0), -INF, 0.0], [-INF] * 4, [1.0, NAN, 0.0, 0.0], [1.0, INF, 0.0, 0.0]], dtype=torch.float64)
    t = torch.tensor([1, 0, 0, 0])
    lp, H = R.token_logprobs(z, t)
    assert math.isclose(lp[0], math.log(0.6)) and math.isclose(H[0], -0.6 * math.log(0.6) - 0.4 * math.log(0.2))
    assert lp[1] == -INF and H[1] == 0 and lp[2:].isnan().all() and H[2:].isnan().all()
    lp, H = R.token_logprobs(z, torch.tensor([4, -1, -100, 7]))
    assert lp.tolist() == H.tolist() == [0.0] * 4
    lp, H = R.token_logprobs(torch.zeros(1, 8), torch.tensor([3]))
    assert math.isclose(lp[0], -math.log(8)) and math.isclose(H[0], math.log(8))


def test_oracle_token_gradient_matches_differences():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(4, 9, generator=g).double()
    t = torch.tensor([0, 8, 3, -1])
    s, h = torch.randn(4, generator=g).double(), torch.randn(4, generator=g).double()
    x = z.clone().requires_grad_()
    assert torch.autograd.gradcheck(lambda a: R.token_logprobs(a, t, 1.5), x, eps=1e-6, atol=1e-7)
    lp, H = R.token_logprobs(x, t, 1.5)
    (want,) = torch.autograd.grad((lp, H), x, (s, h))
    assert torch.allclose(R.token_logprobs_grad(z, t, s, h, 1.5), want, rtol=1e-12, atol=1e-13)
    z[0, 2] = -INF  # a masked entry takes no part
    got = R.token_logprobs_grad(z, t, s, h, 1.5)
    assert got[0, 2] == 0 and got.isfinite().all()


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    buf = (ctypes.c_char * 64)()
    p = ctypes.addressof(buf)  # never read: every call is refused on the host
    EINVAL, ESHAPE, EWORKSPACE = 1, 2, 3

    def emb(w=p, dt=0, ld=8, tok=p, out=p, N=4, V=16, C=8):
        return lib.rwkv7_embed(w, dt, ld, tok, 1.0, out, N, V, C, None)

    assert emb(w=None) == emb(tok=None) == emb(out=None) == emb(dt=-1) == emb(dt=3) == EINVAL
    assert emb(ld=7) == emb(N=0) == emb(N=2**24) == emb(V=0) == emb(V=2**20 + 1) == emb(C=0) == ESHAPE
    assert emb(C=65537, ld=65537) == ESHAPE

    size = lib.rwkv7_embed_backward_workspace_bytes
    assert 0 < size(0, 1, 16, 8) < size(0, 65, 16, 8) and size(0, 0, 16, 8) == size(0, 65, 0, 8) == size(0, 2**24, 16, 8) == 0

    def embg(g=p, dt=0, ld=8, tok=p, out=p, N=65, V=16, C=8, ws=p, nb=None):
        return lib.rwkv7_embed_backward(g, dt, ld, tok, 1.0, out, N, V, C, ws, size(0, 65, 16, 8) if nb is None else nb, None)

    assert embg(g=None) == embg(tok=None) == embg(out=None) == embg(dt=3) == embg(ws=None) == EINVAL
    assert embg(ld=7) == embg(N=0) == embg(V=0) == embg(V=2**20 + 1) == embg(C=0) == ESHAPE
    assert embg(nb=size(0, 65, 16, 8) - 1) == EWORKSPACE

    def norm(x=p, dt=0, ld=8, w=p, b=p, wt=1, eps=1e-5, y=p, m=p, r=p, N=3, C=8):
        return lib.rwkv7_layer_norm_forward(x, dt, ld, w, b, wt, eps, y, m, r, N, C, None)

    assert norm(x=None) == norm(w=None) == norm(b=None) == norm(y=None) == norm(m=None) == norm(r=None) == EINVAL
    assert norm(dt=3) == norm(wt=2) == norm(dt=1, wt=0) == norm(wt=-1) == EINVAL
    for eps in (0.0, -1e-5, NAN, INF, 1e-31, 1e31):
        assert norm(eps=eps) == EINVAL
    assert norm(ld=7) == norm(N=0) == norm(C=0) == norm(C=16385, ld=16385) == ESHAPE

    nsize = lib.rwkv7_layer_norm_backward_workspace_bytes
    assert nsize(0, 0, 8) == nsize(0, 3, 0) == nsize(0, 3, 16385) == 0 < nsize(0, 3, 8)

    def normg(g=p, ldg=8, x=p, ld=8, dt=0, w=p, wt=1, m=p, r=p, gx=p, gw=p, gb=p, N=3, C=8, ws=p, nb=1 << 20):
        return lib.rwkv7_layer_norm_backward(g, ldg, x, ld, dt, w, wt, m, r, gx, gw, gb, N, C, ws, nb, None)

    for bad in ("g", "x", "w", "m", "r", "gx", "gw", "gb", "ws"):
        assert normg(**{bad: None}) == EINVAL
    assert normg(dt=3) == normg(wt=2) == normg(dt=1, wt=2) == EINVAL
    assert normg(ldg=7) == normg(ld=7) == normg(N=0) == normg(C=0) == normg(C=16385, ld=16385, ldg=16385) == ESHAPE
    assert normg(nb=nsize(0, 3, 8) - 1) == EWORKSPACE

    def tok(z=p, dt=0, ld=16, N=1, V=16, t=p, T=1.0, k=0, lp=p, H=p, tl=p, ti=p):
        return lib.rwkv7_token_logprobs(z, dt, ld, N, V, t, T, k, lp, H, tl, ti, None)

    assert tok(z=None) == tok(t=None) == tok(lp=None) == tok(H=None) == tok(dt=3) == EINVAL
    assert tok(k=2, tl=None) == tok(k=2, ti=None) == EINVAL
    assert tok(N=0) == tok(V=0) == tok(V=65537, ld=65537) == tok(ld=15) == tok(k=-1) == tok(k=17) == ESHAPE
    assert tok(V=1000, ld=1000, k=257) == ESHAPE

    def tokg(z=p, dt=0, ld=16, N=1, V=16, t=p, T=1.0, g=p):
        return lib.rwkv7_token_logprobs_grad(z, dt, ld, N, V, t, T, None, 1.0, None, 0.0, None, None, g, None)

    assert tokg(z=None) == tokg(t=None) == tokg(g=None) == tokg(dt=-1) == EINVAL
    assert tokg(N=0) == tokg(V=0) == tokg(V=65537, ld=65537) == tokg(ld=15) == ESHAPE
    for T in (0.0, -1.0, NAN, INF):
        assert tok(T=T) == tokg(T=T) == EINVAL


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    i = _t(2, dtype=torch.int64)
    for call in (
        lambda: K.embed(_t(4, 8), i),
        lambda: K.embed_backward(_t(2, 8), i, 4),
        lambda: K.layer_norm_forward(_t(2, 8), _t(8), _t(8)),
        lambda: K.layer_norm_backward(_t(2, 8), _t(2, 8), _t(8), _t(2, dtype=torch.float32), _t(2, dtype=torch.float32)),
        lambda: K.token_logprobs(_t(2, 8), i),
        lambda: K.token_logprobs_grad(_t(2, 8), i),
    ):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    for call in (lambda: ops.embed(_t(4, 8), i), lambda: ops.layer_norm(_t(2, 8), _t(8), _t(8)),
                 lambda: ops.token_logprobs(_t(2, 8), i)):
        with pytest.raises(NotImplementedError):
            call()


def test_meta_shapes():
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    w, t = meta(100, 24).requires_grad_(), meta(2, 5, dtype=torch.int64)
    x = ops.embed(w, t, 2.0)
    assert x.shape == (2, 5, 24) and x.dtype == torch.bfloat16
    g, b = meta(24, dtype=torch.float32).requires_grad_(), meta(24, dtype=torch.float32).requires_grad_()
    y = ops.layer_norm(x, g, b)
    assert y.shape == x.shape and y.dtype == x.dtype
    z = y @ meta(24, 100)
    lp, H = ops.token_logprobs(z, t, 0.7)
    assert lp.shape == H.shape == (2, 5) and lp.dtype == H.dtype == torch.float32
    grads = torch.autograd.grad(lp.sum() + H.sum(), (w, g, b), create_graph=True)
    assert [(v.shape, v.dtype) for v in grads] == [(v.shape, v.dtype) for v in (w, g, b)]
    _, mean, rstd = ops.layer_norm_forward(x.detach(), g.detach(), b.detach())
    assert mean.shape == rstd.shape == (2, 5) and mean.dtype == torch.float32


@pytest.mark.parametrize("name", ["embed", "layer_norm", "token_logprobs"])
def test_second_derivatives_are_refused(name):
    meta = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    x, t = meta(6, 8).requires_grad_(), meta(6, dtype=torch.int64)
    y = {"embed": lambda: ops.embed(x, t), "layer_norm": lambda: ops.layer_norm(x, meta(8), meta(8)),
         "token_logprobs": lambda: ops.token_logprobs(x, t)[0]}[name]()
    (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match=f"{name} has no second derivative"):
        torch.autograd.grad(g.sum(), x)
