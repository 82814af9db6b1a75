"""``token_logprobs`` and its gradient on the GPU, against float64 on the CPU
(``oracle.training_ref``).

Tolerances (U = 2^-24, half a step of float32). With a_j = (M - z_j) / T >= 0 the
distance from the row's largest logit, an exponential exp(-a_j) is off by three
roundings of its argument and the instruction's last place, U (3 a + 2); the
additions of a thread, a wave and a workgroup add 24 U at most (eight threads' 32,
in pairs: 12; wave 6; the rest in 64 bits). With S' the sum without the largest and A its mean a, S' is so
within rel = U (3 A + 26) of itself, and log S within rel S' / S. A log probability
and an entropy of n alike largest are within that, U of the stored value, and the
entropy's second sum, U sum a exp(-a) (3 a + 26) / S, once and by the other's error.

Gradient g_j = -q_j (s + h (log q_j + H)) / T: q_j within U (3 a + 2 + 6) and log S's; the
bracket within U of 4 (|s| + |h| (|H - log S| + a)) and the entropy's error times |h|. The
token's own: 1 - q within q times log S's error. Then half a step of the stored type, 2^-25 in
float16, and what exponentials below 2^-126 lose.
"""

from __future__ import annotations

import math

import pytest

import torch

import rwkv_tl_amd  # noqa: F401
from oracle import training_ref as R
from rwkv_tl_amd import kernels as K

pytestmark = pytest.mark.gpu
ops = torch.ops.rwkv_tl
H, B16, F = torch.float16, torch.bfloat16, torch.float32
DTYPES = pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
U = 2.0**-24
INF, NAN = float("inf"), float("nan")


def _gen(*key):
    return torch.Generator().manual_seed(sum((i + 3) * 1009**i * k for i, k in enumerate(key)) % (1 << 40))


def _zipf(g, *shape):
    return -1.3 * torch.empty(*shape).exponential_(generator=g).log()


def _tokens(g, N, V, pad=0.15):
    t = torch.randint(0, V, (N,), generator=g)
    out = torch.tensor([-1, V, -100, 2**40])
    return torch.where(torch.rand(N, generator=g) < pad, out[torch.randint(0, 4, (N,), generator=g)], t)


class Bounds:
    """Of rows that have a distribution (others: no bounds, their outputs are compared as they are)."""

    def __init__(self, z, T):
        d = z.double() / T
        self.y = R._log_softmax(d)
        self.M = d.amax(-1, keepdim=True)
        self.a = (self.M - d).clamp_min(0).nan_to_num(posinf=1e300)
        e = (-self.a).exp()
        self.a = torch.where(e == 0, torch.zeros_like(e), self.a)
        S = e.sum(-1)
        rest = torch.where(d == self.M, torch.zeros_like(e), e)
        S1 = rest.sum(-1)
        A = (rest * self.a).sum(-1) / S1.clamp_min(1e-300)
        self.log_S = S.log()
        rel = U * (3 * A + 26) * S1 / S
        self.lse = rel + 1e-10 * self.log_S
        T2 = U * (rest * self.a * (3 * self.a + 26)).sum(-1) / S
        self.H = rel * (1 + (rest * self.a).sum(-1) / S) + T2 + 1e-10

    def logp(self, want):
        return self.lse + U * want.abs() + 1e-12

    def entropy(self, want):
        return self.H + U * want.abs() + 1e-12

    def grad(self, want, H, s, h, T, dtype):
        s, h, H = s.abs()[:, None], h.abs()[:, None], H[:, None]
        q = self.y.exp()
        size = s + h * ((H - self.log_S[:, None]).abs() + self.a)
        err = q * (size * U * (3 * self.a + 12) + size * self.lse[:, None] + h * (self.H + self.lse)[:, None])
        own = (s + h) * q * self.lse[:, None]
        return (err + own) / T + (torch.finfo(dtype).eps / 2 + 2 * U) * want.abs() + (2.0**-25 if dtype is H16 else 0.0) + 2.0**-126 * (1 + size / T)


H16 = torch.float16


def _close(got, want, bound, name):
    got = got.double().cpu()
    fine = want.isfinite()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), name
    rest = ~fine & ~want.isnan()
    assert torch.equal(got[rest], want[rest]), name
    off = ((got - want).abs() / bound)[fine]
    assert not (off > 1).any(), f"{name}: {int((off > 1).sum())} off, the worst by {float(off.max())} bounds"


def _check(cuda, z, t, T=1.0, k=0, grad=True, key=0):
    zc, tc = z.to(cuda), t.to(cuda)
    B = Bounds(z, T)
    lp, ent = R.token_logprobs(z, t, T)
    out = K.token_logprobs(zc, tc, k, temperature=T)
    _close(out[0], lp, B.logp(lp), "logp")
    _close(out[1], ent, B.entropy(ent), "entropy")
    assert len(out) == (4 if k else 2) and out[0].dtype is out[1].dtype is F
    there = (t >= 0) & (t < z.shape[-1])
    if k:
        order = torch.sort(z.double().nan_to_num(nan=-INF, posinf=INF, neginf=-INF) if z.isnan().any() else z.double(),
                           dim=-1, descending=True, stable=True).indices[:, :k]
        order = torch.where(there[:, None], order, -1)
        clean = ~z.isnan().any(-1) | ~there
        assert torch.equal(out[3].cpu()[clean], order[clean])
        want = torch.where(there[:, None], B.y.gather(1, order.clamp_min(0)), -INF)
        _close(out[2][clean.to(cuda)], want[clean], (B.lse[:, None] + U * want.abs() + 1e-12)[clean], "top_logp")
    if grad:
        g = _gen(*z.shape, key, 77)
        s, h = torch.randn(z.shape[0], generator=g), torch.randn(z.shape[0], generator=g)
        s[::7] = 0
        h[::3] = 0
        for sv, hv in ((s, h), (s, torch.zeros_like(h)), (torch.zeros_like(s), h)):
            got = K.token_logprobs_grad(zc, tc, temperature=T, scale=sv.to(cuda), entropy_scale=hv.to(cuda))
            _close(got[0], lp, B.logp(lp), "logp with gradient")
            _close(got[1], ent, B.entropy(ent), "entropy with gradient")
            want = R.token_logprobs_grad(z, t, sv, hv, T)
            assert got[2].dtype is z.dtype
            _close(got[2], want, B.grad(want, ent, sv.double(), hv.double(), T, z.dtype), "gradient")
            alone = K.token_logprobs_backward(sv.to(cuda), hv.to(cuda), zc, tc, T)
            assert torch.equal(alone.nan_to_num(7.0), got[2].nan_to_num(7.0))


@DTYPES
@pytest.mark.parametrize("N,V,T,k", [
    (1, 1, 1.0, 1), (3, 2, 1.0, 2), (3, 7, 0.5, 7), (2, 8, 1.0, 0), (5, 100, 1.0, 100), (4, 257, 3.0, 256), (4, 1000, 1.0, 17),
    (3, 2047, 1.0, 1), (3, 5001, 0.8, 64), (2, 16384, 1.0, 200), (2, 16385, 1.0, 256), (3, 32769, 2.0, 0), (2, 65535, 1.0, 128),
    (2, 65536, 1.0, 20), (2, 65536, 0.1, 1), (301, 777, 1.0, 5)])
def test_token_logprobs(cuda, dtype, N, V, T, k):
    g = _gen(N, V, k)
    _check(cuda, _zipf(g, N, V).to(dtype), _tokens(g, N, V), T, k)


@DTYPES
@pytest.mark.parametrize("V", [9, 3000, 20000, 65536])
def test_likely_tokens(cuda, dtype, V):
    """Probabilities up to 1 - 1e-30: the rest of the row is what the log probability is made of."""
    g = _gen(V, 2)
    z = torch.randn(14, V, generator=g)
    t = torch.randint(0, V, (14,), generator=g)
    for i in range(14):
        z[i, t[i]] = 4.0 + 5.5 * i
    t[::3] = (t[::3] + 1) % V
    _check(cuda, z.to(dtype), t, 1.0, 3)


@DTYPES
@pytest.mark.parametrize("V", [40, 3000, 65536])
def test_masks_ties_and_nan(cuda, dtype, V):
    g = _gen(V, 3)
    N = 16
    z = torch.randn(N, V, generator=g)
    t = torch.randint(0, V, (N,), generator=g)
    z[0] = -INF                       # nothing left
    z[1, 1:] = -INF                   # one left, the token or not
    t[1] = 0
    z[2, 1:] = -INF
    t[2] = 5
    z[3, V // 3 :] = -INF             # a masked end
    z[4, ::2] = -INF
    t[4] = 1
    z[5] = 1.25                       # all alike
    z[6] = torch.randint(0, 2, (V,), generator=g).float()
    z[7, 3:9] = torch.finfo(dtype).min
    z[8] = torch.finfo(dtype).min     # masked by the lowest value throughout: uniform
    z[9] = torch.finfo(dtype).min
    z[9, 7] = 0.5
    t[9] = 7
    z[10, 4] = NAN
    z[11] = NAN
    z[12, 9] = INF
    z[13, 2], z[13, 3:] = NAN, -INF
    z[14] = torch.finfo(dtype).max
    z[15] = -INF
    t[15] = -1
    _check(cuda, z.to(dtype), t, 1.0, 6)
    pad = torch.full((N,), -1)
    for out in K.token_logprobs(z.to(dtype).to(cuda), pad.to(cuda)):
        assert (out == 0).all()
    assert (K.token_logprobs_grad(z.to(dtype).to(cuda), pad.to(cuda))[2] == 0).all()
    none = K.token_logprobs_grad(z.to(dtype).to(cuda), t.to(cuda), scale=0.0)[2]
    assert (none == 0).all()


@pytest.mark.parametrize("T", [1e-3, 30.0, 1e4])
@pytest.mark.parametrize("offset", [0.0, 1e4, -3e6])
def test_offsets_and_temperatures(cuda, T, offset):
    g = _gen(int(T * 1e3), int(offset), 4)
    z = _zipf(g, 4, 3001) * max(T, 1.0) + offset
    _check(cuda, z, _tokens(g, 4, 3001, 0.0), T, 4)


@DTYPES
def test_layouts(cuda, dtype):
    g = _gen(5)
    base = _zipf(g, 24, 2100).to(dtype).to(cuda)
    for z in (base[:, 3:2050], base[::2, 1:1000], base.t()[:, 2:], base[0, :50].expand(4, 50), base[:, 7:8]):
        t = _tokens(g, z.shape[0], z.shape[1]).to(cuda)
        k = min(5, z.shape[1])
        c = z.contiguous()
        want = K.token_logprobs(c, t, k) + K.token_logprobs_grad(c, t, entropy_scale=0.5)
        got = K.token_logprobs(z, t, k) + K.token_logprobs_grad(z, t, entropy_scale=0.5)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        rows = torch.full((z.shape[0],), 0.5, device=cuda)
        wide = torch.stack([rows, rows * 3], 1)[:, 0]
        assert torch.equal(K.token_logprobs_grad(z, t, scale=torch.ones_like(rows), entropy_scale=wide)[2], want[-1])
    t = _tokens(g, 24, 2100).to(cuda)
    lp, ent, top, idx = K.token_logprobs(base.view(2, 3, 4, 2100), t.view(2, 3, 4), 3)
    assert lp.shape == ent.shape == (2, 3, 4) and top.shape == idx.shape == (2, 3, 4, 3)
    flat = K.token_logprobs(base, t, 3)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip((lp, ent, top, idx), flat))
    lp, ent, grad = K.token_logprobs_grad(base[0], t[0] * 0 + 4)
    assert lp.shape == ent.shape == () and grad.shape == (2100,)
    lp, ent, top, idx = K.token_logprobs(base[:0], t[:0], 3)
    assert lp.shape == ent.shape == (0,) and top.shape == idx.shape == (0, 3)
    assert K.token_logprobs_grad(base[:0], t[:0])[2].shape == (0, 2100)


def test_agrees_with_top_logits_and_distill_loss(cuda):
    """The same order of alternatives; cross entropy is the divergence from a teacher of one entry."""
    g = _gen(6)
    z, t = _zipf(g, 30, 5003).to(B16).to(cuda), torch.randint(0, 5003, (30,), generator=g).to(cuda)
    v, i, lse = K.top_logits(z, 40)
    lp, _, top, idx = K.token_logprobs(z, t, 40)
    assert torch.equal(idx, i)
    assert (top.double() - (v.double() - lse.double()[:, None])).abs().max() < 112 * U + U * 40
    loss, grad = K.distill_loss_grad(z, z.gather(1, t[:, None]), t[:, None])
    got = K.token_logprobs_grad(z, t, scale=-1.0)
    assert (loss + got[0]).abs().max() < 112 * U + 2 * U * 40
    assert (grad.double() - got[2].double()).abs().max() <= 2.0**-8 * 1.01


def test_autograd(cuda):
    g = _gen(7)
    z = _zipf(g, 6, 5, 900).to(cuda).requires_grad_()
    t = _tokens(g, 30, 900).to(cuda).view(6, 5)
    s, h = torch.randn(6, 5, generator=g).to(cuda), torch.randn(6, 5, generator=g).to(cuda)
    lp, ent = ops.token_logprobs(z, t, 0.7)
    zero = torch.zeros_like(s)
    want = K.token_logprobs_grad(z.detach(), t, temperature=0.7, scale=s, entropy_scale=h)
    assert torch.equal(lp, want[0]) and torch.equal(ent, want[1])
    grad = lambda out, up: torch.autograd.grad(out, z, up, retain_graph=True)[0]  # noqa: E731
    assert torch.equal(grad((lp, ent), (s, h)), want[2])
    assert torch.equal(grad(lp, s), K.token_logprobs_backward(s, zero, z.detach(), t, 0.7))
    assert torch.equal(grad(ent, h), K.token_logprobs_backward(zero, h, z.detach(), t, 0.7))
    assert torch.equal(grad(lp.sum(), None), K.token_logprobs_grad(z.detach(), t, temperature=0.7)[2])
    two = torch.autograd.grad(lp, z, torch.stack([s, -s]), is_grads_batched=True, retain_graph=True)[0]
    assert torch.equal(two[0], grad(lp, s)) and torch.equal(two[1], -two[0])
    with pytest.raises(NotImplementedError, match="no second derivative"):
        (a,) = torch.autograd.grad((lp * lp).sum(), z, create_graph=True)
        torch.autograd.grad(a.sum(), z)
    with torch.no_grad():
        assert not ops.token_logprobs(z, t)[0].requires_grad


def test_gradients_match_differences(cuda):
    g = _gen(8)
    z = _zipf(g, 5, 300).to(cuda)
    t = _tokens(g, 5, 300, 0.0).to(cuda)
    s, h = torch.randn(5, generator=g).to(cuda), torch.randn(5, generator=g).to(cuda)
    f = lambda x: sum((a.double() * b.double()).sum() for a, b in zip(K.token_logprobs(x, t), (s, h)))  # noqa: E731
    grad = K.token_logprobs_grad(z, t, scale=s, entropy_scale=h)[2].double()
    for i in range(5):
        d = torch.randn(5, 300, generator=g).to(cuda)
        step = 2.0**-5
        diff = (8 * (f(z + step * d) - f(z - step * d)) - (f(z + 2 * step * d) - f(z - 2 * step * d))) / (12 * step)
        # ten values of about 5, each to 45 U, times 18 / 12 / step: 1.3e-3; the fifth derivative, 243 at d = 3, times
        # step^4 4 / 30: 3e-5 a row
        assert abs(float(diff - (grad * d.double()).sum())) < 2e-3


def test_rows_past_2_to_the_31_elements(cuda):
    N = 33600
    z = torch.zeros(N, 65536, dtype=H, device=cuda)
    hot = (torch.arange(N, device=cuda) * 7919) % 65536
    z[torch.arange(N, device=cuda), hot] = 3.0
    want = 3.0 - math.log(65535 + math.exp(3.0))
    lp, ent, top, idx = K.token_logprobs(z, hot, 1)
    assert torch.equal(idx[:, 0], hot) and torch.equal(top[:, 0], lp) and (lp - want).abs().max() < 60 * U * 12
    lp, ent, grad = K.token_logprobs_grad(z, hot)
    assert (lp - want).abs().max() < 60 * U * 12
    own = grad[torch.arange(N, device=cuda), hot].float()
    assert (own - (1 - math.exp(want))).abs().max() < 2.0**-11 and bool((grad != 0).all(1).all())


def test_more_rows_than_a_launch_has(cuda):
    N = (1 << 21) + 5
    z = torch.zeros(N, 3, dtype=H, device=cuda)
    hot = torch.arange(N, device=cuda) % 3
    z[torch.arange(N, device=cuda), hot] = 1.0
    want = 1 - math.log(math.e + 2)
    for lp in (K.token_logprobs(z, hot)[0], K.token_logprobs(z, hot, 2)[0], K.token_logprobs_grad(z, hot)[0]):
        assert (lp - want).abs().max() < 60 * U
    grad = K.token_logprobs_grad(z, hot)[2]
    assert torch.equal(grad.argmax(1), hot) and (grad.float().sum(1).abs() < 2e-3).all()


def test_graph_replays(cuda):
    g = _gen(9)
    z, t = _zipf(g, 20, 20011).to(B16).to(cuda), _tokens(g, 20, 20011).to(cuda)
    s = torch.randn(20, generator=g).to(cuda)

    def step():
        return K.token_logprobs(z, t, 9) + K.token_logprobs(z, t) + K.token_logprobs_grad(z, t, scale=s, entropy_scale=0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        z.copy_(_zipf(g, 20, 20011))
        t.copy_(_tokens(g, 20, 20011))
        s.neg_()
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda):
    z, t = torch.zeros(3, 20, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    for match, call in (
        ("int64", lambda: K.token_logprobs(z, t.int())),
        ("int64", lambda: K.token_logprobs(z, t[:2])),
        ("int64", lambda: K.token_logprobs(z, [0, 0, 0])),
        ("float16, bfloat16 or float32", lambda: K.token_logprobs(z.double(), t)),
        ("k must be", lambda: K.token_logprobs(z, t, -1)),
        ("k must be", lambda: K.token_logprobs(z, t, 21)),
        ("k must be", lambda: K.token_logprobs(z, t, 2.0)),
        ("k must be", lambda: K.token_logprobs(torch.zeros(3, 300, device=cuda), t, 257)),
        ("temperature", lambda: K.token_logprobs(z, t, temperature=0.0)),
        ("temperature", lambda: K.token_logprobs(z, t, temperature=NAN)),
        ("vocabulary", lambda: K.token_logprobs(torch.zeros(3, 65537, device=cuda), t)),
        ("tensors on", lambda: K.token_logprobs(z, t.cpu())),
        ("scale must be", lambda: K.token_logprobs_grad(z, t, scale=torch.zeros(2, device=cuda))),
        ("scale must be", lambda: K.token_logprobs_grad(z, t, scale=torch.zeros(3, device=cuda, dtype=torch.float64))),
        ("entropy_scale must be", lambda: K.token_logprobs_grad(z, t, entropy_scale=torch.zeros(3, 1, device=cuda))),
        ("tensors on", lambda: K.token_logprobs_grad(z, t, scale=torch.zeros(3))),
    ):
        with pytest.raises(ValueError, match=match):
            call()
