"""Embedding and LayerNorm with their gradients (``rwkv_tl_amd.training``) on the GPU,
against float64 on the CPU (``oracle.training_ref``).

Tolerances (U = 2^-24, half a step of float32; h = half a step of the stored type,
and 2^-25 where float16 has subnormals).

Embedding: one product in float32, then the stored type: equal bits. Gradient: n rows
are n additions and a factor: (n + 1) U sum |s dy|, and h of the value.

LayerNorm, of d = x - m about a first mean m, with xh the normalised value and D the
deviation. A sum over a row is at most 32 additions of a thread, 6 of a wave and 16
of the waves: 54 U, say 64 U, of its terms' sum. The differences' mean is so within
64 U D; the variance within 66 U of itself, the reciprocal deviation 34 U, say 40 U
with its own roundings. xh is off by U (40 |xh| + 64 + |xh|), y by |w| as much and U of
the sum, then h. Where the mean is many deviations, m itself is off by up to 64 U mean|x|,
which the differences' mean takes out again to 64 U of the differences: these are
larger by that much, the factor `far` below.

Gradient: c1 = mean g within 66 U mean |g|; c2 = mean g xh within U mean |g| (110 |xh| + 70),
from xh's 41 |xh| + 64 and the sum's 66; dx = r (g - c1 - xh c2) so within r U of
4 |g| + 70 mean |g| + |xh| mean |g| (110 |xh| + 70) + |c2| (45 |xh| + 70), and 40 U + h of
itself. dw: R additions of a wave's rows, 4 waves, the product and the rounded part: (R + 8) U sum
|dy xh| and xh's own error, U sum |dy| (41 |xh| + 64); db (R + 8) U sum |dy|; then h.
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


def _half(dtype, want):
    """Half a step of the stored type at each value."""
    return torch.finfo(dtype).eps / 2 * want.abs() + (2.0**-25 if dtype is H else 0.0)


def _within(got, want, bound):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} off, the worst by {float(((got - want).abs() / bound).nan_to_num(INF).max())} bounds"


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------


def _tokens(g, N, V, pad=0.1):
    """Low ids often; some ids outside the table."""
    t = ((torch.rand(N, generator=g).double() * math.log(V + 1)).exp() - 1).long().clamp(0, V - 1)
    out = torch.tensor([-1, V, -(2**40), 2**40 + 1, -100])
    return torch.where(torch.rand(N, generator=g) < pad, out[torch.randint(0, 5, (N,), generator=g)], t)


def _bits(x):
    return x.view({2: torch.int16, 4: torch.int32}[x.element_size()])


@DTYPES
@pytest.mark.parametrize("N,V,C,scale", [(1, 1, 1, 1.0), (1, 300, 2048, 1.0), (3, 7, 5, 0.3), (16, 1000, 768, 27.5), (65, 300, 1001, -1.7),
                                         (4, 2, 8200, 2.0), (1000, 65536, 8, 1.0), (257, 5000, 63, 1e-3)])
def test_embed(cuda, dtype, N, V, C, scale):
    g = _gen(N, V, C)
    w, t = torch.randn(V, C, generator=g).to(dtype), _tokens(g, N, V)
    got = K.embed(w.to(cuda), t.to(cuda), scale=scale).cpu()
    there = (t >= 0) & (t < V)
    want = torch.where(there[:, None], w[t.clamp(0, V - 1)].float() * torch.tensor(scale).float(), 0.0).to(dtype)
    assert got.dtype is dtype and torch.equal(_bits(got), _bits(want))
    if N * C < 1e5:
        _within(got, R.embed(w, t, float(torch.tensor(scale).float())), _half(dtype, want.double()) + U * want.double().abs())


@DTYPES
def test_embed_layouts(cuda, dtype):
    g = _gen(2)
    base = torch.randn(40, 101, generator=g).to(dtype).to(cuda)
    t = _tokens(g, 60, 20).to(cuda)
    for w in (base[:20, 1:], base[::2, 3:50], base.t()[:20], base[0].expand(20, 101)):  # odd offsets, strides, columns, one row
        want = K.embed(w.contiguous(), t)
        assert torch.equal(K.embed(w, t), want)
        assert torch.equal(K.embed(w, t.view(3, 4, 5)), want.view(3, 4, 5, -1))
        assert torch.equal(K.embed(w, torch.stack([t, t], 1)[:, 0]), want)
    assert K.embed(base, t[:0]).shape == (0, 101) and K.embed(base, t[0]).shape == (101,)
    assert K.embed(base, t[:0].view(0, 3)).shape == (0, 3, 101)
    w = torch.full((3, 5), INF, dtype=dtype, device=cuda)
    w[1, 2] = NAN
    got = K.embed(w, torch.tensor([0, 1, -1], device=cuda), scale=0.5)
    assert got[0].isinf().all() and got[1].isnan().tolist() == [False, False, True, False, False] and (got[2] == 0).all()


def _embed_grad_close(got, dy, t, V, scale):
    s = float(torch.tensor(scale).float())
    want = R.embed_grad(dy, t, V, s)
    size = R.embed_grad(dy.abs(), t, V, abs(s))
    n = torch.bincount(t[(t >= 0) & (t < V)], minlength=V).double()[:, None]
    _within(got, want, (n + 1) * U * size + _half(got.dtype, want) * (1 + n * U))


@DTYPES
@pytest.mark.parametrize("N,V,C,scale", [
    (1, 1, 1, 1.0), (1, 500, 768, 2.0), (7, 3, 5, 0.3), (64, 1, 9, 1.0), (65, 1, 513, 1.0), (64, 400, 100, 1.0), (65, 300, 33, 1.0),
    (129, 2, 1000, 1.0), (500, 17, 96, 1.0), (509, 2011, 768, 1.0), (1000, 257, 515, -0.5), (2048, 70000, 24, 1.0),
    (4096, 65536, 64, 1.0), (5000, 5, 40, 1.0), (20000, 1000, 16, 1.0)])
def test_embed_gradient(cuda, dtype, N, V, C, scale):
    g = _gen(N, V, C, 1)
    dy, t = torch.randn(N, C, generator=g).to(dtype), _tokens(g, N, V)
    got = K.embed_backward(dy.to(cuda), t.to(cuda), V, scale=scale)
    assert got.dtype is dtype
    _embed_grad_close(got, dy, t, V, scale)
    assert torch.equal(got, K.embed_backward(dy.to(cuda), t.to(cuda), V, scale=scale))


@pytest.mark.parametrize("V", [1, 300, 65536])
@pytest.mark.parametrize("N", [64, 65, 66, 128, 129, 4000, 17000, 40000])
def test_embed_gradient_of_one_token(cuda, N, V):
    """Every position the same token: a wave's share, several units, the most units a row has."""
    g = _gen(N, V, 2)
    dy, t = torch.randn(N, 24, generator=g), torch.full((N,), V // 2)
    got = K.embed_backward(dy.to(cuda), t.to(cuda), V)
    want = torch.zeros(V, 24, dtype=torch.float64)
    want[V // 2] = dy.double().sum(0)
    _within(got, want, (N + 1) * U * dy.double().abs().sum(0) * (torch.arange(V) == V // 2)[:, None] + U * want.abs())


@pytest.mark.parametrize("counts", [[63, 64, 65, 66], [65] * 40, [96, 97, 127, 128, 129, 192, 193], [1, 2, 3, 700, 64, 0, 5, 1300, 65]], ids=str)
@pytest.mark.parametrize("step", [1, 256], ids=["neighbours", "one workgroup"])
def test_embed_gradient_counts(cuda, counts, step):
    """Rows about the length at which a row is split, of neighbouring workgroups and of one."""
    g = _gen(len(counts), step, 3)
    ids = torch.arange(len(counts)) * step + 7
    t = torch.repeat_interleave(ids, torch.tensor(counts))
    t = t[torch.randperm(t.numel(), generator=g)]
    V = int(ids[-1]) + 3
    dy = torch.randn(t.numel(), 40, generator=g).to(B16)
    _embed_grad_close(K.embed_backward(dy.to(cuda), t.to(cuda), V), dy, t, V, 1.0)


@pytest.mark.parametrize("counts", [[993, 2, 1], [4097, 3, 1], [5000, 1, 1, 1], "all"], ids=str)
@pytest.mark.parametrize("step", [1, 256], ids=["neighbours", "one workgroup"])
def test_embed_gradient_units_before_short_rows(cuda, counts, step):
    """Rows of every length that is cut, each before one of a single position: a row's last part is never taken for a row."""
    g = _gen(step, 20)
    if counts == "all":
        counts = [c for n in (range(33, 1100) if step == 1 else range(33, 200)) for c in (n, 1)]
    ids = torch.arange(len(counts)) * step
    t = torch.repeat_interleave(ids, torch.tensor(counts))
    t = t[torch.randperm(t.numel(), generator=g)]
    V = int(ids[-1]) + 1
    dy = torch.randint(-8, 9, (t.numel(), 8), generator=g).float()
    want = torch.zeros(V, 8).index_add_(0, t, dy)
    assert torch.equal(K.embed_backward(dy.to(cuda), t.to(cuda), V).cpu(), want)


def test_embed_gradient_adds_whole_numbers_exactly(cuda):
    """Sums of whole numbers have one value whatever their order: no row is left out or taken twice."""
    g = _gen(4)
    N, V, C = 30000, 3000, 72
    t = _tokens(g, N, V, 0.02)
    dy = torch.randint(-8, 9, (N, C), generator=g).float()
    want = torch.zeros(V + 1, C).index_add_(0, torch.where((t >= 0) & (t < V), t, V), dy)[:V]
    assert torch.equal(K.embed_backward(dy.to(cuda), t.to(cuda), V).cpu(), want)


def test_embed_gradient_of_the_largest_table(cuda):
    """2^20 rows: sixteen times the workgroups, rows far apart."""
    g = _gen(18)
    V, C = 2**20, 5
    t = torch.cat([torch.randint(0, V, (3000,), generator=g), torch.tensor([0, V - 1, V, -1]), torch.full((200,), V - 4097)])
    dy = torch.randint(-8, 9, (t.numel(), C), generator=g).float()
    want = torch.zeros(V + 1, C).index_add_(0, torch.where((t >= 0) & (t < V), t, V), dy)[:V]
    assert torch.equal(K.embed_backward(dy.to(cuda), t.to(cuda), V).cpu(), want)
    w = torch.randn(V, C, generator=g)
    assert torch.equal(K.embed(w.to(cuda), t[:3002].to(cuda)).cpu(), w[t[:3002]])


@DTYPES
def test_embed_gradient_layouts(cuda, dtype):
    g = _gen(5)
    base = torch.randn(300, 205, generator=g).to(dtype).to(cuda)
    t = _tokens(g, 100, 3).to(cuda)
    for dy in (base[:100, 1:], base[::3, 4:60], base.t()[:100, 2:], base[3].expand(100, 205), base[0, 0].expand(100, 31)):
        want = K.embed_backward(dy.contiguous(), t, 3)
        assert torch.equal(K.embed_backward(dy, t, 3), want)
        shaped = K.embed_backward(dy.reshape(2, 50, -1), t.view(2, 50), 3)
        assert torch.equal(shaped, want)
    assert torch.equal(K.embed_backward(base[:0], t[:0], 4), torch.zeros(4, 205, dtype=dtype, device=cuda))
    assert torch.equal(K.embed_backward(base[0], t[0] * 0 + 2, 4)[2], base[0])
    none = torch.full((100,), -1, device=cuda)
    assert (K.embed_backward(base[:100] * NAN, none, 500) == 0).all()


def test_embed_gradient_leaves_other_rows_alone(cuda):
    """NaN and infinities stay in their token's row."""
    dy = torch.ones(200, 64, device=cuda)
    t = torch.arange(200, device=cuda) % 2 * 5
    dy[3] = NAN
    dy[4, 7] = INF
    got = K.embed_backward(dy, t, 9)
    assert got[5].isnan().all() and got[0, 7] == INF and (got[0, :7] == 100).all() and (got[[1, 2, 3, 4, 6, 7, 8]] == 0).all()


# ---------------------------------------------------------------------------
# LayerNorm
# ---------------------------------------------------------------------------


def _norm_bounds(x, w, b, eps=1e-5):
    d = x.double()
    C = x.shape[-1]
    y, mean, rstd = R.layer_norm(x, w, b, eps)
    one, zero = torch.ones(C).double(), torch.zeros(C).double()
    xh = R.layer_norm(x, one, zero, eps)[0]
    dev = (d - mean[..., None]).abs().mean(-1)
    far = 1 + 64 * U * d.abs().mean(-1) * rstd  # how much larger the differences about the first mean are
    xerr = U * (41 * xh.abs() + 64) * far[..., None] ** 2
    return y, mean, rstd, xh, dev, far, xerr


def _check_norm(cuda, x, w, b, eps=1e-5):
    got = K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda), eps=eps)
    y, mean, rstd, xh, dev, far, xerr = _norm_bounds(x, w, b, eps)
    assert got[0].dtype is x.dtype and got[1].dtype is got[2].dtype is F
    _within(got[0], y, w.double().abs() * xerr + 2 * U * (y.abs() + b.double().abs()) + _half(x.dtype, y))
    _within(got[1], mean, 64 * U * dev * far**2 + 2 * U * mean.abs())
    _within(got[2], rstd, 40 * U * rstd * far**2)
    return got


def _check_norm_grad(cuda, x, w, b, dy, eps=1e-5, rows_per_wave=None):
    _, mean, rstd, xh, dev, far, xerr = _norm_bounds(x, w, b, eps)
    _, m, r = K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda), eps=eps)
    got = K.layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), m, r)
    gx, gw, gb = R.layer_norm_grad(dy, x, w, eps)
    g = (dy.double() * w.double()).abs()
    gm, gxm = g.mean(-1, keepdim=True), (g * xh.abs()).mean(-1, keepdim=True)
    ax, f2 = xh.abs(), far[..., None] ** 2
    bound = rstd[..., None] * U * f2 * (4 * g + 70 * gm + ax * (110 * gxm + 70 * gm) + gxm * (45 * ax + 70)) + 40 * U * f2 * gx.abs()
    _within(got[0], gx, bound + _half(x.dtype, gx))
    C = x.shape[-1]
    flat = lambda v: v.reshape(-1, C)  # noqa: E731
    ad, N = flat(dy.double().abs()), flat(x).shape[0]
    Rw = N // 512 + 1  # rows of a wave, of 512 workgroups
    _within(got[1], gw, (Rw + 8) * U * (ad * flat(ax)).sum(0) + (ad * flat(xerr)).sum(0) + _half(w.dtype, gw))
    _within(got[2], gb, (Rw + 8) * U * ad.sum(0) + _half(w.dtype, gb))
    assert [v.dtype for v in got] == [x.dtype, w.dtype, w.dtype]
    again = K.layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), m, r)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    return got


def _norm_inputs(g, N, C, dtype, wdtype):
    x = (torch.randn(N, C, generator=g) * (torch.randn(C, generator=g) * 0.6).exp() + torch.randn(C, generator=g)).to(dtype)
    w, b = (1 + 0.2 * torch.randn(C, generator=g)).to(wdtype), torch.randn(C, generator=g).to(wdtype)
    return x, w, b, torch.randn(N, C, generator=g).to(dtype)


@pytest.mark.parametrize("dtype,wdtype", [(H, H), (H, F), (B16, B16), (B16, F), (F, F)], ids=str)
@pytest.mark.parametrize("N,C", [
    (1, 1), (3, 2), (2, 7), (5, 8), (4, 9), (9, 63), (1, 64), (2, 511), (7, 512), (3, 513), (6, 768), (5, 1001), (3, 1024), (4, 1025),
    (7, 2048), (3, 2049), (2, 4096), (3, 4099), (2, 8192), (3, 8193), (2, 16384), (700, 40), (5000, 72), (2100, 1030)])
def test_layer_norm(cuda, dtype, wdtype, N, C):
    x, w, b, dy = _norm_inputs(_gen(N, C, 6), N, C, dtype, wdtype)
    _check_norm(cuda, x, w, b)
    _check_norm_grad(cuda, x, w, b, dy)


@pytest.mark.parametrize("dtype,wdtype", [(H, H), (B16, F), (F, F)], ids=str)
@pytest.mark.parametrize("C", [520, 1000, 1032, 2040, 2056, 4088, 4104, 8184, 8200, 16376])
def test_layer_norm_whole_eights_of_some_threads(cuda, dtype, wdtype, C):
    """Multiples of 8 channels that leave threads without any, in rows of any alignment."""
    x, w, b, dy = _norm_inputs(_gen(C, 11), 5, C, dtype, wdtype)
    x, dy = (torch.cat((v, v[:, :3]), 1)[:, 3:] for v in (x, dy))  # rows of C + 3, from the fourth channel
    _check_norm(cuda, x, w, b)
    _check_norm_grad(cuda, x, w, b, dy)


@pytest.mark.parametrize("eps", [1e-12, 1e-5, 64e-5, 3.0, 1e6])
def test_layer_norm_eps(cuda, eps):
    x, w, b, dy = _norm_inputs(_gen(7), 6, 300, F, F)
    x[1] = 0.25  # no deviation
    x[2] *= 1e-6
    x[3] *= 1e6
    _check_norm(cuda, x, w, b, eps)
    _check_norm_grad(cuda, x, w, b, dy, eps)


@pytest.mark.parametrize("C", [100, 1500, 9000])
def test_layer_norm_far_means(cuda, C):
    """Means many times the deviation."""
    g = _gen(C, 8)
    x = torch.randn(4, C, generator=g) + torch.tensor([10.0, -1e3, 3e4, -1e5])[:, None]
    w, b, dy = torch.randn(C, generator=g), torch.randn(C, generator=g), torch.randn(4, C, generator=g)
    _check_norm(cuda, x, w, b)
    _check_norm_grad(cuda, x, w, b, dy)


@pytest.mark.parametrize("dtype", [B16, F], ids=str)
@pytest.mark.parametrize("C", [50, 2048, 5000])
def test_layer_norm_of_any_size(cuda, dtype, C):
    """From values whose squares are 0 in float32 to the type's largest."""
    g = _gen(C, 9)
    x = torch.randn(8, C, generator=g).clamp(-3, 3) * torch.tensor([1e-30, 1e-10, 1e10, 1e15, 1e16, 1e25, 1e37, 1e38])[:, None]
    x[7, 0::2], x[7, 1::2] = torch.finfo(dtype).max, torch.finfo(dtype).min
    x = x.to(dtype)
    w, b, dy = torch.randn(C, generator=g), torch.randn(C, generator=g), torch.randn(8, C, generator=g).to(dtype)
    _check_norm(cuda, x, w, b)
    _check_norm_grad(cuda, x[:6], w, b, dy[:6])  # (of the others grad_x is subnormal)
    _, m, r = K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda))
    gx, gw, gb = K.layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), m, r)
    want = R.layer_norm_grad(dy, x, w)
    assert gx.isfinite().all()
    # (a reciprocal deviation of 2^-128, the least of float32, is stored to 2^-149: 2^-22, 4 U, more for xh)
    xh = R.layer_norm(x, torch.ones(C), torch.zeros(C))[0]
    ad = dy.double().abs()
    _within(gw, want[1], U * (ad * (55 * xh.abs() + 64)).sum(0) + U * want[1].abs())
    _within(gb, want[2], 10 * U * ad.sum(0))


def test_layer_norm_nan_and_infinity_stay_in_their_row(cuda):
    x, w, b, dy = _norm_inputs(_gen(10), 6, 700, F, F)
    x[1, 5], x[3, 0], x[4, 699] = NAN, INF, -INF
    y, m, r = K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda))
    bad = torch.tensor([1, 3, 4])
    good = torch.tensor([0, 2, 5])
    assert y[bad].isnan().all() and m[bad].logical_not().sum() == 0 and r[bad].isnan().all()
    assert torch.equal(y[good], K.layer_norm_forward(x[good].to(cuda), w.to(cuda), b.to(cuda))[0])
    gx, gw, _ = K.layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), m, r)
    assert gx[bad].isnan().all() and gx[good].isfinite().all() and gw.isnan().all()


@DTYPES
def test_layer_norm_layouts(cuda, dtype):
    g = _gen(11)
    base, other = (torch.randn(60, 130, generator=g).to(dtype).to(cuda) for _ in range(2))
    for cut in (lambda t: t[:, 1:100], lambda t: t[::3, 5:], lambda t: t.t()[:, 2:], lambda t: t[4].expand(7, 130), lambda t: t[:, :1]):
        x, dy = cut(base), cut(other)
        C = x.shape[-1]
        w, b = torch.randn(2 * C, device=cuda)[::2], torch.randn(C, device=cuda)
        want = K.layer_norm_forward(x.contiguous(), w.contiguous(), b)
        got = K.layer_norm_forward(x, w, b)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        gwant = K.layer_norm_backward(dy.contiguous(), x.contiguous(), w.contiguous(), *want[1:])
        assert all(torch.equal(p, q) for p, q in zip(K.layer_norm_backward(dy, x, w, *want[1:]), gwant))
    w, b = torch.ones(130, device=cuda), torch.zeros(130, device=cuda)
    y, m, r = K.layer_norm_forward(base.view(3, 20, 130), w, b)
    assert y.shape == (3, 20, 130) and m.shape == r.shape == (3, 20)
    y, m, r = K.layer_norm_forward(base[0], w, b)
    assert y.shape == (130,) and m.shape == r.shape == ()
    assert [t.shape for t in K.layer_norm_backward(other[0], base[0], w, m, r)] == [(130,)] * 3
    y, m, r = K.layer_norm_forward(base[:0], w, b)
    gx, gw, gb = K.layer_norm_backward(other[:0], base[:0], w, m, r)
    assert y.shape == gx.shape == (0, 130) and m.shape == (0,) and (gw == 0).all() and (gb == 0).all()


def test_layer_norm_agrees_with_the_inference_operator(cuda):
    x, w, b, _ = _norm_inputs(_gen(12), 9, 768, F, F)
    a, c = K.layer_norm(x.to(cuda), w.to(cuda), b.to(cuda)), K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda))[0]
    y, *_, xerr = _norm_bounds(x, w, b)
    _within(a - c, torch.zeros_like(y), 2 * (w.double().abs() * xerr + 3 * U * (y.abs() + b.double().abs())))


def test_rows_past_2_to_the_31_elements(cuda):
    """Row offsets past 32 bits, of inputs and outputs."""
    N, C = 140000, 16384
    x = torch.zeros(N, C, dtype=B16, device=cuda)
    rows = torch.tensor([0, 70000, 131071, 131072, 139999], device=cuda)
    x[rows, 5] = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0], dtype=B16, device=cuda)
    w, b = torch.ones(C, device=cuda), torch.zeros(C, device=cuda)
    y, m, r = K.layer_norm_forward(x, w, b)
    want = K.layer_norm_forward(x[rows], w, b)
    assert all(torch.equal(p[rows], q) for p, q in zip((y, m, r), want)) and int((y != 0).any(1).sum()) == 5
    gx = K.layer_norm_backward(x, x, w, m, r)[0]
    assert torch.equal(gx[rows], K.layer_norm_backward(x[rows], x[rows], w, *want[1:])[0]) and int((gx != 0).any(1).sum()) == 5
    del gx, y
    t = torch.full((N,), -1, device=cuda)
    t[rows] = torch.tensor([3, 1, 3, 0, 1], device=cuda)
    dw = K.embed_backward(x, t, 4)
    assert dw[:, 5].tolist() == [4.0, 7.0, 0.0, 4.0] and int((dw != 0).sum()) == 3
    got = K.embed(x, rows)
    assert torch.equal(got, x[rows])


# ---------------------------------------------------------------------------
# as a program has them
# ---------------------------------------------------------------------------


@DTYPES
def test_autograd(cuda, dtype):
    g = _gen(13)
    w = torch.randn(50, 96, generator=g).to(dtype).to(cuda).requires_grad_()
    t = _tokens(g, 40, 50).to(cuda).view(5, 8)
    ln = [torch.randn(96, generator=g).to(cuda).requires_grad_() for _ in range(2)]
    dy = torch.randn(5, 8, 96, generator=g).to(dtype).to(cuda)
    x = ops.embed(w, t, 1.5)
    y = ops.layer_norm(x, *ln, 1e-4)
    got = torch.autograd.grad(y, (w, *ln), dy)
    y0, m, r = K.layer_norm_forward(K.embed(w.detach(), t, scale=1.5), *(v.detach() for v in ln), eps=1e-4)
    gx, gw, gb = K.layer_norm_backward(dy, x.detach(), ln[0].detach(), m, r)
    assert torch.equal(y, y0)
    assert torch.equal(got[0], K.embed_backward(gx, t, 50, scale=1.5)) and torch.equal(got[1], gw) and torch.equal(got[2], gb)
    # parameters, as modules have them
    params = [torch.nn.Parameter(v.detach()) for v in (w, *ln)]
    again = torch.autograd.grad(ops.layer_norm(ops.embed(params[0], t, 1.5), *params[1:], 1e-4), params, dy)
    assert all(torch.equal(a, b) for a, b in zip(again, got))
    # one of the inputs alone, and none
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x.detach(), ln[0].detach(), ln[1], 1e-4), ln[1], dy)[0], gb)
    with torch.no_grad():
        assert not ops.layer_norm(ops.embed(w, t), *ln).requires_grad
    # a gradient that is one number for all, and batches of gradients
    (one,) = torch.autograd.grad(ops.embed(w, t).sum(), w)
    assert torch.equal(one, K.embed_backward(torch.ones(5, 8, 96, dtype=dtype, device=cuda), t, 50))
    y = ops.embed(w, t, 1.5)
    two = torch.autograd.grad(y, w, torch.stack([dy, -dy]), is_grads_batched=True)[0]
    assert torch.equal(two[0], K.embed_backward(dy, t, 50, scale=1.5)) and torch.equal(two[1], -two[0])
    with pytest.raises(NotImplementedError, match="no second derivative"):
        y = ops.layer_norm(x, *ln)
        (a,) = torch.autograd.grad((y.float() ** 2).sum(), x, create_graph=True)
        torch.autograd.grad(a.float().sum(), ln[0])


def test_traced(cuda):
    """Through torch.compile, whole and with its gradients: the operators, not their kernels, are traced."""
    g = _gen(19)
    w = torch.randn(60, 64, generator=g).to(cuda).requires_grad_()
    ln = [torch.randn(64, generator=g).to(cuda).requires_grad_() for _ in range(2)]
    t = _tokens(g, 30, 60).to(cuda)

    def f(w, a, b, t):
        x = ops.layer_norm(ops.embed(w, t, 1.5), a, b)
        lp, H = ops.token_logprobs(x @ w.t(), t)
        return lp.sum() + 0.1 * H.sum()

    want = f(w, *ln, t)
    grads = torch.autograd.grad(want, (w, *ln))
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(w, *ln, t)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, (w, *ln)), grads):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-6)  # (the table's two gradients are added in either order)


def test_gradients_match_differences(cuda):
    g = _gen(14)
    w = torch.randn(12, 40, generator=g).to(cuda)
    t = torch.tensor([3, 3, 5, -1, 11, 0, 3], device=cuda)
    ln = [torch.randn(40, generator=g).to(cuda) for _ in range(2)]
    proj = torch.randn(7, 40, generator=g).double().to(cuda)
    leaves = [v.clone().requires_grad_() for v in (w, *ln)]

    def f(a, b, c):
        return (ops.layer_norm(ops.embed(a, t, 2.0), b, c).double() * proj).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    for i, (v, gr) in enumerate(zip((w, *ln), grads)):
        d = torch.randn(v.shape, generator=g).to(cuda)
        step = 2.0**-6
        at = lambda s: f(*(u + s * d if j == i else u for j, u in enumerate((w, *ln))))  # noqa: E731
        # the fourth difference: an error of step^4 times the fifth derivative; 280 values to 35 U, times 18 / 12 / step: 0.06
        diff = (8 * (at(step) - at(-step)) - (at(2 * step) - at(-2 * step))) / (12 * step)
        want = (gr.double() * d.double()).sum()
        assert abs(float(diff - want)) < 1e-3 * float((gr.double() * d.double()).abs().sum()) + 0.06


def test_graph_replays(cuda):
    """A step captured once and replayed on other inputs, eager work between the replays."""
    g = _gen(15)
    w = torch.randn(300, 128, generator=g).to(cuda)
    t = _tokens(g, 500, 300).to(cuda)
    ln = [torch.randn(128, generator=g).to(cuda) for _ in range(2)]
    dy = torch.randn(500, 128, generator=g).to(cuda)

    def step():
        x = K.embed(w, t)
        y, m, r = K.layer_norm_forward(x, *ln)
        gx, gw, gb = K.layer_norm_backward(dy, x, ln[0], m, r)
        return y, gw, gb, K.embed_backward(gx, t, 300)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        t.copy_(_tokens(g, 500, 300, 0.3) if i < 2 else torch.full((500,), i))
        dy.copy_(torch.randn(500, 128, generator=g))
        w.mul_(1.25)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_streams(cuda):
    g = _gen(16)
    w, t = torch.randn(500, 256, generator=g).to(cuda), _tokens(g, 3000, 500).to(cuda)
    dy = torch.randn(3000, 256, generator=g).to(cuda)
    want = K.embed_backward(dy, t, 500)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two calls at once, each with its own workspace
        with torch.cuda.stream(s):
            got.append((K.embed_backward(dy, t, 500), K.embed(w, t), K.layer_norm_forward(dy, w[0], w[1])))
    torch.cuda.synchronize()
    assert torch.equal(got[0][0], want) and torch.equal(got[1][0], want) and torch.equal(got[0][1], got[1][1])
    assert all(torch.equal(a, b) for a, b in zip(got[0][2], got[1][2]))


def test_refusals(cuda):
    w, t = torch.zeros(10, 8, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    dy = torch.zeros(3, 8, device=cuda)
    row = torch.zeros(3, device=cuda)
    c = torch.zeros(8, device=cuda)
    z = lambda *s, **k: torch.zeros(*s, device=cuda, **k)  # noqa: E731
    for match, call in (
        ("int64", lambda: K.embed(w, t.int())),
        ("must be", lambda: K.embed(w.double(), t)),
        (r"\[V, C\]", lambda: K.embed(w[0], t)),
        ("a table", lambda: K.embed(z(0, 8), t)),
        ("a table", lambda: K.embed(z(4, 0), t)),
        ("scale", lambda: K.embed(w, t, scale=NAN)),
        ("scale", lambda: K.embed(w, t, scale=1e39)),
        ("tensors on", lambda: K.embed(w, t.cpu())),
        ("grad must be", lambda: K.embed_backward(dy, t[:2], 10)),
        ("grad must be", lambda: K.embed_backward(dy[:, None], t, 10)),
        ("a table", lambda: K.embed_backward(dy, t, 0)),
        ("a table", lambda: K.embed_backward(dy, t, 2**20 + 1)),
        ("vocab", lambda: K.embed_backward(dy, t, 10.0)),
        ("channels", lambda: K.layer_norm_forward(z(2, 16385), z(16385), z(16385))),
        ("channels", lambda: K.layer_norm_forward(z(2, 0), z(0), z(0))),
        ("channels", lambda: K.layer_norm_forward(z(()), c, c)),
        ("weight must be", lambda: K.layer_norm_forward(dy, c[:7], c)),
        ("bias must be", lambda: K.layer_norm_forward(dy, c, c.half())),
        ("weight must be", lambda: K.layer_norm_forward(dy, c.half(), c.half())),
        ("eps", lambda: K.layer_norm_forward(dy, c, c, eps=0.0)),
        ("eps", lambda: K.layer_norm_forward(dy, c, c, eps=NAN)),
        ("grad_y must be", lambda: K.layer_norm_backward(dy.half(), dy, c, row, row)),
        ("grad_y must be", lambda: K.layer_norm_backward(dy[:2], dy, c, row, row)),
        ("mean must be", lambda: K.layer_norm_backward(dy, dy, c, row[:2], row)),
        ("rstd must be", lambda: K.layer_norm_backward(dy, dy, c, row, row.double())),
        ("tensors on", lambda: K.layer_norm_backward(dy, dy, c, row, row.cpu())),
    ):
        with pytest.raises(ValueError, match=match):
            call()


def test_a_training_step(cuda):
    """Tokens to logits to their log probabilities and back: embedding, norm, DPLR sequence, norm, head, against float64
    with the recurrence's own gradient taken from the operator under test elsewhere."""
    g = _gen(17)
    B, T, Hh, V = 2, 33, 2, 200
    C = Hh * 64
    p = {
        "emb": torch.randn(V, C, generator=g) * 0.5, "w1": 1 + 0.1 * torch.randn(C, generator=g), "b1": 0.1 * torch.randn(C, generator=g),
        "w2": 1 + 0.1 * torch.randn(C, generator=g), "b2": 0.1 * torch.randn(C, generator=g), "head": torch.randn(V, C, generator=g) * 0.1}
    t = torch.randint(0, V, (B, T + 1), generator=g)
    t[1, 20:] = -1  # a shorter sequence
    decay = torch.rand(B, T, Hh, 64, generator=g) * 0.5 + 0.5
    leaves = {k: v.to(cuda).requires_grad_() for k, v in p.items()}

    def step(q, embed, norm, logprobs, dev, dt):
        x = norm(embed(q["emb"], t[:, :-1].to(dev)), q["w1"], q["b1"])
        h = x.view(B, T, Hh, 64)
        kk = torch.nn.functional.normalize(h, dim=-1)
        S = torch.zeros(B, Hh, 64, 64, dtype=dt, device=dev)
        args = (h, decay.to(dt).to(dev), h * 0.2, h * 0.3, -kk, kk * 0.5)
        if dt is F:
            y, _ = ops.fused_dplr_seq(S, *args)
        else:
            ys = []
            for i in range(T):
                r, w, k, v, a, b = (u[:, i] for u in args)
                S = S * w[..., None, :] + (S @ a[..., None]) * b[..., None, :] + v[..., None] * k[..., None, :]
                ys.append((S @ r[..., None])[..., 0])
            y = torch.stack(ys, 1)
        z = norm(x + y.reshape(B, T, C), q["w2"], q["b2"]) @ q["head"].t()
        lp, ent = logprobs(z, t[:, 1:].to(dev))
        n = (t[:, 1:] >= 0).sum()
        return -(lp.sum() + 0.01 * ent.sum()) / n

    def norm64(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return d / ((d * d).mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    def embed64(w, i):
        return torch.where((i >= 0)[..., None], w[i.clamp_min(0)], 0.0)

    loss = step(leaves, ops.embed, ops.layer_norm, ops.token_logprobs, cuda, F)
    grads = torch.autograd.grad(loss, list(leaves.values()))
    ref = {k: v.double().requires_grad_() for k, v in p.items()}
    want = step(ref, embed64, norm64, R.token_logprobs, torch.device("cpu"), torch.float64)
    refs = torch.autograd.grad(want, list(ref.values()))
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5 * float(want.detach())
    for k, a, b in zip(p, grads, refs):  # (33 steps of a recurrence in float32 between: 1e-4 of the gradient's size)
        assert float((a.double().cpu() - b).norm() / b.norm()) < 1e-4, k
