"""LayerNorm (``rwkv_tl_amd.training``) of rows without a deviation, on the GPU, against closed forms.

A row of one value x has the mean x, no deviation, and the reciprocal deviation eps^-1/2: y is the bias, bit for bit;
dx = eps^-1/2 (g - mean g); the weight's gradient is 0 and the bias's the sum of dy. U = 2^-24 is half a step of float32.
mean and y are exact, rstd within 2 U (its rounding, and that of the estimate's refinement). Sums over a row are at
most 54 additions of a thread, a wave and the waves: mean g within 56 U mean |g|, dx so within rstd (2 U |g| + 58 U mean
|g|), 3 U of itself and half a step of the stored type.
"""

from __future__ import annotations

import pytest
import torch

import rwkv_tl_amd  # noqa: F401
from rwkv_tl_amd import kernels as K

pytestmark = pytest.mark.gpu
H, B16, F = torch.float16, torch.bfloat16, torch.float32
U = 2.0**-24


def _gen(*key):
    return torch.Generator().manual_seed(sum((i + 3) * 1009**i * k for i, k in enumerate(key)) % (1 << 40))


def _bits(x):
    return x.view({2: torch.int16, 4: torch.int32}[x.element_size()])


def _within(got, want, bound):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} off, the worst by {float(((got - want).abs() / bound).max())} bounds"


def _check_one_value(cuda, values, C, dtype, eps=1e-5):
    """A row for each value, forward and gradient."""
    x = torch.tensor(values, dtype=torch.float64).to(dtype)[:, None].expand(-1, C).contiguous()
    assert x.isfinite().all()
    g = _gen(len(values), C)
    w, b, dy = torch.randn(C, generator=g), torch.randn(C, generator=g), torch.randn(len(values), C, generator=g).to(dtype)
    y, mean, rstd = K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda), eps=eps)
    assert torch.equal(_bits(y.cpu()), _bits(b.to(dtype).expand_as(y)))
    assert torch.equal(mean.cpu(), x[:, 0].float())
    one = torch.tensor(eps, dtype=torch.float64) ** -0.5
    _within(rstd, one.expand(len(values)), 2 * U * one)
    gx, gw, gb = K.layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), mean, rstd)
    q = dy.double() * w.double()
    want = one * (q - q.mean(-1, keepdim=True))
    half = torch.finfo(dtype).eps / 2 * want.abs() + (2.0**-25 if dtype is H else 0.0)
    bound = one * U * (2 * q.abs() + 58 * q.abs().mean(-1, keepdim=True)) + 3 * U * want.abs() + half
    # (float16 ends at 65504: from half a step above it, 65520, a value is infinite)
    past = gx.cpu().isinf() & (want.abs() + bound >= torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)) & (gx.cpu() * want > 0)
    _within(torch.where(past.to(cuda), 0.0, gx.double()), torch.where(past, 0.0, want), bound)
    assert (gw == 0).all()
    _within(gb, dy.double().sum(0), len(values) * U * dy.double().abs().sum(0))


@pytest.mark.parametrize("dtype", [B16, F], ids=str)
@pytest.mark.parametrize("C", [3, 100, 768, 1001, 1500, 2048, 4096, 5001, 9999, 16384])
def test_rows_of_one_value_whose_sum_passes_float32(cuda, dtype, C):
    _check_one_value(cuda, [3e38, -3e38, torch.finfo(dtype).max, torch.finfo(dtype).min], C, dtype)
    _check_one_value(cuda, [3e38, torch.finfo(dtype).min], C, dtype, 1e-30)
    _check_one_value(cuda, [3e38, torch.finfo(dtype).min], C, dtype, 1e6)

def _exact_rows(units, size):
    """Rows of size * (2^23 + units), size a power of two: float32 neighbours, with what float64 has of them exactly."""
    x = ((2.0**23 + units.double()) * size).float()
    assert torch.equal(x.double(), (2.0**23 + units.double()) * size)
    near = units.double() - units[:, 2:3].double()
    d = (near - near.mean(-1, keepdim=True)) * size
    return x, d, (d * d).mean(-1)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("C", [41, 110, 165, 427, 660, 1473, 1699, 1857, 2606, 7680, 8186, 12729, 13141, 14030, 15688, 16113])
def test_rows_of_one_value(cuda, dtype, C):
    """Also where the row's first mean is some roundings beside the value: those are no deviation."""
    far = [float(torch.tensor(2.0**k * f)) for k in range(10, 76 if dtype is not H else 15) for f in (1.0, 1.171875, 1.7265625)]
    near = [0.0, -0.0, 0.1, -1.0, 3.3, 1000.1]
    if dtype is F:  # a few of those whose first mean was off
        far += [27381108.0, 1298594200.0, 4706949700000.0, 2334959000000.0, 2.7584979e17, 1.3984066e19, 4.9142143e13, 2.5621844e16,
                4.7746643e20, 1.1452193e16, 4.3576782e18, 2.4010826e17, 13705251000000.0, 1.590149e11, 8.714119e18]
    _check_one_value(cuda, far + near, C, dtype)
    _check_one_value(cuda, near, C, dtype, 1e-12)


@pytest.mark.parametrize("C", [3, 100, 770, 1001, 2040, 5001, 9999, 16384])
@pytest.mark.parametrize("size", [2.0**-20, 1.0, 2.0**30, 2.0**60])
def test_rows_of_neighbouring_values(cuda, C, size):
    """Deviations of a step of float32 and less: from one value that is a step beside the others to several steps.

    The mean that the differences are formed about is the row's to half a step; or its rounding e is no more than four
    times the deviation D, f = e / D: then too. A sum is within 54 U, say 56 U with the factor 1 / C, of its terms':
    the mean of the differences within 56 U sqrt(1 + f^2) D, the variance within 3 times 56 U (1 + f^2) of itself and the
    reciprocal deviation within 84 U (1 + f^2) and its own 2 U. A normalised value so within U (86 (1 + f^2) |xh| +
    57 sqrt(1 + f^2)), U of the difference; the gradient's sums about the stored mean, half a step from the row's, alike."""
    g = _gen(C, 2)
    units = torch.stack([torch.zeros(C), torch.zeros(C), torch.zeros(C), torch.randint(0, 2, (C,), generator=g).float(),
                         torch.randint(-1, 2, (C,), generator=g).float(), torch.randint(-40, 41, (C,), generator=g).float()])
    units[0, 0], units[1, C // 2], units[2, C - 1], units[3, 0], units[3, 1] = 1, -1, 5, 0, 1
    units[4, :2], units[5, :2] = torch.tensor([0.0, 1.0]), torch.tensor([-9.0, 9.0])
    units += torch.tensor([0.0, 1234567.0, 3.0, 4000000.0, 77.0, 50.0])[:, None]
    x, d, var = _exact_rows(units, size)
    w, b, dy = torch.randn(C, generator=g), torch.randn(C, generator=g), torch.randn(6, C, generator=g)
    y, mean, rstd = K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda))
    r = (var + 1e-5) ** -0.5
    f2 = (1 + torch.maximum(0.2501 * size**2 / var, torch.tensor(16.0).double()))[:, None]
    xh = d * r[:, None]
    xerr = U * (86 * f2 * xh.abs() + 58 * f2.sqrt())
    _within(rstd, r, (86 * U * f2[:, 0]) * r)
    _within(mean, x[:, 0].double() - d[:, 0], 0.501 * size)
    _within(y, xh * w.double() + b.double(), w.double().abs() * xerr + 2 * U * (xh * w.double()).abs() + 2 * U * b.double().abs())
    gx, gw, gb = K.layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), mean, rstd)
    q = dy.double() * w.double()
    c1, c2 = q.mean(-1, keepdim=True), (q * xh).mean(-1, keepdim=True)
    want = r[:, None] * (q - c1 - xh * c2)
    qm, a = q.abs().mean(-1, keepdim=True), xh.abs()
    c2err = U * (q.abs() * 2 * (86 * f2 * a + 58 * f2.sqrt())).mean(-1, keepdim=True) + 57 * U * f2.sqrt() * qm
    bound = 4 * U * q.abs() + 60 * U * qm + a * c2err + c2.abs() * xerr + 3 * U * (a * c2.abs())
    _within(gx, want, r[:, None] * bound + (88 * U * f2) * want.abs())
    ad = dy.double().abs()
    _within(gw, (dy.double() * xh).sum(0), (ad * xerr).sum(0) + 14 * U * (ad * a).sum(0))
    _within(gb, dy.double().sum(0), 14 * U * ad.sum(0))

def _rows_of_a_wave(dtype, N, C):
    """How many rows a wave of the gradient takes: four waves a workgroup have a row each up to 2048 16-bit or 1024 32-bit
    channels, a workgroup has one beyond; 512 workgroups, 256 above 8192 channels."""
    at_once = 4 if C <= (1024 if dtype is F else 2048) else 1
    groups = min(-(-N // at_once), 512 if C <= 8192 else 256)
    return -(-N // (groups * at_once))


@pytest.mark.parametrize("dtype,wdtype", [(H, H), (B16, F), (F, F)], ids=str)
@pytest.mark.parametrize("N,C", [(9000, 72), (5000, 1030), (1500, 2056), (1200, 4096), (1100, 8192), (700, 8200), (600, 16384)])
def test_weight_gradients_of_many_rows(cuda, dtype, wdtype, N, C):
    """Rows added up in a wave's registers, then the waves of a workgroup, then the workgroups in 64 bits.

    R rows of a wave and three more waves: R + 3 roundings, U of the terms each, and the errors of the normalised values,
    U (86 |xh| + 58) (the first mean is off by 54 U of mean |x|, nothing beside the deviation here); then half a step."""
    g = _gen(N, C, 3)
    x = (torch.randn(N, C, generator=g) * (torch.randn(C, generator=g) * 0.6).exp() + torch.randn(C, generator=g)).to(dtype)
    dy, w, b = torch.randn(N, C, generator=g).to(dtype), (1 + 0.2 * torch.randn(C, generator=g)).to(wdtype), torch.zeros(C, dtype=wdtype)
    _, mean, rstd = K.layer_norm_forward(x.to(cuda), w.to(cuda), b.to(cuda))
    _, gw, gb = K.layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), mean, rstd)
    d = x.double() - x.double().mean(-1, keepdim=True)
    xh = d * ((d * d).mean(-1, keepdim=True) + 1e-5) ** -0.5
    R, ad = _rows_of_a_wave(dtype, N, C), dy.double().abs()
    assert R > 1
    for got, want, terms, err in ((gw, (dy.double() * xh).sum(0), (ad * xh.abs()).sum(0), (ad * U * (86 * xh.abs() + 58)).sum(0)),
                                  (gb, dy.double().sum(0), ad.sum(0), 0.0)):
        half = torch.finfo(wdtype).eps / 2 * want.abs() + (2.0**-25 if wdtype is H else 0.0)
        _within(got, want, (R + 3) * U * terms + err + half + U * want.abs())
