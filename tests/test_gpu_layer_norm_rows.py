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
