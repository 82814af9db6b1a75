"""``verify_draft`` on logits with NaN of every kind, which count as -inf: the same tokens, bit for bit, as with -inf there
(the exponentials of both are the same numbers)."""

from __future__ import annotations

import pytest
import torch

from rwkv_tl_amd import verify_draft

pytestmark = pytest.mark.gpu
H, B16, F = torch.float16, torch.bfloat16, torch.float32
# of each type: quiet and signalling NaN of either sign, the least and the largest
PAYLOADS = {H: (torch.int16, [0x7E00, 0x7C01, 0x7FFF, -0x200, -0x3FF, -1]),
            B16: (torch.int16, [0x7FC0, 0x7F81, 0x7FFF, -0x40, -0x7F, -1]),
            F: (torch.int32, [0x7FC00000, 0x7F800001, 0x7FFFFFFF, -0x400000, -0x7FFFFF, -1])}


def _with_nan(x, where):
    """x with NaN of all kinds in turn, and with -inf, in the same places."""
    ints, kinds = PAYLOADS[x.dtype]
    bits = x.clone().view(ints)
    n = int(where.sum())
    bits[where] = torch.tensor(kinds, dtype=ints)[torch.arange(n) % 6]
    nan = bits.view(x.dtype)
    assert torch.equal(nan.isnan(), where)
    return nan, x.masked_fill(where, -torch.inf)


def _places(g, *shape):
    """In each row: a few, half of them, every other one, a whole end; all but a few; none."""
    out = torch.zeros(shape, dtype=torch.bool)
    flat = out.view(-1, shape[-1])
    V = shape[-1]
    for i, row in enumerate(flat):
        kind = i % 6
        if kind == 0:
            row[torch.randint(0, V, (3,), generator=g)] = True
        elif kind == 1:
            row[torch.rand(V, generator=g) < 0.5] = True
        elif kind == 2:
            row[1::2] = True
        elif kind == 3:
            row[V // 3 :] = True
        elif kind == 4:
            row[torch.rand(V, generator=g) < 0.99] = True
    return out


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("V", [5, 300, 5000, 8200, 65536])
@pytest.mark.parametrize("offset", [0.0, -2000.0])
def test_every_nan_counts_as_minus_infinity(cuda, dtype, V, offset):
    g = torch.Generator().manual_seed(V)
    B, K = 6, 4
    x = (2 * torch.randn(B, K + 1, V, generator=g) + offset).to(dtype)
    d = (x[:, :K].float() + torch.randn(B, K, V, generator=g)).to(dtype)
    t_nan, t_inf = _with_nan(x, _places(g, B, K + 1, V))
    d_nan, d_inf = _with_nan(d, _places(g, B, K, V).flip(0))
    up = lambda *a: [v.to(cuda) for v in a]  # noqa: E731
    t_nan, t_inf, d_nan, d_inf = up(t_nan, t_inf, d_nan, d_inf)
    best = torch.where(t_inf.isneginf().all(-1), 0, t_inf.float().argmax(-1))[:, :K]
    for tok in (best, torch.randint(0, V, (B, K), generator=g).to(cuda)):
        want = verify_draft(t_inf, tok, None)
        assert all(torch.equal(a, b) for a, b in zip(verify_draft(t_nan, tok, None), want))
        for _ in range(3):
            u = torch.rand(B, K + 1, generator=g).to(cuda)
            for draft in ((None, None), (d_nan, d_inf)):
                got = verify_draft(t_nan, tok, u, draft[0], temperature=0.8)
                want = verify_draft(t_inf, tok, u, draft[1], temperature=0.8)
                assert all(torch.equal(a, b) for a, b in zip(got, want))
