"""Alternatives of ``token_logprobs`` in rows with NaN: their ids are ``top_logits``' (NaN behind everything, ties by the
lowest id), and every log probability of the row is NaN."""

from __future__ import annotations

import pytest
import torch

import rwkv_tl_amd  # noqa: F401
from rwkv_tl_amd import kernels as K

pytestmark = pytest.mark.gpu
H, B16, F = torch.float16, torch.bfloat16, torch.float32
# of each type: quiet and signalling NaN of either sign, the least and the largest
PAYLOADS = {H: (torch.int16, [0x7E00, 0x7C01, 0x7FFF, 0xFE00, 0xFC01, 0xFFFF]),
            B16: (torch.int16, [0x7FC0, 0x7F81, 0x7FFF, 0xFFC0, 0xFF81, 0xFFFF]),
            F: (torch.int32, [0x7FC00000, 0x7F800001, 0x7FFFFFFF, 0xFFC00000, 0xFF800001, 0xFFFFFFFF])}


def _order(z, k):
    """Ids by value, largest first, ties by the lowest id, NaN last (in the order of their ids)."""
    d = z.double()
    d = torch.where(d == 0, 0.0, d)
    nan = d.isnan()
    first = torch.sort(torch.where(nan, -torch.inf, d), dim=-1, descending=True, stable=True).indices
    behind = torch.gather(nan, 1, first).long()
    return torch.gather(first, 1, torch.sort(behind, dim=-1, stable=True).indices)[:, :k]


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("V,k", [(7, 7), (300, 5), (300, 256), (2047, 64), (5001, 200), (16385, 20), (40001, 128), (65536, 5), (65536, 256)])
def test_alternatives_beside_nan(cuda, dtype, V, k):
    ints, payloads = PAYLOADS[dtype]
    g = torch.Generator().manual_seed(V + k)
    places = [  # where the NaN are
        [0], [V - 1], [V // 2], list(range(0, V, max(1, V // 37))),  # one, and some in every wave
        list(range(min(V - 1, 8), min(V, 520))),  # one wave's first chunk and its neighbour's
        list(range(1, V, 2)), list(range(V - k // 2, V)),  # half of them; fewer than k others are left out only in short rows
        list(range(V - 1)), list(range(V)),  # all but one; all
    ]
    rows = []
    for i, at in enumerate(places):
        for few in (False, True):  # values all unlike, or of a few kinds (long ties)
            z = (torch.randint(-2, 3, (V,), generator=g).float() if few else torch.randn(V, generator=g)) - (5.0 if i % 2 else 0.0)
            bits = z.to(dtype).view(ints)
            p = torch.tensor(payloads, dtype=torch.int64)
            p = torch.where(p >= 2 ** (8 * bits.element_size() - 1), p - 2 ** (8 * bits.element_size()), p)  # (as signed)
            which = torch.arange(len(at)) % 6 if i != 3 else torch.full((len(at),), 0 if few else 3)
            bits[torch.tensor(at)] = p[which].to(ints)
            rows.append(bits.view(dtype))
    rows.append(torch.where(torch.arange(V) % 3 == 0, torch.nan, -torch.inf).to(dtype))
    z = torch.stack(rows)
    assert z.isnan().any(-1).all()
    t = torch.randint(0, V, (len(rows),), generator=g).to(cuda)
    lp, ent, top, idx = K.token_logprobs(z.to(cuda), t, k)
    assert lp.isnan().all() and ent.isnan().all() and top.isnan().all()
    assert torch.equal(idx.cpu(), _order(z, k))
    assert torch.equal(idx, K.top_logits(z.to(cuda), k)[1])


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
def test_nan_beside_sound_rows(cuda, dtype):
    """The rows beside those have what they have without them."""
    g = torch.Generator().manual_seed(1)
    z = torch.randn(9, 65536, generator=g).to(dtype).to(cuda)
    t = torch.randint(0, 65536, (9,), generator=g).to(cuda)
    want = K.token_logprobs(z, t, 50)
    z[1::2, 77] = torch.nan
    got = K.token_logprobs(z, t, 50)
    assert all(torch.equal(a[::2], b[::2]) for a, b in zip(got, want)) and got[2][1::2].isnan().all()
