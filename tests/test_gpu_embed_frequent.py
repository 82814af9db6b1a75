"""The embedding table's gradient where many of a workgroup's rows occur often: whole numbers, whose sums have one value
whatever their order, and the time of a call, which follows the number of tokens and not the number of frequent rows."""

from __future__ import annotations

import pytest
import torch

import rwkv_tl_amd  # noqa: F401
from rwkv_tl_amd import kernels as K

pytestmark = pytest.mark.gpu
H, B16, F = torch.float16, torch.bfloat16, torch.float32


def _check(cuda, t, V, C, g, dtype=F):
    dy = torch.randint(-8, 9, (t.numel(), C), generator=g).to(dtype)
    there = (t >= 0) & (t < V)
    want = torch.zeros(V + 1, C, dtype=torch.float64).index_add_(0, torch.where(there, t, V), dy.double())[:V].to(dtype)
    got = K.embed_backward(dy.to(cuda), t.to(cuda), V)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(got, K.embed_backward(dy.to(cuda), t.to(cuda), V))


def _mixed(counts, ids, g, pad=0):
    t = torch.cat([torch.repeat_interleave(ids, counts), torch.full((pad,), -1)])
    return t[torch.randperm(t.numel(), generator=g)]


@pytest.mark.parametrize("rows,most", [(2, 8000), (60, 250), (150, 100), (256, 70), (200, 300), (256, 500), (256, 4000)])
@pytest.mark.parametrize("step", [1, 256], ids=["neighbours", "one workgroup"])
def test_many_frequent_rows(cuda, rows, most, step):
    """Up to all 256 rows of one workgroup past 64 positions, of up to and of more than 16384 tokens."""
    g = torch.Generator().manual_seed(rows + most + step)
    counts = torch.randint(60, most + 1, (rows,), generator=g)
    counts[0] = most
    _check(cuda, _mixed(counts, torch.arange(rows) * step + 5, g, 100), rows * step + 9, 8, g)


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("N", [16384, 16385, 70000])
def test_rows_in_runs(cuda, dtype, N):
    """Each id's positions side by side, in alternation, and in blocks of 64 that begin anywhere."""
    g = torch.Generator().manual_seed(N)
    i = torch.arange(N)
    for t in (i // 100 * 256, i % 70 * 256, (i + 37) // 64 % 50 * 256 + (i // 5000), torch.where(i % 3 == 0, 512, i % 101 * 256)):
        _check(cuda, t, 65536, 9, g, dtype)


def test_every_row_frequent(cuda):
    """A million tokens of 8000 ids: 32 frequent rows a workgroup, 128 positions each."""
    g = torch.Generator().manual_seed(7)
    _check(cuda, torch.randint(0, 8000, (1 << 20,), generator=g), 8000, 4, g)


def test_the_time_follows_the_tokens(cuda):
    """The same number of tokens: rows of 16 positions, of which none is frequent, and of 128, where all are. The latter
    reads the tokens twice more, and a workgroup more for each of its 32 rows would be thirty times."""
    N = 1 << 20
    dy = torch.ones(N, 8, device=cuda)

    def best(ids):
        t = torch.randint(0, ids, (N,), device=cuda)
        out = []
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            K.embed_backward(dy, t, 65536)
            b.record()
            b.synchronize()
            out.append(a.elapsed_time(b))
        return min(out[1:])

    rare, often = best(65536), best(8192)
    assert often < 5 * rare, f"{often} ms for frequent rows, {rare} ms for rare ones"


@pytest.mark.parametrize("ids", [1, 3, 60000])
def test_the_most_tokens_of_a_call(cuda, ids):
    """2^24 - 1 of them: all one, of three ids, and 280 of each id. (Sums of at most 2^24 whole numbers of at most 1.)"""
    N = 2**24 - 1
    g = torch.Generator(device=cuda).manual_seed(ids)
    t = torch.randint(0, ids, (N,), generator=g, device=cuda) * (1 if ids > 3 else 256)
    dy = torch.randint(-1, 2, (N, 2), generator=g, device=cuda).float()
    V = int(t.max()) + 2
    got = K.embed_backward(dy, t, V)
    want = torch.stack([torch.bincount(t, dy[:, c].double(), minlength=V) for c in range(2)], 1)
    assert torch.equal(got.double(), want)


def test_a_table_past_2_to_the_32_bytes(cuda):
    """Rows of the table, looked up and filled, past 32 bits of elements."""
    V, C = 150001, 16500
    w = torch.zeros(V, C, dtype=H, device=cuda)
    ids = torch.tensor([0, 65535, 65536, 130149, 130151, V - 1, -1, V], device=cuda)
    w[ids[:6], 7] = torch.arange(1.0, 7.0, device=cuda).half()
    out = K.embed(w, ids)
    assert out[:, 7].tolist() == [1, 2, 3, 4, 5, 6, 0, 0] and int((out != 0).sum()) == 6
    del w
    t = ids.repeat_interleave(torch.tensor([1, 70, 2, 40, 1, 200, 3, 3], device=cuda))
    dy = torch.zeros(t.numel(), C, dtype=H, device=cuda)
    dy[:, 0], dy[:, C - 1] = 1, 2
    grad = K.embed_backward(dy, t, V)
    assert grad[ids[:6], 0].tolist() == [1, 70, 2, 40, 1, 200] and grad[ids[:6], C - 1].tolist() == [2, 140, 4, 80, 2, 400]
    rest = grad.view(torch.int16)
    rest[ids[:6, None], torch.tensor([0, C - 1], device=cuda)] = 0
    assert all(not bool(part.any()) for part in rest.split(20000))
