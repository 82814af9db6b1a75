"""``verify_draft`` over the whole range of its 64-bit exponentials: rows whose sums about 0 come near the range's ends,
masked tokens at u = 0, and goals that the running sum meets within a rounding. Against float64 on the CPU
(``oracle.logits_ref``) and whole numbers. Tokens are compared for equality: the kernel's sums are within 1e-11 of
themselves, a random u meets a border between two of some thousand tokens by that with a chance of 1e-8, and the inputs
are fixed."""

from __future__ import annotations

import pytest
import torch

from oracle import logits_ref as R
from rwkv_tl_amd import verify_draft

pytestmark = pytest.mark.gpu
H, B16, F = torch.float16, torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")
LOG2E = 1.4426950408889634


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _zipf(g, *shape):
    return -1.3 * torch.empty(*shape).exponential_(generator=g).log()


def _check(cuda, target, tok, u, draft, T, Td):
    """Equal to the oracle. But behind the rejection of a token drawn from a row almost the target's own the residual
    max(p - q, 0) is what is left of a cancellation: p and q are known to 2e-12, so of a residual of 1e-3 in all some 9000
    borders are known to 4e-9 (a u meets one of those with a chance of 4e-5), and of one below that less and less, down to
    roundings, the oracle's too. There the token needs only be one that the target allows."""
    up = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    out, n = (o.cpu() for o in verify_draft(up(target), up(tok), up(u), up(draft), temperature=T, draft_temperature=Td))
    want, wn = R.verify_draft(target, tok, u, draft, T, Td)
    assert torch.equal(n, wn)
    if draft is not None and Td > 0:
        p, q = (torch.softmax(x[:, 0].double().nan_to_num(nan=-INF) / t, -1) for x, t in ((target, T), (draft, Td)))
        vague = (n == 0) & ((p - q).clamp_min(0.0).sum(-1) < 1e-3)
        assert bool((p.gather(1, out[:, :1].clamp_min(0))[:, 0] > 0)[vague].all()) and bool((out[vague, 1] == -1).all())
        out, want = out[~vague], want[~vague]
    assert torch.equal(out, want)


def _shifted(row, shifts, dtype):
    """``row`` [V], largest 0, moved so that its largest is each of ``shifts``."""
    return (row + shifts[:, None]).to(dtype)


# ---------------------------------------------------------------------------
# rows whose sum about 0 comes near the lower end of the range
# ---------------------------------------------------------------------------

# (largest logit) * log2(e) / T: where a slice's sum about 0 is and is not taken, and the range's own end
SWEEPS = {"-920..-880": torch.arange(-920.0, -879.0), "-600..-560": torch.arange(-600.0, -559.0, 2.0),
          "-420..-380": torch.arange(-420.0, -379.0), "-1010..-980": torch.arange(-1010.0, -979.0)}


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("sweep", SWEEPS)
@pytest.mark.parametrize("T", [1.0, 0.1, 0.01])
def test_rows_near_the_ends_of_the_range(cuda, dtype, sweep, T):
    at = SWEEPS[sweep] * (T / LOG2E)
    g = _gen(int(100 * T) + len(sweep))
    two = torch.full((8192,), -100.0)
    two[0], two[600] = 0.0, -0.002 * T / 0.01  # two tokens of weight in different blocks of 512
    for row in (torch.zeros(1000), torch.zeros(8192), two * max(1.0, T), T * _zipf(g, 9001)):
        row = row - row.max()
        x = _shifted(row, at, dtype)
        n, V = x.shape
        u = torch.rand(n, 2, generator=g)
        none = torch.zeros(n, 0, dtype=torch.int64)
        _check(cuda, x[:, None], none, u[:, :1], None, T, 0.0)                       # no drafts
        tok = torch.randint(0, V, (n, 1), generator=g)
        both = torch.stack([x, x], 1)
        _check(cuda, both, tok, u, None, T, 0.0)                                     # drafts without a draw
        mild = x.float() + T * torch.randn(n, V, generator=g)
        _check(cuda, both, tok, u, mild.to(dtype)[:, None], T, T)                    # drawn from a row near the target's
        _check(cuda, both, tok, u, (T * torch.randn(n, 1, V, generator=g)).to(dtype), T, T)  # and from one near 0


@pytest.mark.parametrize("dtype", [H, F], ids=str)
def test_flat_rows_at_every_shift(cuda, dtype):
    g = _gen(7)
    at = -torch.arange(600.0, 641.0, 0.5)
    for V in (1000, 65536):
        x = _shifted(torch.zeros(V), at, dtype)
        _check(cuda, x[:, None], torch.zeros(len(at), 0, dtype=torch.int64), torch.rand(len(at), 1, generator=g), None, 1.0, 0.0)

# ---------------------------------------------------------------------------
# masked tokens are never drawn
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [H, B16, F], ids=str)
@pytest.mark.parametrize("mask", [-INF, NAN])
@pytest.mark.parametrize("T", [1.0, 0.05])
def test_masked_blocks_are_passed_over_at_u_0(cuda, dtype, mask, T):
    """u_K = 0 draws the first token with any weight: 512 and 1024 masked ones before it, rows at many distances from 0."""
    g = _gen(8)
    at = T * torch.tensor([0.0, 50.0, 500.0, -30.0, -60.0, -64.0, -70.0, -100.0, -120.0, -200.0, -270.0, -280.0, -300.0,
                           -500.0, -600.0, -620.0, -630.0, -700.0])
    for V, gone in ((1000, 512), (3000, 1024), (9001, 8192), (20003, 8704)):
        n = len(at)
        x = torch.stack([_shifted(T * _zipf(g, V), at, dtype)] * 2, 1)
        tok = torch.full((n, 1), V - 3)
        x[:, :, :gone] = mask
        x[:, 0, V - 3] = (x[:, 0, V - 3].float() - 30.0 * T).to(dtype)  # rejected at the u below
        u = torch.tensor([[1.0 - 2.0**-24, 0.0]]).repeat(n, 1)
        _check(cuda, x, tok, u, None, T, 0.0)
        draft = T * _zipf(g, n, 1, V)
        draft[:, :, V - 3] = draft.amax(-1) + 20.0 * T
        for q in (draft, draft.masked_fill(torch.arange(V) < gone, mask), draft + at[:, None, None]):
            _check(cuda, x, tok, u, q.to(dtype), T, T)
        u[:, 0] = 0.0  # accepted: the draw from p itself
        _check(cuda, x, tok, u, draft.to(dtype), T, T)
        u[:, 1] = 1.0  # (the documented range ends below it: the last token with any weight)
        _check(cuda, x, tok, u, draft.to(dtype), T, T)


def test_masked_blocks_in_wide_batches(cuda):
    """The same in batches whose decisive rows are dealt 8192 logits to a workgroup."""
    g = _gen(10)
    V, gone = 9001, 2048
    at = torch.tensor([0.0, -60.0, -70.0, -120.0, -270.0, -290.0, -500.0, -630.0, -700.0])
    x = torch.stack([_shifted(_zipf(g, V), at, F)] * 2, 1)
    x[:, :, :gone] = -INF
    x[:, 0, V - 3] -= 30.0
    draft = _zipf(g, len(at), 1, V)
    draft[:, :, V - 3] = draft.amax(-1) + 20.0
    tok = torch.full((len(at), 1), V - 3)
    for last in (0.0, 0.3, 1.0 - 2.0**-24):
        u = torch.tensor([[1.0 - 2.0**-24, last]]).repeat(len(at), 1)
        for q in (None, draft):
            want = R.verify_draft(x, tok, u, q, 1.0, 0.0 if q is None else 1.0)[0]
            many = [None if t is None else t.repeat(26, *[1] * (t.ndim - 1)).to(cuda) for t in (x, tok, u, q)]
            out, n = verify_draft(*many, temperature=1.0)
            assert bool((n == 0).all()) and torch.equal(out.cpu(), want.repeat(26, 1))


def test_a_residual_of_roundings_alone_draws_no_masked_token(cuda):
    """One token before the others whose p and q are a rounding apart: whether that leaves it any weight is a matter of
    roundings, but the masked ones around it have none."""
    n, V = 4000, 1500
    g = _gen(9)
    x = torch.full((n, 2, V), -INF)
    x[:, :, 300] = -6.0 * torch.rand(n, 1, generator=g) - 0.5
    x[:, :, 600:856] = 0.0
    x[:, :, 1100] = 0.0
    q = x[:, :1].clone()
    q[:, :, 1100], q[:, :, 1200] = -INF, 0.0
    q[:, 0, 700] = 2.0**-45 * torch.randint(-6, 7, (n,), generator=g)
    out, acc = verify_draft(x.to(cuda), torch.full((n, 1), 1200, device=cuda), torch.zeros(n, 2, device=cuda), q.to(cuda),
                            temperature=0.7)
    assert (acc == 0).all()
    assert x[:, 0].gather(1, out[:, :1].cpu()).isfinite().all()


# ---------------------------------------------------------------------------
# goals within a rounding of a border
# ---------------------------------------------------------------------------

# Sums of blocks of 512 tokens, as multiples of one weight: those of the first lanes of three blocks are a few units more
# than half of all, so that at u = 0.5 the exact sum passes the goal at the last token of the last of them, while the
# running sum in 64 bits, from block to block, ends on the goal.
BLOCK_SUMS = [
    [1145859633778797, 352630542926771, 973175940787175, 613593555701514, 536808607908891, 881530479136178] + 9 * [450359876023932]
    + [450359876023937],
    [759373514701697, 1214240432488022, 128677358106348, 661252096165449, 1158952546121088, 581103048745430] + 9 * [450359899632803]
    + [450359899632806],
    [246368824764733, 548419992108399, 854323041859110, 396816985282743, 343466264402641, 358936908495985, 575037014482333,
     752082123627653, 428147725270595] + 6 * [643371268613455] + [643371268613458],
    [816075089083930, 362505266396518, 577498043038902, 604518220769384, 81891060324226, 196261183937186, 358973546335445,
     802100149714336, 703776430349826] + 6 * [643371284278536] + [643371284278536],
]


@pytest.mark.parametrize("case", range(len(BLOCK_SUMS)))
@pytest.mark.parametrize("dtype", [H, F], ids=str)
def test_a_goal_that_the_running_sum_just_misses(cuda, case, dtype):
    """Weights that are powers of two (T = log2(e), whole logits), the largest of each block last."""
    x = torch.full((1, 1, 8192), -INF)
    weight = [0] * 8192
    for b, s in enumerate(BLOCK_SUMS[case]):
        for j, e in enumerate(e for e in range(53) if s >> e & 1):
            x[0, 0, 512 * b + 9 * j + 3] = float(e)
            weight[512 * b + 9 * j + 3] = 1 << e
    acc, want = 0, None
    for v, w in enumerate(weight):  # the first whose exact sum exceeds half
        acc += w
        if 2 * acc > sum(weight):
            want = v
            break
    out, _ = verify_draft(x.to(dtype).to(cuda), torch.zeros(1, 0, dtype=torch.int64, device=cuda),
                          torch.full((1, 1), 0.5, device=cuda), temperature=LOG2E)
    assert out.tolist() == [[want]]
