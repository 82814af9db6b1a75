"""``prefill_logits``, ``generate_speculative``, and the operators between a large
and a small model used together: answers of one model, their top logits, the
other's divergence from them and its gradient. Against the CPU oracle."""

from __future__ import annotations

import pytest
import torch

from oracle import logits_ref as LR
from oracle import rwkv7_ref as R
from rwkv_tl_amd import RWKV7HIP, RWKV7HIPBF16, RWKV7HIPInt8, HIPGraph, generate_speculative
from rwkv_tl_amd import kernels as K
from rwkv_tl_amd.checkpoint import make_random_state_dict
from rwkv_tl_amd.weight import RWKV7Weight

pytestmark = pytest.mark.gpu
ATOL, RTOL = 1e-2, 1e-3  # the logits' bar of the model tests


def _model(cuda, shape="tiny", seed=0, cls=RWKV7HIP, scale=1.0):
    dt = cls.kernel_dtype
    sd = make_random_state_dict(shape, seed=seed, dtype=dt)
    sd["head.weight"] = (sd["head.weight"].float() * scale).to(dt)
    w = RWKV7Weight.from_state_dict(sd, device=cuda, dtype=dt)
    return cls(w, is_torch_compile=False), R.Weights.from_emb(sd, w.emb.cpu(), torch.float32)


def _oracle_logits(ref, model, toks):
    s = R.new_state(model.L, model.C, dtype=model.kernel_dtype)
    out = []
    for t in toks:
        logits, s = R.decode(ref, t.reshape(1), s)
        out.append(logits.reshape(-1))
    return torch.stack(out)


def _tokens(*shape, vocab=512, seed=1):
    return torch.randint(0, vocab, shape, generator=torch.Generator().manual_seed(seed))


def _same_states(a, b):
    return all(torch.equal(x, y) for x, y in zip(a.arenas, b.arenas))


# 1 token: decode; up to 16 rows: the few-row kernel; 17 and 40: the GEMM path; 130: the chunked scan
@pytest.mark.parametrize("cls", [RWKV7HIP, RWKV7HIPBF16])
@pytest.mark.parametrize("path", ["auto", "kernels"])
@pytest.mark.parametrize("B,T", [(None, 1), (None, 2), (None, 5), (None, 16), (None, 17), (None, 40), (None, 130), (1, 3), (2, 3), (4, 4),
                                 (3, 11)])
def test_prefill_logits_matches_oracle(cuda, cls, path, B, T):
    model, ref = _model(cuda, cls=cls)
    model.decode_path = path
    toks = _tokens(*((T,) if B is None else (B, T)), seed=T)
    S, S2 = model.new_state(batch=B), model.new_state(batch=B)
    logits, S1 = model.prefill_logits(toks.to(cuda), S)
    assert S1 is S and logits.shape == (*toks.shape, 512) and logits.dtype == model.kernel_dtype
    atol = ATOL if cls is RWKV7HIP else 4e-2  # bf16 logits near 1 are 2^-8 apart, shift states 2^-8 of themselves off
    for b in range(B or 1):
        want = _oracle_logits(ref, model, toks if B is None else toks[b])
        got = (logits if B is None else logits[b]).float().cpu()
        assert ((got - want).abs() <= atol + RTOL * want.abs()).all(), float((got - want).abs().max())
    if T > 1:  # the state is the prefill's, bit for bit
        model.prefill(toks.to(cuda), S2)
        assert _same_states(S, S2)


def test_prefill_logits_of_many_rows_in_blocks(cuda):
    """3001 rows: head products of 1024, 1024 and 953 rows, against two calls that split elsewhere."""
    model, _ = _model(cuda)
    toks = _tokens(3001).to(cuda)
    whole, S = model.prefill_logits(toks, model.new_state())
    S2 = model.new_state()
    parts = [model.prefill_logits(t, S2)[0] for t in (toks[:1800], toks[1800:])]
    assert ((whole.float() - torch.cat(parts).float()).abs() <= ATOL + RTOL * whole.float().abs()).all()
    one = model.new_state()
    model.prefill(toks[:-1], one)
    last, _ = model.decode(toks[-1:], one)
    assert ((whole[-1].float() - last.float()).abs() <= ATOL + RTOL * last.float().abs()).all()


def test_prefill_logits_through_a_graph_wrapper_and_a_rebound_state(cuda):
    model, _ = _model(cuda)
    toks = _tokens(6).to(cuda)
    want, S = model.prefill_logits(toks, model.new_state())
    got, _ = HIPGraph(model).prefill_logits(toks, model.new_state())
    assert torch.equal(got, want)
    S2 = model.new_state()
    S2[0][0]["x"] = S2[0][0]["x"].clone()
    got, _ = model.prefill_logits(toks, S2)
    assert torch.equal(got, want) and torch.equal(S2[0][0]["x"], S[0][0]["x"])
    with pytest.raises(RuntimeError):
        model.prefill_logits(toks[:0], S)
    with pytest.raises(ValueError):
        model.prefill_logits(toks.view(2, 3), S)


@pytest.mark.parametrize("same", [True, False])
@pytest.mark.parametrize("n_draft,max_tokens", [(1, 7), (4, 24), (15, 20), (20, 3), (4, 1), (3, 0)])
def test_speculative_greedy_ids_are_the_targets(cuda, same, n_draft, max_tokens):
    """Along the ids that come out, each is the target's argmax as it decodes one by one, up to the rounding between its
    paths (twice the logits' bar); the states are those after the prompt and all ids but the last."""
    model, _ = _model(cuda, scale=8.0)
    draft = model if same else _model(cuda, seed=7, scale=8.0)[0]
    prompt = _tokens(9, seed=3)
    ids, S, Sd = generate_speculative(model, draft, prompt.tolist(), model.new_state(), draft.new_state(), max_tokens, n_draft=n_draft)
    assert len(ids) == max_tokens
    for m, s in ((model, S), (draft, Sd)):
        ref = m.new_state()
        m.prefill(prompt[:-1].to(cuda), ref)
        last = int(prompt[-1])
        for t in ids:
            logits, ref = m.decode(torch.tensor([last], device=cuda), ref)
            if m is model:
                assert float(logits.max()) - float(logits[t]) <= 2 * (ATOL + RTOL * float(logits.abs().max()))
            last = t
        for x, y in zip(s.arenas, ref.arenas):
            assert float((x.float() - y.float()).norm()) <= 5e-3 * float(y.float().norm())


def test_speculative_sampling_draws_and_repeats(cuda):
    model, _ = _model(cuda, scale=8.0)
    draft, _ = _model(cuda, seed=7, scale=8.0)
    prompt = _tokens(5, seed=4).tolist()
    runs = []
    for _ in range(2):
        torch.manual_seed(11)
        runs.append(generate_speculative(model, draft, prompt, model.new_state(), draft.new_state(), 30, n_draft=5, temperature=0.9)[0])
    assert runs[0] == runs[1] and len(runs[0]) == 30 and all(0 <= t < 512 for t in runs[0])
    torch.manual_seed(12)
    assert generate_speculative(model, draft, prompt, model.new_state(), draft.new_state(), 30, n_draft=5, temperature=0.9)[0] != runs[0]


def test_speculative_follows_the_targets_distribution(cuda):
    """The first two ids of 1500 runs (a draft that disagrees with a peaked target): each frequency of the likely ids
    within 5 standard deviations, plus the 1e-2 that a logit may be off (a relative 1e-2 of a probability)."""
    model, _ = _model(cuda, scale=40.0)
    draft, _ = _model(cuda, seed=7, scale=20.0)
    prompt = _tokens(3, seed=5)
    n = 1500
    torch.manual_seed(13)
    got = torch.tensor([generate_speculative(model, draft, prompt.tolist(), model.new_state(), draft.new_state(), 2, n_draft=1,
                                             temperature=1.0)[0] for _ in range(n)])
    S = model.new_state()
    first = torch.softmax(model.prefill_logits(prompt.to(cuda), S)[0][-1].double(), -1).cpu()
    second = torch.zeros(512, dtype=torch.float64)
    arenas = [a.clone() for a in S.arenas]
    for t in range(512):
        for a, b in zip(S.arenas, arenas):
            a.copy_(b)
        second += first[t] * torch.softmax(model.decode(torch.tensor([t], device=cuda), S)[0].double(), -1).cpu()
    for i, p in enumerate((first, second)):
        f = torch.bincount(got[:, i], minlength=512).double() / n
        big = p > 0.01
        assert ((f - p).abs()[big] <= 5 * (p * (1 - p) / n).sqrt()[big] + 2e-2 * p[big]).all()


def test_speculative_refusals(cuda):
    model, _ = _model(cuda)
    S = model.new_state
    bf, _ = _model(cuda, cls=RWKV7HIPBF16)
    for bad in (lambda: generate_speculative(model, model, [1], S(), S()), lambda: generate_speculative(model, model, [1, 2], S(), S(), n_draft=0),
                lambda: generate_speculative(model, model, [1, 2], S(), S(), n_draft=64),
                lambda: generate_speculative(model, bf, [1, 2], S(), bf.new_state()),
                lambda: generate_speculative(model, model, [1, 2], S(batch=1), S())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("T", [None, 0.9])
def test_speculative_through_graph_wrappers_and_an_int8_draft(cuda, T):
    """The same ids as of the bare models (the same kernels run); an int8 copy of the target drafts for it."""
    model, _ = _model(cuda, scale=8.0)
    draft, _ = _model(cuda, seed=7, scale=8.0)
    prompt = _tokens(9, seed=3).tolist()

    def ids(m, d):
        torch.manual_seed(5)
        return generate_speculative(m, d, prompt, m.new_state(), d.new_state(), 25, n_draft=4, temperature=T)[0]

    assert ids(HIPGraph(model), HIPGraph(draft)) == ids(model, draft)
    q, _ = _model(cuda, cls=RWKV7HIPInt8, scale=8.0)
    got = ids(model, q)
    assert len(got) == 25
    with pytest.raises(ValueError, match="int8"):
        ids(q, model)


def test_speculative_refuses_before_it_touches_a_state(cuda):
    model, _ = _model(cuda)
    S, Sd = model.new_state(), model.new_state()
    before = [a.clone() for a in S.arenas]
    for prompt, T in (([1, 512], None), ([-1, 3], None), ([1.0, 2.0], None), ([1, 2], float("nan")), ([1, 2], 1e-40), ([[1, 2]], None)):
        with pytest.raises(ValueError):
            generate_speculative(model, model, prompt, S, Sd, temperature=T)
    assert all(torch.equal(a, b) for a, b in zip(S.arenas, before))


def test_speculative_refuses_one_state_for_both_models(cuda):
    model, _ = _model(cuda)
    S = model.new_state()
    before = [a.clone() for a in S.arenas]
    with pytest.raises(ValueError, match="share"):
        generate_speculative(model, model, [1, 2], S, S)
    assert all(torch.equal(a, b) for a, b in zip(S.arenas, before))


@pytest.mark.parametrize("cls", [RWKV7HIP, RWKV7HIPBF16])
def test_distillation_step_from_one_model_to_another(cuda, cls):
    """A teacher's answers to two sequences (the last tokens of one padding), its top logits, and a student's head trained
    on them: loss and the gradient of the head's matrix against float64 from the same logits and inputs."""
    teacher, _ = _model(cuda, scale=8.0, cls=cls)
    student, _ = _model(cuda, seed=7, scale=8.0, cls=cls)
    toks = _tokens(2, 21, seed=6).to(cuda)
    answers, _ = teacher.prefill_logits(toks, teacher.new_state(batch=2))
    val, idx, lse = K.top_logits(answers, 24, temperature=2.0)
    idx[1, 15:] = -1
    logits, _ = student.prefill_logits(toks, student.new_state(batch=2))
    g = torch.Generator().manual_seed(1)
    hidden = torch.randn(2, 21, 64, generator=g).to(cuda)
    add = torch.zeros(512, 64, device=cuda, requires_grad=True)  # a low-rank correction of the head
    z = logits.float() + hidden @ add.t()
    loss = torch.ops.rwkv_tl.distill_loss(z, val, idx, lse, 2.0)
    weight = (idx[..., 0] >= 0).float() / float((idx[..., 0] >= 0).sum())
    (loss * weight).sum().backward()
    zr = logits.double().cpu().view(42, 512).requires_grad_()
    want = LR.distill_loss(zr, val.cpu().view(42, 24), idx.cpu().view(42, 24), lse.cpu().view(42), 2.0)
    assert torch.allclose(loss.detach().double().cpu().view(42), want.detach(), rtol=1e-6, atol=1e-5)
    assert (loss[1, 15:] == 0).all()
    (gz,) = torch.autograd.grad((want * weight.double().cpu().view(42)).sum(), zr)
    gw = gz.t() @ hidden.double().cpu().view(42, 64)
    assert float((add.grad.double().cpu() - gw).norm() / gw.norm()) < 1e-4  # (the f32 product of 42 rows)
    both = K.distill_loss_grad(logits, val, idx, lse, temperature=2.0, scale=weight)
    eps = torch.finfo(cls.kernel_dtype).eps
    ref = gz.view(2, 21, 512)
    assert ((both[1].double().cpu() - ref).abs() <= eps / 2 * ref.abs() + 2.0**-24 + 1e-6).all()
