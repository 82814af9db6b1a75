"""Generation by a large model from a small one's drafts (speculative decoding).

The small model drafts a few tokens one by one, the large one takes them in a
single call (``prefill_logits``), and ``verify_draft`` keeps those that pass and
draws the token behind them: the ids are distributed as the large model's own
(at temperature None or <= 0 they are its greedy ones, up to ties within the
rounding of its two paths). No counterpart in the reference.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .logits import MAX_DRAFT, _temperature, verify_draft
from .rwkv7_hip import RWKV7HIP
from .sampling import Sampler
from .state import State


def _arenas(model, S: State) -> list[Tensor]:
    model._check_state(S)
    if not (isinstance(S, State) and S.arena_intact() and S.batch is None):
        raise ValueError("generate_speculative takes single-sequence States whose tensors were not rebound")
    return list(S.arenas)


def _advance(model, tokens: Tensor, S: State) -> None:
    """``S`` on by ``tokens``; one token by the decode kernel (0.4B: 0.32 ms, as a prefill of one 0.73)."""
    if tokens.numel() == 1:
        model.decode(tokens, S)
    else:
        model.prefill(tokens, S)


def generate_speculative(
    model: RWKV7HIP,
    draft: RWKV7HIP,
    tokens: list[int] | Tensor,
    S: State,
    S_draft: State,
    max_tokens: int = 32,
    *,
    n_draft: int = 4,
    temperature: float | None = None,
) -> tuple[list[int], State, State]:
    """``model.generate`` with ``draft`` (a smaller model of the same vocabulary)
    proposing up to ``n_draft`` tokens at a time, 1 <= n_draft <= 63.

    ``S`` and ``S_draft`` are the two models' states before the prompt ``tokens``
    (two or more). The models may be wrapped in ``HIPGraph``; an int8 one can only
    draft. Returns ``(ids, S, S_draft)``; the states hold everything but
    the last id, as after ``generate``. The host waits once per round of drafts,
    for the number accepted."""
    dev, V = model.w.device, model.w.head.shape[0]
    if draft.w.head.shape[0] != V or draft.w.device != dev:
        raise ValueError("the draft model must share the target's vocabulary and device")
    if draft.kernel_dtype != model.kernel_dtype:
        raise ValueError(f"the draft model is {draft.kernel_dtype}, the target {model.kernel_dtype}")
    if not 1 <= n_draft <= MAX_DRAFT:
        raise ValueError(f"n_draft must be in 1..{MAX_DRAFT}, got {n_draft}")
    if model.weight_quant is not None:
        raise ValueError("an int8 model prefills with its 16-bit weights and decodes with the int8 ones: it can draft, not verify")
    greedy = temperature is None or temperature <= 0
    if not greedy:
        _temperature(temperature)
    tokens = torch.as_tensor(tokens)
    if tokens.ndim != 1 or tokens.numel() < 2:
        raise ValueError(f"expected a prompt of two or more token ids, got shape {tuple(tokens.shape)}")
    tokens = model._tokens(tokens, tuple(tokens.shape))
    states = ((model, S, _arenas(model, S)), (draft, S_draft, _arenas(draft, S_draft)))
    if {a.data_ptr() for a in states[0][2]} & {a.data_ptr() for a in states[1][2]}:
        raise ValueError("S and S_draft share their tensors")
    for m, s, _ in states:
        _advance(m, tokens[:-1], s)
    sampler = Sampler(V, dev, temperature=temperature)
    ids: list[int] = []
    row = torch.empty(n_draft + 1, dtype=torch.int64, device=dev)  # the last token, then the drafts
    row[:1] = tokens[-1:]
    q = torch.empty(n_draft, V, dtype=draft.kernel_dtype, device=dev)
    while len(ids) < max_tokens:
        k = min(n_draft, max_tokens - len(ids) - 1)
        saved = [[a.clone() for a in arenas] for _, _, arenas in states]
        for i in range(k):
            logits, _ = draft.decode(row[i], S_draft)
            q[i] = logits
            sampler(logits, row[i + 1 : i + 2])
        p, _ = model.prefill_logits(row[: k + 1], S)
        u = None if greedy else torch.rand(k + 1, device=dev)
        out, n = verify_draft(p, row[1 : k + 1], u, None if greedy else q[:k], temperature=temperature)
        n_ok, *new = torch.cat([n.view(1), out]).tolist()  # the round's only wait
        if n_ok < k:  # both states back, and on by what was accepted
            for (m, s, arenas), old in zip(states, saved):
                for a, b in zip(arenas, old):
                    a.copy_(b)
                _advance(m, row[: n_ok + 1], s)
        else:  # the draft model has not taken its own last token
            _advance(draft, row[k : k + 1], S_draft)
        ids += new[: n_ok + 1]
        row[:1] = out[n_ok : n_ok + 1]
    for m, _, _ in states:
        m.raise_if_aborted()
    return ids, S, S_draft
