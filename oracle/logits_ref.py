"""Plain float64 restatements of the operators between a large and a small model
(``rwkv_tl_amd.logits``), a row and a token at a time, on the CPU."""

from __future__ import annotations

import math

import torch
from torch import Tensor

def least_rest(lse: float) -> float:
    """A teacher's mass outside its entries below this is none: half a step of ``lse`` as float32 (which rounding it may
    take from 1), 2^-20 at least."""
    return max(2.0**-20, math.ldexp(1.0, math.frexp(float(torch.tensor(lse).float()))[1] - 25))


def top_logits(logits: Tensor, k: int, temperature: float = 1.0) -> tuple[Tensor, Tensor, Tensor]:
    """Ids by (value descending, NaN last, id ascending), their values, and log-sum-exp."""
    x = logits.double()
    vals, ids = [], []
    for row in x:
        order = sorted(range(len(row)), key=lambda i: (bool(row[i].isnan()), -float(row[i]) if not row[i].isnan() else 0.0, i))
        ids.append(order[:k])
        vals.append([float(row[i]) for i in order[:k]])
    return torch.tensor(vals, dtype=torch.float64), torch.tensor(ids), torch.logsumexp(x / temperature, -1)


def distill_loss(logits: Tensor, top_val: Tensor, top_idx: Tensor, lse: Tensor | None, temperature: float = 1.0) -> Tensor:
    """Differentiable in ``logits`` (float64): the loss of each row."""
    V = logits.shape[-1]
    out = []
    for r in range(logits.shape[0]):
        live = (top_idx[r] >= 0) & (top_idx[r] < V)
        ids, t = top_idx[r][live], top_val[r][live].double() / temperature
        if not len(ids) or (bool((t == -torch.inf).all()) if lse is None else float(lse[r]) <= -(2.0**24)):
            out.append(logits[r].detach().new_zeros(()))
            continue
        if lse is not None and bool(lse[r].isnan()):
            out.append(logits[r].sum() * torch.nan)
            continue
        y = torch.log_softmax(logits[r] / temperature, -1)
        logp = t - (torch.logsumexp(t, -1) if lse is None else lse[r].double())
        p = logp.exp()
        some = p > 0
        loss = (p[some] * (logp[some] - y[ids[some]])).sum()
        rest = max(0.0, 1.0 - float(p.sum())) if lse is not None else 0.0
        outside = torch.ones(V, dtype=torch.bool)
        outside[ids] = False
        if lse is not None and rest >= least_rest(float(lse[r])) and bool(outside.any()):
            # about its own largest logit: far below the row's, the others' differences would be lost
            z = logits[r][outside]
            m = z.detach().max()
            m = m if bool(m.isfinite()) else torch.zeros_like(m)
            top = logits[r].detach().max()
            log_all = torch.logsumexp((logits[r] - top) / temperature, -1)
            log_out = torch.logsumexp((z - m) / temperature, -1) + (m - top) / temperature - log_all
            loss = loss + rest * (torch.tensor(rest, dtype=torch.float64).log() - log_out)
        out.append(loss)
    return torch.stack(out) if out else logits.new_zeros(0)


def _softmax(row: Tensor, temperature: float) -> Tensor:
    """Probabilities; NaN counts as -inf, +inf takes all, nothing at all gives zeros."""
    z = row.double().clone()
    z[z.isnan()] = -torch.inf
    m = z.max()
    if m == -torch.inf:
        return torch.zeros_like(z)
    w = (z == m).double() if m == torch.inf else ((z - m) / temperature).exp()
    return w / w.sum()


def verify_draft(target: Tensor, tokens: Tensor, uniforms: Tensor | None, draft: Tensor | None, temperature: float,
                 draft_temperature: float, lengths: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """One sequence after the other, one drafted token after the other."""
    B, K = tokens.shape
    V = target.shape[-1]
    outs, accepted = [], []
    for b in range(B):
        n = K if lengths is None else min(max(int(lengths[b]), 0), K)
        seq: list[int] = []
        for i in range(n + 1):
            x = int(tokens[b, i]) if i < n else -1
            if temperature <= 0:
                z = target[b, i].double().clone()
                z[z.isnan()] = -torch.inf
                best = int((z == z.max()).nonzero()[0])
                seq.append(best)
                if i == n or x != best:
                    break
                continue
            p = _softmax(target[b, i], temperature)
            r = p
            if i < n:
                if draft is None or draft_temperature <= 0:
                    q = torch.zeros_like(p)
                    if 0 <= x < V:
                        q[x] = 1.0
                else:
                    q = _softmax(draft[b, i], draft_temperature)
                if 0 <= x < V and p[x] > 0 and float(uniforms[b, i].double() * q[x]) < float(p[x]):
                    seq.append(x)
                    continue
                r = (p - q).clamp_min(0.0)
                r = r if float(r.sum()) > 0 else p
            c = r.cumsum(0)
            over = ((c > uniforms[b, K].double() * c[-1]) & (r > 0)).nonzero()
            some = (r > 0).nonzero()
            seq.append(int(over[0]) if len(over) else int(some[-1]) if len(some) else 0)
            break
        accepted.append(len(seq) - 1)
        outs.append(seq + [-1] * (K + 1 - len(seq)))
    return torch.tensor(outs), torch.tensor(accepted)
