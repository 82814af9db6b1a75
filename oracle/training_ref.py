"""The ends and the norms of a training step in float64: embedding and LayerNorm with
their gradients, log probabilities of tokens with entropy and gradient. Straight from
the formulas, no kernel's order or shape; used by the tests only."""

from __future__ import annotations

import torch
from torch import Tensor


def embed(weight: Tensor, tokens: Tensor, scale: float = 1.0) -> Tensor:
    V, C = weight.shape
    flat = tokens.reshape(-1)
    out = torch.zeros(flat.numel(), C, dtype=torch.float64)
    for i, t in enumerate(flat.tolist()):
        if 0 <= t < V:
            out[i] = scale * weight[t].double()
    return out.reshape(*tokens.shape, C)


def embed_grad(grad: Tensor, tokens: Tensor, vocab: int, scale: float = 1.0) -> Tensor:
    C = grad.shape[-1]
    out = torch.zeros(vocab, C, dtype=torch.float64)
    for g, t in zip(grad.reshape(-1, C).double(), tokens.reshape(-1).tolist()):
        if 0 <= t < vocab:
            out[t] += scale * g
    return out


def layer_norm(x: Tensor, weight: Tensor, bias: Tensor, eps: float = 1e-5) -> tuple[Tensor, Tensor, Tensor]:
    d = x.double()
    mean = d.mean(-1)
    d = d - mean[..., None]
    rstd = ((d * d).mean(-1) + eps) ** -0.5
    return d * rstd[..., None] * weight.double() + bias.double(), mean, rstd


def layer_norm_grad(grad: Tensor, x: Tensor, weight: Tensor, eps: float = 1e-5) -> tuple[Tensor, Tensor, Tensor]:
    C = x.shape[-1]
    one, zero = torch.ones(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)
    xh, _, rstd = layer_norm(x, one, zero, eps)
    dy = grad.double()
    g = dy * weight.double()
    gx = rstd[..., None] * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return gx, (dy * xh).reshape(-1, C).sum(0), dy.reshape(-1, C).sum(0)


def _log_softmax(z: Tensor) -> Tensor:
    """-inf throughout a row of -inf alone."""
    m = z.amax(-1, keepdim=True)
    masked = (z == -torch.inf).all(-1, keepdim=True)
    d = torch.where(masked, torch.zeros_like(z), z - torch.where(masked, torch.zeros_like(m), m))
    d = torch.where(m == torch.inf, torch.full_like(d, torch.nan), d)
    return torch.where(masked, torch.full_like(d, -torch.inf), d - d.exp().sum(-1, keepdim=True).log())


def token_logprobs(logits: Tensor, tokens: Tensor, temperature: float = 1.0) -> tuple[Tensor, Tensor]:
    V = logits.shape[-1]
    there = (tokens >= 0) & (tokens < V)
    y = _log_softmax(logits.double() / temperature)
    p = y.exp()
    H = -torch.where(p == 0, torch.zeros_like(p), p * y).sum(-1)
    lp = y.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0]
    zero = torch.zeros_like(H)
    return torch.where(there, lp, zero), torch.where(there, H, zero)


def token_logprobs_grad(logits: Tensor, tokens: Tensor, scale: Tensor, entropy_scale: Tensor, temperature: float = 1.0) -> Tensor:
    """scale * d logprob + entropy_scale * d entropy by the formulas; both scales [...]."""
    V = logits.shape[-1]
    there = (tokens >= 0) & (tokens < V)
    y = _log_softmax(logits.double() / temperature)
    p = y.exp()
    _, H = token_logprobs(logits, tokens, temperature)
    s, h = scale.double()[..., None], entropy_scale.double()[..., None]
    one = torch.zeros_like(y).scatter_(-1, tokens.clamp(0, V - 1)[..., None], 1.0)
    slope = torch.where(p == 0, torch.zeros_like(p), p * (y + H[..., None]))
    g = (s * (one - p) - h * slope) / temperature
    none = ~there | (logits == -torch.inf).all(-1) | ((scale == 0) & (entropy_scale == 0))
    return torch.where(none[..., None], torch.zeros_like(g), g)
