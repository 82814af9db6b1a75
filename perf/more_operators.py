"""The two ends and the norms of a training step around the DPLR recurrence, as cases that can be timed and compared.

* ``kernels.embed`` / ``kernels.embed_backward`` / ``torch.ops.rwkv_tl.embed``: rows of an embedding table times a
  factor, and the table's gradient, each token's rows added up in the order of their positions.
* ``kernels.layer_norm_forward`` / ``kernels.layer_norm_backward`` / ``torch.ops.rwkv_tl.layer_norm``: LayerNorm that
  keeps its statistics, and its gradients to the input, the weight and the bias.
* ``kernels.token_logprobs`` / ``kernels.token_logprobs_grad`` / ``torch.ops.rwkv_tl.token_logprobs``: the log
  probability of a given token of each row of logits, the row's entropy, its most likely alternatives, and the gradient.

``listed`` holds the cases, ``draw`` makes more of the same ranges, ``prepare`` builds what a program holds before the
call, ``run`` is one pass, ``work`` its unavoidable bytes and operations, and ``exact`` the same outputs in 64 bits.
With ``own`` false ``run`` computes the plain form: elementary torch operations in 32 bits (in 64 for a row's sums over
a vocabulary, since the logarithm of a likely token's probability is what is left of nearly equal numbers).
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-5


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # the tokens of sixteen conversations entering one step: all latency
        {"name": "embed_16", "kind": "embed", "dtype": "f16", "N": 16, "V": 65536, "C": 2048, "scale": 1.0, "pad": 0.0},
        # one document's gradient of a small odd table in float32, padded positions among its tokens
        {"name": "embed_grad_509_f32", "kind": "embed_grad", "dtype": "f32", "N": 509, "V": 20011, "C": 768, "scale": 1.0,
         "pad": 0.1},
        # a micro-batch of eight sequences of 1024 tokens
        {"name": "embed_grad_8192", "kind": "embed_grad", "dtype": "bf16", "N": 8192, "V": 65536, "C": 1024, "scale": 1.0,
         "pad": 0.0},
        # a large batch of a scaled table through autograd: lookup and gradient
        {"name": "embed_train_16384", "kind": "embed_train", "dtype": "bf16", "N": 16384, "V": 65536, "C": 2048,
         "scale": 2048**0.5, "pad": 0.05},
        # the norm of a few rows, as a small evaluation step has it: all latency
        {"name": "norm_7", "kind": "norm", "dtype": "f16", "N": 7, "C": 2048, "w_f32": True},
        # the gradient of a ragged batch in float32, of a width no power of two divides
        {"name": "norm_grad_331_f32", "kind": "norm_grad", "dtype": "f32", "N": 331, "C": 1001, "w_f32": True},
        # a training step's norm through autograd, float32 weights beside bfloat16 activations
        {"name": "norm_train_4096", "kind": "norm_train", "dtype": "bf16", "N": 4096, "C": 2048, "w_f32": True},
        # the gradient over a large batch: the reduction of the weight's gradient over many rows
        {"name": "norm_grad_16384", "kind": "norm_grad", "dtype": "bf16", "N": 16384, "C": 2048, "w_f32": False},
        # one served token with its alternatives: all latency
        {"name": "score_1", "kind": "score", "dtype": "f16", "N": 1, "V": 65536, "K": 20, "T": 1.0, "pad": 0.0},
        # the score of one ragged document with five alternatives a token
        {"name": "score_2039", "kind": "score", "dtype": "bf16", "N": 2039, "V": 65536, "K": 5, "T": 1.0, "pad": 0.0},
        # a policy's step through autograd: weighted log probabilities and an entropy bonus, padded rows, float32
        {"name": "policy_train_331_f32", "kind": "policy_train", "dtype": "f32", "N": 331, "V": 20011, "T": 1.0, "pad": 0.1},
        # next-token training on four sequences of 1024 tokens, loss and gradient in one call: the largest
        {"name": "token_grad_4096", "kind": "token_grad", "dtype": "bf16", "N": 4096, "V": 65536, "T": 1.0, "pad": 0.05},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "embed_train", "norm", "norm_grad", "norm_grad", "norm_train",
                       "score", "score", "policy_train", "token_grad"])
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    V = 65536 if rng.random() < 0.5 else _log(rng, 1000, 65536)
    pad = rng.choice([0.0, 0.0, 0.05, 0.2])
    if kind.startswith("embed"):
        C = rng.choice([768, 1024, 2048, _log(rng, 64, 2048)])
        return {"kind": kind, "dtype": dtype, "N": _log(rng, 1, 16384), "V": V, "C": C,
                "scale": rng.choice([1.0, 1.0, C**0.5]), "pad": pad}
    if kind.startswith("norm"):
        C = rng.choice([768, 1024, 2048, _log(rng, 64, 4096), _log(rng, 64, 4096)])
        return {"kind": kind, "dtype": dtype, "N": _log(rng, 1, 16384), "C": C, "w_f32": rng.random() < 0.5}
    c = {"kind": kind, "dtype": dtype, "N": _log(rng, 1, 2048), "V": V, "T": rng.choice([1.0, 1.0, 0.7, 1.5]), "pad": pad}
    return {**c, "K": rng.choice([0, 0, 5, 20, _log(rng, 1, 200)])} if kind == "score" else c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _tokens(g: torch.Generator, N: int, V: int, pad: float) -> torch.Tensor:
    """Ids as often as ranks of words are, the n-th about 1 / n times the first; -1 at padded positions."""
    u = torch.rand(N, generator=g, device=DEV, dtype=torch.float64)
    t = ((u * math.log(V + 1)).exp() - 1.0).long().clamp_(0, V - 1)
    return t.masked_fill_(torch.rand(N, generator=g, device=DEV) < pad, -1) if pad else t


def _activations(g: torch.Generator, N: int, C: int) -> torch.Tensor:
    """Rows of a residual stream: channels of unlike sizes, a few large, about a mean of their own."""
    size = (torch.randn(C, generator=g, device=DEV) * 0.6).exp()
    mean = torch.randn(C, generator=g, device=DEV) * 0.3
    return torch.randn(N, C, generator=g, device=DEV) * size + mean


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, kind = DTYPES[case["dtype"]], case["kind"]
    s: dict = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if kind.startswith("embed"):
        N, V, C = case["N"], case["V"], case["C"]
        s["tokens"] = _tokens(g, N, V, case["pad"])
        if kind != "embed_grad":
            s["weight"] = (normal(V, C) * 0.02).to(dt)
        if kind != "embed":
            s["grad"] = (normal(N, C) * 0.05).to(dt)
        return s
    if kind.startswith("norm"):
        N, C = case["N"], case["C"]
        wdt = torch.float32 if case["w_f32"] else dt
        s["x"] = _activations(g, N, C).to(dt)
        s["weight"] = (1.0 + 0.1 * normal(C)).to(wdt)
        s["bias"] = (0.05 * normal(C)).to(wdt)
        if kind != "norm":
            s["grad"] = (normal(N, C) * 0.05).to(dt)
        if kind == "norm_grad":  # what the forward pass kept
            s["mean"], s["rstd"] = _stats(s["x"])
        return s
    N, V = case["N"], case["V"]
    # probabilities that fall with their rank as r^-1.3, as tokens' do, in a random order of the ids
    z = torch.empty(N, V, device=DEV).exponential_(generator=g).log_().mul_(-1.3)
    s["logits"] = z.to(dt)
    # a token drawn from them (the Gumbel maximum)
    s["tokens"] = (z - torch.empty_like(z).exponential_(generator=g).log_()).argmax(-1)
    if case["pad"]:
        s["tokens"].masked_fill_(torch.rand(N, generator=g, device=DEV) < case["pad"], -1)
    # advantages or weights of the rows, and an entropy bonus, with a loss scale
    s["scale"] = normal(N) / N * 256.0 if kind == "policy_train" else torch.full((N,), -256.0 / N, device=DEV)
    s["entropy_scale"] = torch.full((N,), -0.01 * 256.0 / N, device=DEV) if kind == "policy_train" else None
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _plain_embed(weight, tokens, scale):
    V = weight.shape[0]
    there = (tokens >= 0) & (tokens < V)
    rows = weight[tokens.clamp(0, V - 1)].float() * scale
    return torch.where(there[:, None], rows, 0.0).to(weight.dtype)


def _plain_embed_grad(grad, tokens, V, scale):
    there = (tokens >= 0) & (tokens < V)
    out = torch.zeros(V + 1, grad.shape[1], device=grad.device)
    out.index_add_(0, torch.where(there, tokens, V), grad.float())
    return (out[:V] * scale).to(grad.dtype)


def _stats(x):
    x = x.float()
    mean = x.mean(-1)
    return mean, ((x - mean[:, None]).square().mean(-1) + EPS).rsqrt()


def _plain_norm(x, weight, bias):
    mean, rstd = _stats(x)
    y = (x.float() - mean[:, None]) * rstd[:, None] * weight.float() + bias.float()
    return y.to(x.dtype), mean, rstd


def _plain_norm_grad(grad, x, weight, mean, rstd):
    dy = grad.float()
    xh = (x.float() - mean[:, None]) * rstd[:, None]
    gw = dy * weight.float()
    dx = rstd[:, None] * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), (dy * xh).sum(0).to(weight.dtype), dy.sum(0).to(weight.dtype)


def _ordered(x: torch.Tensor) -> torch.Tensor:
    """Whole numbers in the order of the logits, and of ties by the lowest id first: no two of a row are alike."""
    i = (x.float() + 0.0).view(torch.int32)
    i = torch.where(i < 0, i ^ 0x7FFFFFFF, i).long()
    return (i << 17) - torch.arange(x.shape[-1], device=x.device)


def _plain_logprobs(logits, tokens, T, K=0, scale=None, entropy_scale=None):
    """Log probability of each row's token and the row's entropy; with K the most likely alternatives, with `scale`
    (and `entropy_scale`), the rows' upstream gradients, the gradient. Sums over a row are in 64 bits."""
    V = logits.shape[1]
    there = (tokens >= 0) & (tokens < V)
    at = tokens.clamp(0, V - 1)[:, None]
    d = logits.float()
    m = d.amax(-1, keepdim=True)
    d = (d - m) / T
    e = d.exp()
    Z = e.sum(-1, keepdim=True, dtype=torch.float64)
    log_z = Z.log()
    mean = (e * d.clamp_min(-1e4)).sum(-1, keepdim=True, dtype=torch.float64) / Z
    logp = torch.where(there, (d.gather(1, at).double() - log_z)[:, 0], 0.0).float()
    entropy = torch.where(there, (log_z - mean)[:, 0], 0.0).float()
    out = [logp, entropy]
    if K:
        idx = _ordered(logits).topk(K).indices
        out.append(torch.where(there[:, None], d.gather(1, idx).double() - log_z, -torch.inf).float())
        out.append(torch.where(there[:, None], idx, -1))
    if scale is not None:
        # d (s l + h H) / d z_j = 1/T (s (token) - q_j (s + h (log q_j + H)))
        q = (e / Z).float()
        f = scale.double()[:, None].expand_as(Z)
        if entropy_scale is not None:
            f = f - entropy_scale.double()[:, None] * mean
            grad = -q * (f.float() + entropy_scale[:, None] * d.clamp_min(-1e4))
        else:
            grad = -q * f.float()
        grad.scatter_add_(1, at, scale[:, None])
        out.append(torch.where(there[:, None], grad / T, 0.0).to(logits.dtype))
    return tuple(out)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

_PACKAGE: list = []


def _package():
    """The framework, imported once and only where its kernels run."""
    if not _PACKAGE:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "rwkv-tl_amd"))
        tree = Path.cwd() / "rwkv-tl_amd"
        if tree.is_dir():
            sys.path.insert(0, str(tree))
        import rwkv_tl_amd

        _PACKAGE.append(rwkv_tl_amd)
    return _PACKAGE[0]


def _own(s: dict):
    kernels, c = _package().kernels, s["case"]
    kind, ops = c["kind"], torch.ops.rwkv_tl
    if kind == "embed":
        return kernels.embed(s["weight"], s["tokens"], scale=c["scale"])
    if kind == "embed_grad":
        return kernels.embed_backward(s["grad"], s["tokens"], c["V"], scale=c["scale"])
    if kind == "embed_train":
        w = s["weight"].detach().requires_grad_()
        y = ops.embed(w, s["tokens"], c["scale"])
        return y.detach(), *torch.autograd.grad(y, w, s["grad"])
    if kind == "norm":
        return kernels.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=EPS)
    if kind == "norm_grad":
        return kernels.layer_norm_backward(s["grad"], s["x"], s["weight"], s["mean"], s["rstd"])
    if kind == "norm_train":
        x, w, b = (s[k].detach().requires_grad_() for k in ("x", "weight", "bias"))
        y = ops.layer_norm(x, w, b, EPS)
        return y.detach(), *torch.autograd.grad(y, (x, w, b), s["grad"])
    if kind == "score":
        return kernels.token_logprobs(s["logits"], s["tokens"], c["K"], temperature=c["T"])
    if kind == "token_grad":
        return kernels.token_logprobs_grad(s["logits"], s["tokens"], temperature=c["T"], scale=s["scale"])
    x = s["logits"].detach().requires_grad_()
    logp, entropy = ops.token_logprobs(x, s["tokens"], c["T"])
    grads = torch.autograd.grad((logp, entropy), x, (s["scale"], s["entropy_scale"]))
    return logp.detach(), entropy.detach(), *grads


def run(state: dict):
    if own:
        return _own(state)
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "embed":
        return _plain_embed(s["weight"], s["tokens"], c["scale"])
    if kind == "embed_grad":
        return _plain_embed_grad(s["grad"], s["tokens"], c["V"], c["scale"])
    if kind == "embed_train":
        return _plain_embed(s["weight"], s["tokens"], c["scale"]), _plain_embed_grad(s["grad"], s["tokens"], c["V"], c["scale"])
    if kind == "norm":
        return _plain_norm(s["x"], s["weight"], s["bias"])
    if kind == "norm_grad":
        return _plain_norm_grad(s["grad"], s["x"], s["weight"], s["mean"], s["rstd"])
    if kind == "norm_train":
        y, mean, rstd = _plain_norm(s["x"], s["weight"], s["bias"])
        return y, *_plain_norm_grad(s["grad"], s["x"], s["weight"], mean, rstd)
    if kind == "score":
        return _plain_logprobs(s["logits"], s["tokens"], c["T"], c["K"])
    return _plain_logprobs(s["logits"], s["tokens"], c["T"], 0, s["scale"], s["entropy_scale"])


def work(case: dict) -> dict:
    kind, N, e = case["kind"], case["N"], BYTES[case["dtype"]]
    if kind.startswith("embed"):
        C, V = case["C"], case["V"]
        look, back = 2 * N * C * e + 8 * N, N * C * e + 8 * N + V * C * e
        b = {"embed": look, "embed_grad": back, "embed_train": look + back - 8 * N}[kind]
        return {"bytes": b, "flops": N * C * (2 if kind == "embed_train" else 1)}
    if kind.startswith("norm"):
        C = case["C"]
        w = C * (4 if case["w_f32"] else e)
        # (a step needs its forward pass's result and statistics, and reads x again)
        ahead, back = 2 * N * C * e + 2 * w + 8 * N, 3 * N * C * e + 3 * w + 8 * N
        b = {"norm": ahead, "norm_grad": back, "norm_train": 4 * N * C * e + 4 * w}[kind]
        return {"bytes": b, "flops": N * C * {"norm": 8, "norm_grad": 14, "norm_train": 22}[kind]}
    V = case["V"]
    b = N * (V * e + 16)
    if kind == "score":
        return {"bytes": b + 12 * N * case["K"], "flops": N * V * 6}
    return {"bytes": b + N * V * e + 4 * N * (2 if kind == "policy_train" else 1), "flops": N * V * 10}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_embed(s: dict):
    """By a table with a row of zeros behind the vocabulary, and its derivative by adding at sorted places."""
    c, t = s["case"], s["tokens"]
    V = c["V"]
    t = torch.where((t < 0) | (t >= V), V, t)
    out = []
    if "weight" in s:
        table = torch.cat([s["weight"].double(), torch.zeros(1, c["C"], dtype=torch.float64, device=DEV)])
        out.append(c["scale"] * table.index_select(0, t))
        del table
    if "grad" in s:
        order = torch.argsort(t, stable=True)
        ids, counts = torch.unique_consecutive(t[order], return_counts=True)
        rows = s["grad"].double()[order]
        sums = torch.segment_reduce(rows, "sum", lengths=counts) * c["scale"]
        back = torch.zeros(V + 1, c["C"], dtype=torch.float64, device=DEV)
        back[ids] = sums
        out.append(back[:V])
    return out[0] if len(out) == 1 else tuple(out)


def _exact_norm(s: dict):
    kind = s["case"]["kind"]
    x, w, b = (s[k].double().requires_grad_() for k in ("x", "weight", "bias"))
    mean = x.sum(-1, keepdim=True) / x.shape[-1]
    var = ((x - mean) ** 2).sum(-1, keepdim=True) / x.shape[-1]
    rstd = 1.0 / torch.sqrt(var + EPS)
    y = (x - mean) * rstd * w + b
    if kind == "norm":
        return y.detach(), mean.detach()[:, 0], rstd.detach()[:, 0]
    grads = torch.autograd.grad(y, (x, w, b), s["grad"].double())
    return grads if kind == "norm_grad" else (y.detach(), *grads)


def _exact_logprobs(s: dict):
    """Through log softmax; the gradient by the chain rule through it."""
    c, kind = s["case"], s["case"]["kind"]
    K = c.get("K", 0)
    N, V = s["logits"].shape
    parts = []
    n = max(1, (1 << 25) // V)
    for r in range(0, N, n):
        z, t = s["logits"][r : r + n].double(), s["tokens"][r : r + n]
        live = (t >= 0) & (t < V)
        y = torch.log_softmax(z / c["T"], -1)
        p = y.exp()
        H = -(p * y).sum(-1)
        at = torch.where(live, t, 0)[:, None]
        part = [y.gather(1, at)[:, 0] * live, H * live]
        if K:
            i = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :K]  # stable: ties in the ids' order
            part += [y.gather(1, i).masked_fill(~live[:, None], -torch.inf), i.masked_fill(~live[:, None], -1)]
        if kind != "score":
            # d / dy: the token's weight, and the entropy's -(log p + 1) p as a sum over p y with p = exp(y)
            dy = torch.zeros_like(y).scatter_(1, at, s["scale"][r : r + n].double()[:, None])
            if s["entropy_scale"] is not None:
                dy -= s["entropy_scale"][r : r + n].double()[:, None] * p * (y + 1.0)
            dz = (dy - p * dy.sum(-1, keepdim=True)) / c["T"]
            part.append(dz * live[:, None])
        parts.append(part)
    return tuple(torch.cat(x) for x in zip(*parts))


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"].startswith("embed"):
        return _exact_embed(s)
    if case["kind"].startswith("norm"):
        return _exact_norm(s)
    return _exact_logprobs(s)
