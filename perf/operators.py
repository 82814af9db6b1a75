"""The operators on rows of logits between a large model and a small one, as cases that can be timed and compared.

* ``kernels.top_logits``: what a teacher hands on of each row (its k largest logits, their token ids, log-sum-exp).
* ``torch.ops.rwkv_tl.distill_loss`` / ``kernels.distill_loss`` / ``kernels.distill_loss_grad``: the divergence of a
  student's distribution from a teacher's top logits, its gradient, and both in one pass.
* ``verify_draft``: drafted tokens against the target's probabilities, from given random numbers.

``listed`` holds the cases, ``draw`` makes more of the same ranges, ``prepare`` builds what a program holds before the
call, ``run`` is one pass, ``work`` its unavoidable bytes and operations, and ``exact`` the same outputs in 64 bits.
With ``own`` false ``run`` computes the plain form: elementary torch operations in 32 bits (in 64 for a loss's sums, and
for the verification, where whole tokens hang on borders between sums of up to 65536 probabilities).
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
LEAST_REST = 2.0**-20  # a teacher's mass outside its top logits below this is none: a float32 log-sum-exp cannot tell it


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # the alternatives of one served token, beside its sampling: all latency
        {"name": "top_1", "kind": "top", "dtype": "f16", "N": 1, "V": 65536, "K": 20, "T": 1.0},
        # a teacher's answers of one ragged document
        {"name": "top_509", "kind": "top", "dtype": "bf16", "N": 509, "V": 65536, "K": 64, "T": 1.0},
        # four documents of 1024 tokens for a softened distillation, many logits a token
        {"name": "top_4096_k200", "kind": "top", "dtype": "bf16", "N": 4096, "V": 65536, "K": 200, "T": 2.0},
        # a float32 head of a small odd vocabulary
        {"name": "top_257_f32", "kind": "top", "dtype": "f32", "N": 257, "V": 20011, "K": 100, "T": 1.0},
        # evaluation of a student on a few rows: the loss alone
        {"name": "loss_16", "kind": "loss", "dtype": "f16", "N": 16, "V": 65536, "K": 20, "T": 1.0, "rest": False, "pad": 0.0},
        # a student's training step through autograd, padded rows among them, half precision
        {"name": "train_1021", "kind": "train", "dtype": "f16", "N": 1021, "V": 65536, "K": 50, "T": 1.0, "rest": False, "pad": 0.1},
        # the same in float32 with a softened teacher and the mass outside its top logits
        {"name": "train_331_f32", "kind": "train", "dtype": "f32", "N": 331, "V": 20011, "K": 100, "T": 2.0, "rest": True, "pad": 0.1},
        # four sequences of 1024 tokens, loss and gradient in one call: the largest
        {"name": "both_4096", "kind": "both", "dtype": "bf16", "N": 4096, "V": 65536, "K": 64, "T": 1.0, "rest": True, "pad": 0.05},
        # one conversation's four drafted tokens: the smallest verification, all latency
        {"name": "verify_1x4", "kind": "verify", "dtype": "f16", "B": 1, "K": 4, "V": 65536, "T": 1.0, "Td": 1.0, "ragged": False},
        # sixteen conversations with drafts of up to eight tokens, a draft model sharper than the target
        {"name": "verify_16x8", "kind": "verify", "dtype": "f16", "B": 16, "K": 8, "V": 65536, "T": 0.9, "Td": 0.7, "ragged": True},
        # greedy drafts (no draft distribution) of a greedy batch
        {"name": "verify_greedy_33x5", "kind": "verify", "dtype": "bf16", "B": 33, "K": 5, "V": 65536, "T": 0.0, "Td": 0.0, "ragged": True},
        # a wide serving batch
        {"name": "verify_96x7", "kind": "verify", "dtype": "bf16", "B": 96, "K": 7, "V": 65536, "T": 1.0, "Td": 1.0, "ragged": True},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["top", "top", "loss", "train", "train", "both", "verify", "verify"])
    V = 65536 if rng.random() < 0.6 else _log(rng, 1000, 65536)
    T = rng.choice([1.0, 1.0, 0.8, 1.5, 2.0])
    if kind == "verify":
        c = {"kind": kind, "dtype": rng.choice(["f16", "bf16", "f32"]), "B": _log(rng, 1, 96), "K": rng.randint(1, 8), "V": V,
             "T": T, "Td": rng.choice([T, T, 0.7, 0.0]), "ragged": rng.random() < 0.5}
        return {**c, "T": 0.0, "Td": 0.0} if rng.random() < 0.25 else c
    c = {"kind": kind, "dtype": rng.choice(["f16", "bf16", "bf16", "f32"]), "N": _log(rng, 1, 2048), "V": V}
    if kind == "top":
        return {**c, "K": _log(rng, 1, 256), "T": T}
    return {**c, "K": _log(rng, 1, 512), "T": T, "rest": rng.random() < 0.5, "pad": rng.choice([0.0, 0.1, 0.3])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _zipf(g: torch.Generator, *shape: int) -> torch.Tensor:
    """Logits whose probabilities fall with their rank as r^-1.3, as tokens' do, in a random order of the ids."""
    return torch.empty(*shape, device=DEV).exponential_(generator=g).log_().mul_(-1.3)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, V = DTYPES[case["dtype"]], case["V"]
    s: dict = {"case": case}
    if case["kind"] == "verify":
        B, K, Td = case["B"], case["K"], case["Td"]
        target = _zipf(g, B, K + 1, V)
        draft = (target[:, :K] + 0.7 * torch.randn(B, K, V, generator=g, device=DEV)).to(dt)
        s["target"] = target.to(dt)
        x = draft.float()
        if Td > 0:  # drafted by sampling: the Gumbel maximum
            x = x / Td - torch.empty_like(x).exponential_(generator=g).log_()
        s["tokens"] = x.argmax(-1)
        s["draft"] = draft if Td > 0 else None
        s["uniforms"] = torch.rand(B, K + 1, generator=g, device=DEV)
        s["lengths"] = torch.randint(0, K + 1, (B,), generator=g, device=DEV) if case["ragged"] else None
        return s
    N, K = case["N"], case["K"]
    z = _zipf(g, N, V)
    if case["kind"] == "top":
        s["logits"] = z.to(dt)
        return s
    s["logits"] = (z + 0.7 * torch.randn(N, V, generator=g, device=DEV) - 1.5).to(dt)
    s["top_val"], s["top_idx"] = z.to(dt).topk(K)
    s["lse"] = torch.logsumexp(z / case["T"], -1) if case["rest"] else None
    if case["pad"]:  # rows without a teacher, and rows with fewer of its logits
        keep = torch.randint(1, K + 1, (N,), generator=g, device=DEV)
        keep[torch.rand(N, generator=g, device=DEV) < 0.5] = K
        keep[torch.rand(N, generator=g, device=DEV) < case["pad"]] = 0
        s["top_idx"].masked_fill_(torch.arange(K, device=DEV) >= keep[:, None], -1)
    s["scale"] = torch.rand(N, generator=g, device=DEV) / N * 256.0  # the loss's weights, and a loss scale
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _lse(z: torch.Tensor) -> torch.Tensor:
    m = z.amax(-1)
    return m + (z - m[..., None]).exp().sum(-1).log()


def _ordered(x: torch.Tensor) -> torch.Tensor:
    """Whole numbers in the order of the logits, and of ties by the lowest id first: no two of a row are alike."""
    i = (x.float() + 0.0).view(torch.int32)
    i = torch.where(i < 0, i ^ 0x7FFFFFFF, i).long()
    return (i << 17) - torch.arange(x.shape[-1], device=x.device)


def _plain_top(logits, K, T):
    idx = _ordered(logits).topk(K).indices
    return logits.gather(-1, idx), idx, _lse(logits.float() / T)


def _plain_distill(logits, top_val, top_idx, lse, T, scale):
    """The loss of each row, and with `scale` (the rows' upstream gradients) the gradient. The few values of the
    teacher's entries and the sums over a row are in 64 bits: the loss is what is left of sums that nearly cancel."""
    N, V = logits.shape
    x = logits.float()
    m = x.amax(-1)
    e = ((x - m[:, None]) / T).exp()
    Z = e.sum(-1, dtype=torch.float64)
    L = m.double() / T + Z.log()
    there = (top_idx >= 0) & (top_idx < V)
    some = there.any(-1)
    at = top_idx.clamp(0, V - 1)
    t = top_val.double() / T
    if lse is None:
        t = t.masked_fill(~there, -torch.inf)
        t_lse = torch.where(some, _lse(torch.where(some[:, None], t, 0.0)), 0.0)
    else:
        t_lse = lse
    logp = t - t_lse[:, None]
    p = torch.where(there, logp.exp(), 0.0)
    P = p.sum(-1)
    loss = torch.where(there, p * (logp - logits.gather(1, at).double() / T + L[:, None]), 0.0).sum(-1)
    inside = torch.zeros(N, V + 1, dtype=torch.bool, device=x.device)
    inside = inside.scatter_(1, torch.where(there, at, V), True)[:, :V]
    R = torch.zeros_like(P)
    share = torch.zeros_like(P)
    if lse is not None:
        R = (1.0 - P).clamp_min(0.0)
        R = torch.where(some & (R >= LEAST_REST), R, 0.0)
        outside = torch.where(inside, 0.0, e).sum(-1, dtype=torch.float64) / Z
        loss = loss + torch.where(R > 0, R * (R.log() - outside.log()), 0.0)
        share = torch.where(R > 0, R / outside, 0.0)
    loss = torch.where(some, loss, 0.0)
    if scale is None:
        return loss.float()
    grad = e * torch.where(inside, ((P + R) / Z).float()[:, None], ((P + R - share) / Z).float()[:, None])
    grad.scatter_add_(1, at, -p.float())
    grad = torch.where(some[:, None], grad * (scale / T)[:, None], 0.0)
    return loss.float(), grad.to(logits.dtype)


def _first_max(x: torch.Tensor) -> torch.Tensor:
    V = x.shape[-1]
    at = torch.arange(V, device=x.device)
    return torch.where(x == x.amax(-1, keepdim=True), at, V).amin(-1)


def _plain_verify(target, tokens, uniforms, draft, T, Td, lengths):
    B, K = tokens.shape
    V = target.shape[-1]
    step = torch.arange(K, device=tokens.device)
    drafted = step < (K if lengths is None else lengths[:, None])
    row = torch.arange(B, device=tokens.device)
    if T <= 0:
        best = _first_max(target)
        ok = (tokens == best[:, :K]) & drafted
        n = ok.long().cumprod(1).sum(1)
        nxt = best[row, n]
    else:
        z = target.double() / T
        p = (z - z.amax(-1, keepdim=True)).exp()
        p /= p.sum(-1, keepdim=True)
        if draft is None:
            q = torch.zeros_like(p[:, :K]).scatter_(2, tokens[..., None], 1.0)
        else:
            z = draft.double() / Td
            q = (z - z.amax(-1, keepdim=True)).exp()
            q /= q.sum(-1, keepdim=True)
        px = p[:, :K].gather(2, tokens[..., None])[..., 0]
        qx = q.gather(2, tokens[..., None])[..., 0]
        ok = (uniforms[:, :K].double() * qx < px) & drafted
        n = ok.long().cumprod(1).sum(1)
        pn = p[row, n]
        rejected = n < (K if lengths is None else lengths)
        r = torch.where(rejected[:, None], (pn - q[row, n.clamp_max(K - 1)]).clamp_min(0.0), pn)
        r = torch.where(r.sum(-1, keepdim=True) > 0, r, pn)
        c = r.cumsum(-1)
        above = c > uniforms[:, K, None].double() * c[:, -1:]
        last = torch.where(r > 0, torch.arange(V, device=r.device), 0).amax(-1)
        nxt = torch.where(above.any(-1), V - above.sum(-1), last)
    at = torch.arange(K + 1, device=tokens.device)
    out = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(at < n[:, None], out, torch.where(at == n[:, None], nxt[:, None], -1))
    return out, n


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
    pkg, c = _package(), s["case"]
    if c["kind"] == "top":
        return pkg.kernels.top_logits(s["logits"], c["K"], temperature=c["T"])
    if c["kind"] == "verify":
        return pkg.verify_draft(s["target"], s["tokens"], s["uniforms"], s["draft"], temperature=c["T"],
                                draft_temperature=c["Td"], lengths=s["lengths"])
    if c["kind"] == "loss":
        return pkg.kernels.distill_loss(s["logits"], s["top_val"], s["top_idx"], s["lse"], temperature=c["T"])
    if c["kind"] == "both":
        return pkg.kernels.distill_loss_grad(s["logits"], s["top_val"], s["top_idx"], s["lse"], temperature=c["T"],
                                             scale=s["scale"])
    x = s["logits"].detach().requires_grad_()
    loss = torch.ops.rwkv_tl.distill_loss(x, s["top_val"], s["top_idx"], s["lse"], c["T"])
    return loss.detach(), *torch.autograd.grad(loss, x, s["scale"])


def run(state: dict):
    if own:
        return _own(state)
    s, c = state, state["case"]
    if c["kind"] == "top":
        return _plain_top(s["logits"], c["K"], c["T"])
    if c["kind"] == "verify":
        return _plain_verify(s["target"], s["tokens"], s["uniforms"], s["draft"], c["T"], c["Td"], s["lengths"])
    return _plain_distill(s["logits"], s["top_val"], s["top_idx"], s["lse"], c["T"], None if c["kind"] == "loss" else s["scale"])


def work(case: dict) -> dict:
    e, V, K = BYTES[case["dtype"]], case["V"], case["K"]
    if case["kind"] == "verify":
        B = case["B"]
        drafted = K if case["T"] > 0 and case["Td"] > 0 else 0
        rows = B * (K + 1 + drafted)
        # a row: an exponential and a sum an element (greedy: a comparison)
        return {"bytes": rows * V * e + B * (8 * K + 4 * (K + 1) + 8 * (K + 1) + 8), "flops": rows * V * (16 if case["T"] > 0 else 1)}
    N = case["N"]
    if case["kind"] == "top":
        return {"bytes": N * (V * e + K * (e + 8) + 4), "flops": N * V * 5}
    top = N * (K * (e + 8) + 4 + (4 if case["rest"] else 0))
    if case["kind"] == "loss":
        return {"bytes": N * V * e + top, "flops": N * V * 4}
    return {"bytes": 2 * N * V * e + top + 4 * N, "flops": N * V * 8}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_top(s: dict):
    c, x = s["case"], s["logits"]
    vals, ids, ls = [], [], []
    for rows in x.split(max(1, (1 << 24) // c["V"])):
        d = rows.double()
        v, i = torch.sort(d, dim=-1, descending=True, stable=True)  # stable: ties stay in the order of their ids
        vals.append(v[:, : c["K"]])
        ids.append(i[:, : c["K"]])
        ls.append(torch.logsumexp(d / c["T"], -1))
    return torch.cat(vals), torch.cat(ids), torch.cat(ls)


def _exact_distill(s: dict):
    """With y = log softmax of the student: sum over the teacher's entries of p (log p - y), and the rest's term; its
    derivative by the chain rule through y."""
    c = s["case"]
    N, V = s["logits"].shape
    losses, grads = [], []
    n = max(1, (1 << 25) // V)
    for r in range(0, N, n):
        y = torch.log_softmax(s["logits"][r : r + n].double() / c["T"], -1)
        idx = s["top_idx"][r : r + n]
        live = idx >= 0
        t = (s["top_val"][r : r + n].double() / c["T"]).masked_fill(~live, -torch.inf)
        norm = torch.logsumexp(t, -1) if s["lse"] is None else s["lse"][r : r + n].double()
        logp = t - torch.where(live.any(-1), norm, 0.0)[:, None]
        teacher = torch.zeros(y.shape[0], V + 1, dtype=torch.float64, device=y.device)
        teacher.scatter_(1, torch.where(live, idx, V), logp.exp().masked_fill(~live, 0.0))
        inside = torch.zeros(y.shape[0], V + 1, dtype=torch.bool, device=y.device).scatter_(1, torch.where(live, idx, V), live)
        teacher, inside = teacher[:, :V], inside[:, :V]
        loss = (torch.special.xlogy(teacher, teacher) - teacher * y).sum(-1)
        dy = -teacher  # derivative by y where y are taken as free
        if s["lse"] is not None:
            rest = (1.0 - teacher.sum(-1)).clamp_min(0.0)
            rest = torch.where(rest < LEAST_REST, 0.0, rest) * live.any(-1)
            log_out = torch.logsumexp(y.masked_fill(inside, -torch.inf), -1)
            loss = loss + torch.where(rest > 0, torch.special.xlogy(rest, rest) - rest * log_out, 0.0)
            dy = dy - (rest[:, None] * (y - log_out[:, None]).exp()).masked_fill(inside | (rest[:, None] == 0), 0.0)
        losses.append(loss)
        if c["kind"] != "loss":
            g = dy - y.exp() * dy.sum(-1, keepdim=True)
            grads.append(g * (s["scale"][r : r + n].double() / c["T"])[:, None])
    return torch.cat(losses) if c["kind"] == "loss" else (torch.cat(losses), torch.cat(grads))


def _exact_verify(s: dict):
    """One conversation after the other, one drafted token after the other."""
    c, K = s["case"], s["case"]["K"]
    toks, counts = [], []
    tokens, u = s["tokens"].tolist(), s["uniforms"].double()
    for b in range(c["B"]):
        length = K if s["lengths"] is None else int(s["lengths"][b])
        seq: list[int] = []
        for i in range(length + 1):
            row = s["target"][b, i].double()
            last = i == length
            if c["T"] <= 0:
                best = int((row == row.max()).nonzero()[0])
                seq.append(best)
                if last or tokens[b][i] != best:
                    break
                continue
            p = torch.softmax(row / c["T"], -1)
            if last:
                r = p
            else:
                x = tokens[b][i]
                if s["draft"] is None:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                else:
                    q = torch.softmax(s["draft"][b, i].double() / c["Td"], -1)
                if float(u[b, i] * q[x]) < float(p[x]):
                    seq.append(x)
                    continue
                r = (p - q).clamp_min(0.0)
                r = r if float(r.sum()) > 0 else p
            cum = r.cumsum(0)
            seq.append(int(torch.searchsorted(cum, u[b, K] * cum[-1], right=True).clamp_max(c["V"] - 1)))
            break
        counts.append(len(seq) - 1)
        toks.append(seq + [-1] * (K + 1 - len(seq)))
    return torch.tensor(toks), torch.tensor(counts)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "top":
        return _exact_top(s)
    if case["kind"] == "verify":
        return _exact_verify(s)
    return _exact_distill(s)
