"""The HIP operators registered with ``torch.library`` as ``torch.ops.rwkv_tl.*``.

Drop-in for ``rwkv_tl.operators`` (``src/rwkv_tl/operators/__init__.py:112-375``):
the same namespace, operator names and schemas, with in-place arguments
declared ``Tensor(a!)``, so code written against ``torch.ops.rwkv_tl`` (as
``demo/_rwkv7_base.py:115-119,149,281`` is) runs on the HIP kernels and can be
traced by ``torch.compile``.

Each operator has two implementations:

* ``CUDA`` (the ROCm device in PyTorch-ROCm): the ``rwkv_tl_amd.kernels``
  function of the same name, i.e. one C-ABI call into ``librwkv7_hip.so``.
* ``Meta``: outputs of the right shape and dtype with no data, which is what
  ``torch.compile`` / FakeTensor tracing runs.

There is no ``CPU`` implementation (the reference has a plain-torch one): a
CPU tensor raises torch's "no kernel for the CPU backend" error instead of
silently taking another code path.

Importing this module registers the operators once per process. It uses the
reference's ``rwkv_tl`` namespace, so it cannot be imported into a process
that has already imported ``rwkv_tl`` itself.
"""

from __future__ import annotations

from collections.abc import Callable

import torch
from torch import Tensor

from . import kernels as K
from . import training as T

NAMESPACE = "rwkv_tl"

# name -> (schema, CUDA implementation, Meta implementation)
_T = "Tensor"


def _like(n: int) -> Callable[..., tuple[Tensor, ...]]:
    return lambda x, *_: tuple(torch.empty_like(x) for _ in range(n))


def _dplr(S, R, W, K_, V, A, B) -> Tensor:
    y, _ = K.fused_dplr(S, R, W, K_, V, A, B)
    return y


def _lerp6_rkv(x, prev, x_r, x_w, x_k, x_v, x_a, x_g, x_copy, rWt_stack):
    r, k, v, xv, xw, xa, xg = K.fused_lerp6_rkv_copy(x, prev, x_r, x_w, x_k, x_v, x_a, x_g, x_copy, rWt_stack)
    # r, k and v are views of one stacked result: outputs must not share storage
    return r.clone(), k.clone(), v.clone(), xv, xw, xa, xg


def _lerp6_copy(*args):
    return tuple(t.clone() for t in K.fused_lerp6_copy(*args))


OPS: dict[str, tuple[str, Callable, Callable]] = {
    "fused_lerp6_copy": (
        "(Tensor x, Tensor prev, Tensor x_r, Tensor x_w, Tensor x_k, Tensor x_v, Tensor x_a, Tensor x_g,"
        " Tensor(a!) x_copy) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        _lerp6_copy,
        _like(6),
    ),
    "fused_lerp1_copy": (
        "(Tensor x, Tensor prev, Tensor w, Tensor(a!) x_copy) -> Tensor",
        K.fused_lerp1_copy,
        lambda x, *_: torch.empty_like(x),
    ),
    "fused_w_gate": ("(Tensor x, Tensor w0) -> Tensor", K.fused_w_gate, lambda x, *_: torch.empty_like(x)),
    "fused_v_gate": (
        "(Tensor v, Tensor v_first, Tensor v0, Tensor v12) -> Tensor",
        K.fused_v_gate,
        lambda v, *_: torch.empty_like(v),
    ),
    "fused_a_kk_k": (
        "(Tensor a0, Tensor a_x, Tensor k, Tensor k_k, Tensor k_a) -> (Tensor, Tensor, Tensor)",
        K.fused_a_kk_k,
        _like(3),
    ),
    "fused_gates": (
        "(Tensor vr, Tensor wr, Tensor ar, Tensor gr, Tensor v, Tensor v_first, Tensor k, Tensor v2t,"
        " Tensor w2t, Tensor a2t, Tensor g2t, Tensor v0, Tensor w0, Tensor a0, Tensor k_k, Tensor k_a)"
        " -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        K.fused_gates,
        lambda vr, wr, ar, gr, v, *_: tuple(torch.empty_like(v) for _ in range(6)),
    ),
    "fused_rank_gemv": (
        "(Tensor xv, Tensor xw, Tensor xa, Tensor xg, Tensor packed, int rv, int rw, int ra, int rg) -> Tensor",
        K.fused_rank_gemv,
        lambda xv, xw, xa, xg, packed, *_: torch.empty(packed.shape[0], dtype=xv.dtype, device=xv.device),
    ),
    "fused_l2norm_neg_kk_a": ("(Tensor kk, Tensor a) -> (Tensor, Tensor)", K.fused_l2norm_neg_kk_a, _like(2)),
    "fused_gn_rkrk": (
        "(Tensor y, Tensor r, Tensor k, Tensor v, Tensor r_k, Tensor ln_xW, Tensor ln_xB) -> Tensor",
        K.fused_gn_rkrk,
        lambda y, *_: torch.empty(y.numel(), dtype=y.dtype, device=y.device),
    ),
    "fused_dplr": (
        "(Tensor(a!) S, Tensor R, Tensor W, Tensor K, Tensor V, Tensor A, Tensor B) -> Tensor",
        _dplr,
        lambda S, R, *_: torch.empty_like(R),
    ),
    "fused_lerp6_rkv_copy": (
        "(Tensor x, Tensor prev, Tensor x_r, Tensor x_w, Tensor x_k, Tensor x_v, Tensor x_a, Tensor x_g,"
        " Tensor(a!) x_copy, Tensor rWt_stack) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        _lerp6_rkv,
        _like(7),
    ),
    "fused_rkv_gemm": (
        "(Tensor xr, Tensor xk, Tensor xv, Tensor Wb) -> Tensor",
        K.fused_rkv_gemm,
        lambda xr, *_: torch.empty(3, xr.shape[0], xr.shape[1], dtype=xr.dtype, device=xr.device),
    ),
}

# The training operator (no counterpart in the reference's registry yet; its
# TODO.md:46-54 plans exactly this: a DPLR custom op with register_autograd).
# Functional, f32: S [H,64,64] or [B,H,64,64] is not modified; returns (y, S_T).
TRAIN_OPS: dict[str, tuple[str, Callable, Callable]] = {
    "fused_dplr_seq": (
        "(Tensor S, Tensor R, Tensor W, Tensor K, Tensor V, Tensor A, Tensor B) -> (Tensor, Tensor)",
        K.dplr_seq_forward,
        lambda S, R, *_: (torch.empty_like(R), torch.empty_like(S)),
    ),
}


# Operators between a large model and a small one (no counterpart in the
# reference): a teacher's top logits, the divergence of a student from them.
# ``distill_loss`` is differentiable to ``logits`` (not to the teacher, and once).
def _top_meta(logits, k, temperature=1.0):
    lead = logits.shape[:-1]
    return (logits.new_empty(*lead, k), logits.new_empty(*lead, k, dtype=torch.int64),
            logits.new_empty(lead, dtype=torch.float32))


LOGITS_OPS: dict[str, tuple[str, Callable, Callable]] = {
    "top_logits": (
        "(Tensor logits, int k, float temperature=1.0) -> (Tensor, Tensor, Tensor)",
        lambda logits, k, temperature=1.0: K.top_logits(logits, k, temperature=temperature),
        _top_meta,
    ),
    "distill_loss": (
        "(Tensor logits, Tensor top_val, Tensor top_idx, Tensor? lse=None, float temperature=1.0) -> Tensor",
        lambda logits, top_val, top_idx, lse=None, temperature=1.0: K.distill_loss(
            logits, top_val, top_idx, lse, temperature=temperature),
        lambda logits, *_: logits.new_empty(logits.shape[:-1], dtype=torch.float32),
    ),
    "distill_loss_backward": (
        "(Tensor grad_loss, Tensor logits, Tensor top_val, Tensor top_idx, Tensor? lse, float temperature) -> Tensor",
        K.distill_loss_backward,
        lambda grad_loss, logits, *_: torch.empty(logits.shape, dtype=logits.dtype, device=logits.device),
    ),
}


# The two ends and the norms of a training step (no counterpart in the reference).
# ``embed`` is differentiable to its table, ``layer_norm`` to its three tensors,
# ``token_logprobs`` to the logits; each once.
def _norm_meta(x, *_):
    stat = x.new_empty(x.shape[:-1], dtype=torch.float32)
    return x.new_empty(x.shape), stat, torch.empty_like(stat)


def _rows_meta(logits, *_):
    row = logits.new_empty(logits.shape[:-1], dtype=torch.float32)
    return row, torch.empty_like(row)


STEP_OPS: dict[str, tuple[str, Callable, Callable]] = {
    "embed": (
        "(Tensor weight, Tensor tokens, float scale=1.0) -> Tensor",
        lambda weight, tokens, scale=1.0: K.embed(weight, tokens, scale=scale),
        lambda weight, tokens, *_: weight.new_empty(*tokens.shape, weight.shape[1]),
    ),
    "embed_backward": (
        "(Tensor grad, Tensor tokens, int vocab, float scale=1.0) -> Tensor",
        lambda grad, tokens, vocab, scale=1.0: K.embed_backward(grad, tokens, vocab, scale=scale),
        lambda grad, tokens, vocab, *_: grad.new_empty(vocab, grad.shape[-1]),
    ),
    "layer_norm": (
        "(Tensor x, Tensor weight, Tensor bias, float eps=1e-05) -> Tensor",
        lambda x, weight, bias, eps=1e-5: T.norm(x, weight, bias, eps),
        lambda x, *_: x.new_empty(x.shape),
    ),
    "layer_norm_forward": (
        "(Tensor x, Tensor weight, Tensor bias, float eps=1e-05) -> (Tensor, Tensor, Tensor)",
        lambda x, weight, bias, eps=1e-5: K.layer_norm_forward(x, weight, bias, eps=eps),
        _norm_meta,
    ),
    "layer_norm_backward": (
        "(Tensor grad_y, Tensor x, Tensor weight, Tensor mean, Tensor rstd) -> (Tensor, Tensor, Tensor)",
        K.layer_norm_backward,
        lambda grad_y, x, weight, *_: (x.new_empty(x.shape), weight.new_empty(weight.shape), weight.new_empty(weight.shape)),
    ),
    "token_logprobs": (
        "(Tensor logits, Tensor tokens, float temperature=1.0) -> (Tensor, Tensor)",
        lambda logits, tokens, temperature=1.0: K.token_logprobs(logits, tokens, temperature=temperature),
        _rows_meta,
    ),
    "token_logprobs_backward": (
        "(Tensor? grad_logprob, Tensor? grad_entropy, Tensor logits, Tensor tokens, float temperature) -> Tensor",
        K.token_logprobs_backward,
        lambda grad_logprob, grad_entropy, logits, *_: logits.new_empty(logits.shape),
    ),
}


def _plain(x: Tensor) -> bool:
    """Whether a call on ``x`` may go straight to the kernel: no tracing, no
    dispatch mode that wants to see the operator, no batch of tensors in one (that of
    ``torch.autograd.grad(..., is_grads_batched=True)``, which has no storage)."""
    return type(x) in (Tensor, torch.nn.Parameter) and x.is_cuda and not torch._C._len_torch_dispatch_stack() and torch._C._has_storage(x)


class _DistillLoss(torch.autograd.Function):
    """The Autograd kernel of ``distill_loss``. (torch.library.register_autograd
    makes one like it that takes 28 us more of a call's host time.)"""

    @staticmethod
    def forward(ctx, logits, top_val, top_idx, lse, temperature):
        ctx.save_for_backward(logits, top_val, top_idx, lse)
        ctx.temperature = temperature
        if _plain(logits):
            return K.distill_loss(logits, top_val, top_idx, lse, temperature=temperature)
        with torch._C._AutoDispatchBelowAutograd():
            return torch.ops.rwkv_tl.distill_loss(logits, top_val, top_idx, lse, temperature)

    @staticmethod
    def backward(ctx, grad_loss):
        args = (grad_loss, *ctx.saved_tensors, ctx.temperature)
        # (a gradient that is to be differentiated goes through the operator, which refuses)
        plain = _plain(grad_loss) and not torch.is_grad_enabled()
        return (K.distill_loss_backward if plain else torch.ops.rwkv_tl.distill_loss_backward)(*args), None, None, None, None


class _DistillLossBackward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        with torch._C._AutoDispatchBelowAutograd():
            return torch.ops.rwkv_tl.distill_loss_backward(*args)

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("distill_loss has no second derivative")


def _distill_autograd(logits, top_val, top_idx, lse=None, temperature=1.0):
    # (here: in forward the grad mode is off, and the flags say the same without it)
    if (top_val.requires_grad or (lse is not None and lse.requires_grad)) and torch.is_grad_enabled():
        raise ValueError("distill_loss has no gradient to the teacher: detach top_val and lse")
    return _DistillLoss.apply(logits, top_val, top_idx, lse, temperature)


def _below(op: Callable, *args):
    """The operator below autograd (for tracing and batched tensors)."""
    with torch._C._AutoDispatchBelowAutograd():
        return op(*args)


def _direct(grad: Tensor) -> bool:
    """Whether a gradient goes straight to its kernel (one that is to be differentiated goes
    through the operator, which refuses)."""
    return _plain(grad) and not torch.is_grad_enabled()


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale):
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale = weight.shape[0], scale
        return K.embed(weight, tokens, scale=scale) if _plain(weight) else _below(torch.ops.rwkv_tl.embed, weight, tokens, scale)

    @staticmethod
    def backward(ctx, grad):
        f = T.embed_backward_checked if _direct(grad) else torch.ops.rwkv_tl.embed_backward
        return f(grad, *ctx.saved_tensors, ctx.vocab, ctx.scale), None, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        if _plain(x):
            y, mean, rstd = K.layer_norm_forward(x, weight, bias, eps=eps)
        else:
            y, mean, rstd = _below(torch.ops.rwkv_tl.layer_norm_forward, x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, grad):
        f = T.layer_norm_backward_checked if _direct(grad) else torch.ops.rwkv_tl.layer_norm_backward
        return *f(grad, *ctx.saved_tensors), None


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        ctx.save_for_backward(logits, tokens)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if _plain(logits):
            return K.token_logprobs(logits, tokens, temperature=temperature)
        return _below(torch.ops.rwkv_tl.token_logprobs, logits, tokens, temperature)

    @staticmethod
    def backward(ctx, grad_logprob, grad_entropy):
        some = [g for g in (grad_logprob, grad_entropy) if g is not None]
        if not some:
            return None, None, None
        # (one of the two may be a batch, the other not)
        f = K.token_logprobs_backward if all(map(_direct, some)) else torch.ops.rwkv_tl.token_logprobs_backward
        return f(grad_logprob, grad_entropy, *ctx.saved_tensors, ctx.temperature), None, None


def _no_gradient(name: str, why: str):
    """The Autograd kernel of an operator without a gradient: a backward pass that reaches it raises
    (torch's own, for want of one, warns and leaves the gradients out)."""

    class Gradient(torch.autograd.Function):
        @staticmethod
        def forward(ctx, *args):
            with torch._C._AutoDispatchBelowAutograd():
                return getattr(torch.ops.rwkv_tl, name)(*args)

        @staticmethod
        def backward(ctx, *_):
            raise NotImplementedError(why)

    return Gradient.apply


def _dplr_seq_setup(ctx, inputs, output) -> None:
    ctx.save_for_backward(*inputs)


def _dplr_seq_backward(ctx, gy, gS):
    S, R, W, K_, V, A, B = ctx.saved_tensors
    if gy is None:
        gy = torch.zeros_like(R)
    return K.dplr_seq_backward(S, R, W, K_, V, A, B, gy.contiguous(), None if gS is None else gS.contiguous())


_registered = False


def register() -> None:
    """Define every operator with its CUDA and Meta implementations (idempotent)."""
    global _registered
    if _registered:
        return
    for name, (schema, cuda, meta) in {**OPS, **TRAIN_OPS, **LOGITS_OPS, **STEP_OPS}.items():
        qual = f"{NAMESPACE}::{name}"
        torch.library.define(qual, schema)
        torch.library.impl(qual, "CUDA")(cuda)
        torch.library.impl(qual, "Meta")(meta)
    torch.library.register_autograd(
        f"{NAMESPACE}::fused_dplr_seq", _dplr_seq_backward, setup_context=_dplr_seq_setup
    )
    torch.library.impl(f"{NAMESPACE}::distill_loss", "Autograd")(_distill_autograd)
    torch.library.impl(f"{NAMESPACE}::distill_loss_backward", "Autograd")(_DistillLossBackward.apply)
    for name, autograd in (
        ("embed", lambda weight, tokens, scale=1.0: _Embed.apply(weight, tokens, scale)),
        ("layer_norm", lambda x, weight, bias, eps=1e-5: _LayerNorm.apply(x, weight, bias, eps)),
        ("token_logprobs", lambda logits, tokens, temperature=1.0: _TokenLogprobs.apply(logits, tokens, temperature)),
    ):
        torch.library.impl(f"{NAMESPACE}::{name}", "Autograd")(autograd)
        torch.library.impl(f"{NAMESPACE}::{name}_backward", "Autograd")(
            _no_gradient(f"{name}_backward", f"{name} has no second derivative")
        )
    torch.library.impl(f"{NAMESPACE}::layer_norm_forward", "Autograd")(
        _no_gradient("layer_norm_forward", "layer_norm_forward has no gradient: layer_norm is the differentiable form")
    )
    _registered = True


register()
