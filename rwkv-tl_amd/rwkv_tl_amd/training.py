"""The input end and the norms of a training step, around the DPLR sequence (no
counterpart in the reference, whose training is a plan, ``TODO.md:46-54``).

* ``embed`` / ``embed_backward``: rows of an embedding table times a factor, and the
  table's gradient.
* ``layer_norm_forward`` / ``layer_norm_backward``: LayerNorm (``weight.py:14-15``) in
  its input's type that keeps its statistics, and its gradients. (``kernels.layer_norm``
  is inference's: float32 out, eps 1e-5, no gradient.)

``torch.ops.rwkv_tl.embed`` and ``torch.ops.rwkv_tl.layer_norm`` are the differentiable
forms. (The output end is ``token_logprobs`` in ``logits.py``.) Tensors are float16,
bfloat16 or float32 on the GPU; rows may lie at any stride. Nothing waits for the
host, so the calls can be captured in a HIP graph. Each call allocates what it returns
and its workspace. The gradients' sums have an order that the inputs alone decide.
"""

from __future__ import annotations

from functools import lru_cache

import torch
from torch import Tensor

from . import _lib
from .logits import LOGIT_DTYPES as DTYPES
from .logits import _empty, _rows, _same_device

MAX_TOKENS = 2**24 - 1  # positions of one call of embed
MAX_VOCAB = 1 << 20  # rows of an embedding table
MAX_WIDTH = 65536  # its columns
MAX_CHANNELS = 16384  # of layer_norm


def _check(x: Tensor, name: str) -> int:
    """The tensor's dtype code."""
    if not isinstance(x, Tensor):
        raise ValueError(f"{name} must be a tensor")
    if not x.is_cuda:
        raise ValueError(f"{name} on {x.device}; the HIP kernels need a ROCm device")
    code = DTYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"{name} must be float16, bfloat16 or float32, got {x.dtype}")
    return code


def _check_tokens(tokens: Tensor) -> int:
    """How many."""
    if not isinstance(tokens, Tensor) or tokens.dtype is not torch.int64:
        raise ValueError(f"tokens must be an int64 tensor, got {getattr(tokens, 'dtype', type(tokens).__name__)}")
    N = tokens.numel()
    if N > MAX_TOKENS:
        raise ValueError(f"{N} tokens are too many for one call: at most {MAX_TOKENS}")
    return N


def _check_table(V: int, C: int) -> None:
    if not 1 <= V <= MAX_VOCAB or not 1 <= C <= MAX_WIDTH:
        raise ValueError(f"a table of 1..{MAX_VOCAB} rows of 1..{MAX_WIDTH} columns, got {V} x {C}")


def _factor(scale: float) -> float:
    scale = float(scale)
    if not abs(scale) <= 3.4028234663852886e38:  # (NaN neither)
        raise ValueError(f"scale must be a float32 number, got {scale}")
    return scale


def embed(weight: Tensor, tokens: Tensor, *, scale: float = 1.0) -> Tensor:
    """``scale * weight[tokens]``: ``[..., C]`` of the type of ``weight [V, C]`` for
    ``tokens [...]`` int64, V <= 2^20. An id outside ``0..V-1`` (say -1, a padded
    position) gives a row of zeros, and has no part in the gradient.

    Without autograd; ``torch.ops.rwkv_tl.embed`` is the differentiable form."""
    code = _check(weight, "weight")
    if weight.ndim != 2:
        raise ValueError(f"weight must be [V, C], got {tuple(weight.shape)}")
    V, C = weight.shape
    _check_table(V, C)
    N = _check_tokens(tokens)
    scale = _factor(scale)
    _same_device(weight, tokens)
    with _lib.device_of(weight):
        out = torch.empty(*tokens.shape, C, dtype=weight.dtype, device=weight.device)
        if N:
            w, _, ld = _rows(weight)
            t = tokens.contiguous()
            rc = _lib.load().rwkv7_embed(w.data_ptr(), code, ld, t.data_ptr(), scale, out.data_ptr(), N, V, C, _lib.stream_of(w))
            _lib.check(rc, "rwkv7_embed")
    return out


@lru_cache(maxsize=64)
def _embed_bytes(code: int, N: int, V: int, C: int) -> int:
    return _lib.load().rwkv7_embed_backward_workspace_bytes(code, N, V, C)


def embed_backward(grad: Tensor, tokens: Tensor, vocab: int, *, scale: float = 1.0) -> Tensor:
    """Gradient of ``embed`` to its table: ``[vocab, C]`` of the type of ``grad [..., C]``,
    ``scale`` times the sum of each token's rows (in 32 bits, rounded once), zeros
    where there is none."""
    _check(grad, "grad")
    _check_tokens(tokens)
    if grad.ndim != tokens.ndim + 1 or grad.shape[:-1] != tokens.shape:
        raise ValueError(f"grad must be [{', '.join(map(str, (*tokens.shape, 'C')))}], got {tuple(grad.shape)}")
    C = grad.shape[-1]
    if not isinstance(vocab, int):
        raise ValueError(f"vocab must be an int, got {vocab!r}")
    _check_table(vocab, C)
    scale = _factor(scale)
    _same_device(grad, tokens)
    return embed_backward_checked(grad, tokens, vocab, scale)


def embed_backward_checked(grad: Tensor, tokens: Tensor, vocab: int, scale: float) -> Tensor:
    """``embed_backward`` of what autograd hands on: shapes, types and device are the forward pass's."""
    code, N, C = DTYPES[grad.dtype], tokens.numel(), grad.shape[-1]
    with _lib.device_of(grad):
        out = torch.empty(vocab, C, dtype=grad.dtype, device=grad.device)
        if N:
            g, _, ld = _rows(grad)
            t = tokens.contiguous()
            nb = _embed_bytes(code, N, vocab, C)
            ws = torch.empty(nb, dtype=torch.uint8, device=grad.device)
            rc = _lib.load().rwkv7_embed_backward(
                g.data_ptr(), code, ld, t.data_ptr(), scale, out.data_ptr(), N, vocab, C, ws.data_ptr(), nb, _lib.stream_of(g)
            )
            _lib.check(rc, "rwkv7_embed_backward")
        else:
            out.zero_()
    return out


def _check_norm(x: Tensor, weight: Tensor, bias: Tensor | None) -> tuple[int, int]:
    """The dtype codes of x and of the weight."""
    code, wcode = _check(x, "x"), _check(weight, "weight")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"x: 1..{MAX_CHANNELS} channels, got {tuple(x.shape)}")
    if wcode != 1 and wcode != code:
        raise ValueError(f"weight must be float32 or {x.dtype}, got {weight.dtype}")
    C = x.shape[-1]
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.shape != (C,) or t.dtype is not weight.dtype):
            raise ValueError(f"{name} must be {weight.dtype} [{C}], got {t.dtype} {tuple(t.shape)}")
    return code, wcode


def layer_norm_forward(x: Tensor, weight: Tensor, bias: Tensor, *, eps: float = 1e-5) -> tuple[Tensor, Tensor, Tensor]:
    """LayerNorm over the last dimension of ``x [..., C]``, C <= 16384: ``(y [..., C] of x's
    type, mean [...], rstd [...])`` float32. ``weight [C]`` and ``bias [C]`` are both
    float32 or both of x's type.

    Without autograd; ``torch.ops.rwkv_tl.layer_norm`` is the differentiable form."""
    return _norm(x, weight, bias, eps, True)


def norm(x: Tensor, weight: Tensor, bias: Tensor, eps: float) -> Tensor:
    """``layer_norm_forward`` without the statistics."""
    return _norm(x, weight, bias, eps, False)[0]


def _norm(x: Tensor, weight: Tensor, bias: Tensor, eps: float, keep: bool):
    code, wcode = _check_norm(x, weight, bias)
    eps = float(eps)
    if not 1e-30 <= eps <= 1e30:
        raise ValueError(f"eps must be within 1e-30..1e30, got {eps}")
    _same_device(x, weight, bias)
    lead, C = x.shape[:-1], x.shape[-1]
    with _lib.device_of(x):
        dev = x.device
        y = torch.empty(*lead, C, dtype=x.dtype, device=dev)
        mean, rstd = (_empty(lead, torch.float32, dev), _empty(lead, torch.float32, dev)) if keep else (None, None)
        r, N, ld = _rows(x)
        if N:
            w, b = weight.contiguous(), bias.contiguous()
            rc = _lib.load().rwkv7_layer_norm_forward(
                r.data_ptr(), code, ld, w.data_ptr(), b.data_ptr(), wcode, eps, y.data_ptr(), _lib.ptr(mean), _lib.ptr(rstd),
                N, C, _lib.stream_of(r),
            )
            _lib.check(rc, "rwkv7_layer_norm_forward")
    return y, mean, rstd


@lru_cache(maxsize=64)
def _norm_bytes(code: int, N: int, C: int) -> int:
    return _lib.load().rwkv7_layer_norm_backward_workspace_bytes(code, N, C)


def layer_norm_backward(grad_y: Tensor, x: Tensor, weight: Tensor, mean: Tensor, rstd: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """Gradients of ``layer_norm_forward`` to ``(x, weight, bias)`` under ``grad_y [..., C]`` of
    x's type, from the input and the statistics that the forward pass returned."""
    _check_norm(x, weight, None)
    lead = x.shape[:-1]
    if grad_y.shape != x.shape or grad_y.dtype is not x.dtype:
        raise ValueError(f"grad_y must be {x.dtype} {tuple(x.shape)}, got {grad_y.dtype} {tuple(grad_y.shape)}")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.shape != lead or t.dtype is not torch.float32:
            raise ValueError(f"{name} must be float32 {tuple(lead)}, got {t.dtype} {tuple(t.shape)}")
    _same_device(x, grad_y, weight, mean, rstd)
    return layer_norm_backward_checked(grad_y, x, weight, mean, rstd)


def layer_norm_backward_checked(grad_y: Tensor, x: Tensor, weight: Tensor, mean: Tensor, rstd: Tensor):
    """``layer_norm_backward`` of what autograd hands on: shapes, types and device are the forward pass's."""
    code, wcode = DTYPES[x.dtype], DTYPES[weight.dtype]
    lead, C = x.shape[:-1], x.shape[-1]
    with _lib.device_of(x):
        dev = x.device
        gx = torch.empty(*lead, C, dtype=x.dtype, device=dev)
        gw = torch.empty(C, dtype=weight.dtype, device=dev)
        gb = torch.empty(C, dtype=weight.dtype, device=dev)
        r, N, ld = _rows(x)
        if N:
            g, _, ldg = _rows(grad_y)
            w, m, s = weight.contiguous(), mean.contiguous(), rstd.contiguous()
            nb = _norm_bytes(code, N, C)
            ws = torch.empty(nb, dtype=torch.uint8, device=dev)
            rc = _lib.load().rwkv7_layer_norm_backward(
                g.data_ptr(), ldg, r.data_ptr(), ld, code, w.data_ptr(), wcode, m.data_ptr(), s.data_ptr(), gx.data_ptr(),
                gw.data_ptr(), gb.data_ptr(), N, C, ws.data_ptr(), nb, _lib.stream_of(r),
            )
            _lib.check(rc, "rwkv7_layer_norm_backward")
        else:
            gw.zero_()
            gb.zero_()
    return gx, gw, gb
