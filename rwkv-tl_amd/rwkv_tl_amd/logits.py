"""Operators on rows of logits: between a large model and a small one of the same
vocabulary, and the output end of a training step (no counterpart in the reference).

* ``top_logits``: what a teacher hands on of each row: its largest logits, their
  token ids, and the row's log-sum-exp.
* ``distill_loss`` / ``distill_loss_grad``: the divergence of a student's
  distribution from a teacher's top logits, alone or with its gradient in the
  same pass. ``torch.ops.rwkv_tl.distill_loss`` is the differentiable form.
* ``token_logprobs`` / ``token_logprobs_grad``: the log probability of a given token of
  each row, the row's entropy, its most likely alternatives, or the gradient in the same
  pass. ``torch.ops.rwkv_tl.token_logprobs`` is the differentiable form.
* ``verify_draft``: drafted tokens against the target model's probabilities,
  from given random numbers (speculative sampling).

Logits are float16, bfloat16 or float32 on the GPU, of up to ``MAX_VOCAB``
tokens; rows may lie at any stride. Nothing waits for the host, so the calls can
be captured in a HIP graph. Each call allocates what it returns, and
``verify_draft`` its workspace.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch
from torch import Tensor

from . import _lib

MAX_VOCAB = 65536
MAX_TOP = 256  # largest k of top_logits
MAX_ENTRIES = 1024  # teacher entries per row of distill_loss
MAX_DRAFT = 63  # drafted tokens per sequence of verify_draft

LOGIT_DTYPES = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 2}


def _check_logits(x: Tensor, name: str) -> int:
    """The logits' dtype code."""
    if not isinstance(x, Tensor):
        raise ValueError(f"{name} must be a tensor")
    if not x.is_cuda:
        raise ValueError(f"{name} on {x.device}; the HIP kernels need a ROCm device")
    code = LOGIT_DTYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"{name} must be float16, bfloat16 or float32, got {x.dtype}")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"{name}: a vocabulary of 1..{MAX_VOCAB}, got {tuple(x.shape)}")
    return code


def _rows(x: Tensor) -> tuple[Tensor, int, int]:
    """``[..., V]`` as rows of adjacent columns that do not overlap: what holds them
    (a copy only where no view is one), their number and their stride."""
    V = x.shape[-1]
    N = x.numel() // V
    if N > 2**31 - 1:
        raise ValueError(f"{N} rows are too many for one call")
    if x.is_contiguous():
        return x, N, V
    x = x.reshape(N, V)
    if (x.stride(1) != 1 and V > 1) or (N > 1 and x.stride(0) < V):
        x = x.contiguous()
    return x, N, x.stride(0) if N > 1 else V


def _empty(shape, dtype: torch.dtype, device: torch.device) -> Tensor:
    # (sizes one by one: torch.empty takes 1 us more for a torch.Size)
    return torch.empty(*shape, dtype=dtype, device=device) if shape else torch.empty((), dtype=dtype, device=device)


def _temperature(t: float) -> float:
    t = float(t)
    if not 1e-30 <= t <= 1e30:  # (NaN neither)
        raise ValueError(f"temperature must be positive and finite, got {t}")
    return t


def _same_device(ref: Tensor, *others: Tensor | None) -> None:
    i = ref.get_device()
    for t in others:
        if t is not None and t.get_device() != i:
            raise ValueError(f"tensors on {ref.device} and on {t.device}")


def top_logits(logits: Tensor, k: int, *, temperature: float = 1.0) -> tuple[Tensor, Tensor, Tensor]:
    """The ``k`` largest of each row of ``logits`` ``[..., V]``, 1 <= k <= min(V, 256).

    Returns ``values [..., k]`` (the logits' dtype, descending; ties by the lowest
    id, NaN last), ``indices [..., k]`` int64, and ``lse [...]`` float32, the log
    of the sum of ``exp(logits / temperature)`` over the whole row: a teacher's
    answers as ``distill_loss`` takes them."""
    code = _check_logits(logits, "logits")
    V = logits.shape[-1]
    if not isinstance(k, int) or not 1 <= k <= min(V, MAX_TOP):
        raise ValueError(f"k must be in 1..{min(V, MAX_TOP)}, got {k}")
    temperature = _temperature(temperature)
    lead = logits.shape[:-1]
    with _lib.device_of(logits):
        x, N, ld = _rows(logits)
        dev = x.device
        val = torch.empty(*lead, k, dtype=x.dtype, device=dev)
        idx = torch.empty(*lead, k, dtype=torch.int64, device=dev)
        lse = _empty(lead, torch.float32, dev)
        if N:
            rc = _lib.load().rwkv7_top_logits(
                x.data_ptr(), code, ld, N, V, k, temperature, val.data_ptr(), idx.data_ptr(), lse.data_ptr(), _lib.stream_of(x)
            )
            _lib.check(rc, "rwkv7_top_logits")
    return val, idx, lse


def _distill(logits, top_val, top_idx, lse, temperature, scale, want_loss: bool, want_grad: bool):
    code = _check_logits(logits, "logits")
    shape = logits.shape
    lead, V = shape[:-1], shape[-1]
    ts = top_val.shape
    if ts[:-1] != lead or top_idx.shape != ts or len(ts) != len(shape):
        raise ValueError(f"top_val and top_idx must be [{', '.join(map(str, (*lead, 'K')))}], got {tuple(ts)} and {tuple(top_idx.shape)}")
    K = ts[-1]
    if K > MAX_ENTRIES:
        raise ValueError(f"at most {MAX_ENTRIES} teacher entries per row, got {K}")
    tcode = LOGIT_DTYPES.get(top_val.dtype)
    if tcode is None:
        raise ValueError(f"top_val must be float16, bfloat16 or float32, got {top_val.dtype}")
    if top_idx.dtype is not torch.int64:
        raise ValueError(f"top_idx must be int64, got {top_idx.dtype}")
    if lse is not None and (lse.shape != lead or lse.dtype is not torch.float32):
        raise ValueError(f"lse must be float32 {tuple(lead)}")
    rows = scale if isinstance(scale, Tensor) else None
    if rows is not None and (rows.shape != lead or rows.dtype is not torch.float32):
        raise ValueError(f"scale must be float32 {tuple(lead)}")
    _same_device(logits, top_val, top_idx, lse, rows)
    temperature = _temperature(temperature)
    with _lib.device_of(logits):
        loss = _empty(lead, torch.float32, logits.device) if want_loss else None
        grad = torch.empty(*shape, dtype=logits.dtype, device=logits.device) if want_grad else None
        x, N, ld = _rows(logits)
        if N and K:
            tv, ti = top_val.contiguous(), top_idx.contiguous()
            ls = None if lse is None else lse.contiguous()
            sc = None if rows is None else rows.contiguous()
            rc = _lib.load().rwkv7_distill(
                x.data_ptr(), code, ld, N, V, tv.data_ptr(), tcode, ti.data_ptr(), K, _lib.ptr(ls), temperature,
                _lib.ptr(sc), 1.0 if rows is not None else float(scale), _lib.ptr(loss), _lib.ptr(grad), V, _lib.stream_of(x),
            )
            _lib.check(rc, "rwkv7_distill")
        else:
            for t in (loss, grad):
                if t is not None:
                    t.zero_()  # rows without any teacher
    return loss, grad


def distill_loss(logits: Tensor, top_val: Tensor, top_idx: Tensor, lse: Tensor | None = None, *,
                 temperature: float = 1.0) -> Tensor:
    """Divergence of the student's ``softmax(logits / temperature)`` from a
    teacher's top logits: float32 ``[...]``, a loss per row of ``logits [..., V]``.

    ``top_val [..., K]`` (any of the three dtypes) and ``top_idx [..., K]`` int64
    are the teacher's entries, K <= 1024; an id outside ``0..V-1`` (say -1) means
    no entry, so rows may have fewer, and a row without any, or with values of -inf
    alone, or with an ``lse`` of -2^24 or less (as ``top_logits`` gives of a row that is
    all masked, by -inf or by the lowest value of bfloat16 or float32), has loss 0 and gradient 0 whatever its logits hold (a padded position). With ``lse [...]``
    float32, the teacher's log-sum-exp over its whole vocabulary at the same
    temperature, ``p_k = exp(top_val_k / temperature - lse)`` and the mass that
    this leaves (2^-20 or more, or half a step of ``lse`` where that is more: beyond
    +-32; of a row that does not list every id) is held against the student's mass
    outside the row's ids; without it, ``p`` is the softmax of the
    entries. There is no factor ``temperature ** 2``.

    Without autograd; ``torch.ops.rwkv_tl.distill_loss`` is the differentiable form."""
    return _distill(logits, top_val, top_idx, lse, temperature, 1.0, True, False)[0]


def distill_loss_grad(logits: Tensor, top_val: Tensor, top_idx: Tensor, lse: Tensor | None = None, *,
                      temperature: float = 1.0, scale: Tensor | float = 1.0) -> tuple[Tensor, Tensor]:
    """``distill_loss`` and ``scale`` times its gradient to ``logits`` in one pass
    over them: ``(loss [...] float32, grad [..., V] of the logits' dtype)``.
    ``scale``: a number, or float32 ``[...]`` (each row's weight in the loss and a
    loss scale; a row with 0 has gradient 0); ``scale / temperature`` within float32.
    For ``logits.backward(grad)``."""
    return _distill(logits, top_val, top_idx, lse, temperature, scale, True, True)


def distill_loss_backward(grad_loss: Tensor, logits: Tensor, top_val: Tensor, top_idx: Tensor, lse: Tensor | None,
                          temperature: float) -> Tensor:
    """Gradient of ``distill_loss`` to ``logits`` under ``grad_loss`` float32 ``[...]``."""
    return _distill(logits, top_val, top_idx, lse, temperature, grad_loss, False, True)[1]


def _check_rows(logits: Tensor, tokens: Tensor, temperature: float) -> tuple[int, float]:
    """The logits' dtype code and the temperature."""
    code = _check_logits(logits, "logits")
    if not isinstance(tokens, Tensor) or tokens.dtype is not torch.int64 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must be int64 {tuple(logits.shape[:-1])}")
    _same_device(logits, tokens)
    return code, _temperature(temperature)


def token_logprobs(logits: Tensor, tokens: Tensor, k: int = 0, *, temperature: float = 1.0) -> tuple[Tensor, ...]:
    """Log probabilities of given tokens, with entropy and alternatives: of each row of
    ``logits [..., V]``, with ``q = softmax(logits / temperature)``, ``log q`` of the row's
    token (``tokens [...]`` int64) and the entropy ``-sum q log q``.

    Returns ``(logprob [...], entropy [...])`` float32, and for ``k`` from 1 to
    min(V, 256) also ``(top_logprob [..., k]`` float32, ``top_index [..., k]`` int64``)``:
    the k most likely tokens in descending order, ties by the lowest id.

    An id outside ``0..V-1`` (say -1) makes its row a padded one: logprob and entropy 0,
    alternatives -inf and -1, whatever its logits hold. A row of -inf alone has logprobs
    -inf and entropy 0; a NaN or +inf makes its row NaN. Without autograd;
    ``torch.ops.rwkv_tl.token_logprobs`` is the differentiable form."""
    code, temperature = _check_rows(logits, tokens, temperature)
    V = logits.shape[-1]
    if not isinstance(k, int) or not 0 <= k <= min(V, MAX_TOP):
        raise ValueError(f"k must be in 0..{min(V, MAX_TOP)}, got {k}")
    lead = logits.shape[:-1]
    with _lib.device_of(logits):
        x, N, ld = _rows(logits)
        dev = x.device
        logp, entropy = _empty(lead, torch.float32, dev), _empty(lead, torch.float32, dev)
        top = idx = None
        if k:
            top = torch.empty(*lead, k, dtype=torch.float32, device=dev)
            idx = torch.empty(*lead, k, dtype=torch.int64, device=dev)
        if N:
            t = tokens.contiguous()
            rc = _lib.load().rwkv7_token_logprobs(
                x.data_ptr(), code, ld, N, V, t.data_ptr(), temperature, k, logp.data_ptr(), entropy.data_ptr(), _lib.ptr(top),
                _lib.ptr(idx), _lib.stream_of(x),
            )
            _lib.check(rc, "rwkv7_token_logprobs")
    return (logp, entropy, top, idx) if k else (logp, entropy)


def _token_grad(logits, tokens, temperature, scale, entropy_scale, want: bool):
    code, temperature = _check_rows(logits, tokens, temperature)
    shape = logits.shape
    lead, V = shape[:-1], shape[-1]
    rows = [s if isinstance(s, Tensor) else None for s in (scale, entropy_scale)]
    for s, name in zip(rows, ("scale", "entropy_scale")):
        if s is not None and (s.shape != lead or s.dtype is not torch.float32):
            raise ValueError(f"{name} must be float32 {tuple(lead)}")
    _same_device(logits, *rows)
    one = [1.0 if r is not None else float(s) for r, s in zip(rows, (scale, entropy_scale))]
    with _lib.device_of(logits):
        dev = logits.device
        logp, entropy = (_empty(lead, torch.float32, dev), _empty(lead, torch.float32, dev)) if want else (None, None)
        grad = torch.empty(*shape, dtype=logits.dtype, device=dev)
        x, N, ld = _rows(logits)
        if N:
            t = tokens.contiguous()
            s, h = (None if r is None else r.contiguous() for r in rows)
            rc = _lib.load().rwkv7_token_logprobs_grad(
                x.data_ptr(), code, ld, N, V, t.data_ptr(), temperature, _lib.ptr(s), one[0], _lib.ptr(h), one[1],
                _lib.ptr(logp), _lib.ptr(entropy), grad.data_ptr(), _lib.stream_of(x),
            )
            _lib.check(rc, "rwkv7_token_logprobs_grad")
    return logp, entropy, grad


def token_logprobs_grad(logits: Tensor, tokens: Tensor, *, temperature: float = 1.0, scale: Tensor | float = 1.0,
                        entropy_scale: Tensor | float = 0.0) -> tuple[Tensor, Tensor, Tensor]:
    """``token_logprobs`` and ``scale`` times the gradient of the log probability plus
    ``entropy_scale`` times that of the entropy, to ``logits``, in one pass over them:
    ``(logprob [...], entropy [...]`` float32, ``grad [..., V]`` of the logits' dtype``)``.
    The scales: numbers, or float32 ``[...]`` (each row's weight in the loss, -1 / rows
    for a mean cross entropy, and a loss scale), each / temperature within float32.
    Padded rows, rows of -inf alone and rows with both scales 0 have gradient 0. For
    ``logits.backward(grad)``."""
    return _token_grad(logits, tokens, temperature, scale, entropy_scale, True)


def token_logprobs_backward(grad_logprob: Tensor | None, grad_entropy: Tensor | None, logits: Tensor, tokens: Tensor,
                            temperature: float) -> Tensor:
    """Gradient of ``token_logprobs`` to ``logits`` under ``grad_logprob`` and
    ``grad_entropy`` float32 ``[...]`` (None: zeros)."""
    zero = lambda g: 0.0 if g is None else g  # noqa: E731
    return _token_grad(logits, tokens, temperature, zero(grad_logprob), zero(grad_entropy), False)[2]


def _strides(x: Tensor, V: int) -> Tensor:
    """``[B, R, V]`` with adjacent columns and rows that do not overlap."""
    ok = (x.stride(2) == 1 or V == 1) and (x.shape[1] <= 1 or x.stride(1) >= V) and x.stride(0) >= 0
    return x if ok else x.contiguous()


@lru_cache(maxsize=64)
def _verify_bytes(B: int, K: int, V: int) -> int:
    return _lib.load().rwkv7_verify_workspace_bytes(B, K, V)


def verify_draft(
    target_logits: Tensor,
    draft_tokens: Tensor,
    uniforms: Tensor | None,
    draft_logits: Tensor | None = None,
    *,
    temperature: float | None = None,
    draft_temperature: float | None = None,
    lengths: Tensor | None = None,
) -> tuple[Tensor, Tensor]:
    """Keep the drafted tokens that the target model lets pass, and draw the next.

    ``target_logits [B, K + 1, V]``: the target's logits after 0..K of the drafted
    tokens; ``draft_tokens [B, K]`` int64, K <= 63; ``uniforms [B, K + 1]`` float32
    in ``[0, 1)`` (K for the tokens, one for the draw); ``draft_logits [B, K, V]``:
    the logits the drafts were drawn from at ``draft_temperature`` (default:
    ``temperature``), of the target's dtype, or None for drafts without a draw
    (greedy ones, looked-up ones; ``draft_temperature <= 0`` is the same);
    ``lengths [B]`` int64: how many of each sequence's drafts count (None: all).
    Without the dimension B for a single sequence.

    Returns ``tokens [B, K + 1]`` int64 (the accepted ones, the next one, -1 behind
    it) and ``accepted [B]`` int64. The tokens are distributed as the target's own
    at ``temperature``; with ``temperature`` None or <= 0 they are its greedy ones
    and ``uniforms`` is not read. NaN logits count as -inf; ids outside ``0..V-1``
    are rejected."""
    code = _check_logits(target_logits, "target_logits")
    target, tokens, draft = target_logits, draft_tokens, draft_logits
    single = target.ndim == 2
    if single:
        up = lambda t: None if t is None else t.unsqueeze(0)  # noqa: E731
        target, tokens, draft, uniforms, lengths = up(target), up(tokens), up(draft), up(uniforms), up(lengths)
    if target.ndim != 3 or target.shape[1] < 1:
        raise ValueError(f"target_logits must be [B, K + 1, V], got {tuple(target_logits.shape)}")
    B, K, V = target.shape
    K -= 1
    if K > MAX_DRAFT:
        raise ValueError(f"at most {MAX_DRAFT} drafted tokens, got {K}")
    if B * (2 * K + 1) > 65535:
        raise ValueError(f"a batch of {B} with {K} drafts is too large: at most {65535 // (2 * K + 1)}")
    if tokens.shape != (B, K) or tokens.dtype is not torch.int64:
        raise ValueError(f"draft_tokens must be int64 [{B}, {K}], got {tokens.dtype} {tuple(tokens.shape)}")
    temperature = 0.0 if temperature is None else float(temperature)
    greedy = temperature <= 0
    if not greedy:
        _temperature(temperature)
        if uniforms is None:
            raise ValueError("uniforms are needed unless the temperature is None or <= 0")
    draft_temperature = temperature if draft_temperature is None else float(draft_temperature)
    if math.isnan(draft_temperature):
        raise ValueError("draft_temperature is NaN")
    if uniforms is not None:
        if uniforms.shape != (B, K + 1) or uniforms.dtype is not torch.float32:
            raise ValueError(f"uniforms must be float32 [{B}, {K + 1}], got {uniforms.dtype} {tuple(uniforms.shape)}")
    if draft is not None:
        _check_logits(draft, "draft_logits")
        if draft.shape != (B, K, V) or draft.dtype is not target.dtype:
            raise ValueError(f"draft_logits must be {target.dtype} [{B}, {K}, {V}], got {draft.dtype} {tuple(draft.shape)}")
        if not greedy and draft_temperature > 0:
            _temperature(draft_temperature)
        else:
            draft = None
    if lengths is not None:
        if lengths.shape != (B,) or lengths.dtype is not torch.int64:
            raise ValueError(f"lengths must be int64 [{B}]")
    _same_device(target, tokens, None if greedy else uniforms, draft, lengths)
    with _lib.device_of(target):
        dev = target.device
        out = torch.empty(B, K + 1, dtype=torch.int64, device=dev)
        accepted = torch.empty(B, dtype=torch.int64, device=dev)
        if B:
            lib = _lib.load()
            t = _strides(target, V)
            d = None if draft is None or K == 0 else _strides(draft, V)
            tok = tokens.contiguous()
            u = None if greedy else uniforms.contiguous()
            n = None if lengths is None else lengths.contiguous()
            nb = _verify_bytes(B, K, V)
            ws = torch.empty(nb, dtype=torch.uint8, device=dev)
            rc = lib.rwkv7_verify(
                t.data_ptr(), t.stride(0), t.stride(1) if K else V, _lib.ptr(d), 0 if d is None else d.stride(0),
                V if d is None or K == 1 else d.stride(1), code, tok.data_ptr() if K else None,
                _lib.ptr(u), _lib.ptr(n), B, K, V, temperature, draft_temperature, out.data_ptr(), accepted.data_ptr(),
                ws.data_ptr(), nb, _lib.stream_of(t),
            )
            _lib.check(rc, "rwkv7_verify")
    return (out[0], accepted[0]) if single else (out, accepted)
