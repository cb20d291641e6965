"""Drafted tokens against the target's probabilities: which of them stand, and the
token after them, from random numbers the caller gives."""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from . import _lib, _registry
from .paged import _ints
from .pkda import _dtype_code, _on, _ptr, _require_cuda, _require_device, _stream
from .sample import _rows, _setting


def verify_tokens(
    logits: Tensor,
    drafts: Tensor,
    uniform: Tensor,
    noise: Tensor,
    cu_seqlens: Tensor,
    *,
    draft_logits: Tensor | None = None,
    temperature: float | Tensor | None = None,
) -> tuple[Tensor, Tensor]:
    """Accept or reject the drafts of every sequence; returns ``(tokens, accepted)``.

    Rows are packed: those of sequence ``n`` are ``cu_seqlens[n] ..
    cu_seqlens[n + 1] - 1`` (int32 ``[S + 1]``), one more than it has drafts.  Row
    ``j`` of them is what the target says after the sequence's first ``j`` drafts:
    ``logits [rows, vocab]`` FP32 or BF16, rows any distance apart.  ``drafts``
    int32, ``uniform`` FP32 numbers of [0, 1) (both ``[rows]``) and ``draft_logits``
    (as ``logits``; what the drafts were drawn from) hold in row ``j`` those of
    draft ``j``, and in a sequence's last row anything.  ``noise [S, vocab]`` FP32
    Gumbel numbers (``torch.empty(...).exponential_().log_().neg_()``);
    ``temperature`` a number or FP32 ``[S]``.

    With ``p = softmax(logits / temperature)`` and ``q = softmax(draft_logits /
    temperature)`` -- without ``draft_logits``, 1 at the draft: one that was looked
    up, or taken greedily -- drafts ``d`` are accepted in turn while ``uniform *
    q[d] < p[d]``.  The next token is then the lowest index that maximises
    ``log(r) + noise`` over ``r > 0``: in the row of the first draft that is not
    accepted ``r = max(p - q, 0)`` (``p`` where that leaves nothing), in a
    sequence's last row, and in one without a draft, ``r = p``.  Drafts and next
    token together are draws from the target alone.  ``temperature <= 0`` accepts a
    draft that is the (first) largest logit's and takes that token next.

    ``tokens [rows]`` int32: in a sequence's rows its accepted drafts, the next
    token, then -1; -1 in rows past ``cu_seqlens[-1]``.  ``accepted [S]`` int32
    counts the drafts that stand (0 for a sequence without rows).

    Logits of NaN or -inf have probability 0, +inf counts as the largest finite
    number: a top-k or top-p cut is made by -inf.  A draft outside the vocabulary
    (-1: the row has none) is not accepted.  A row that holds no logit accepts nothing
    and its token is -1.
    """
    given = [t for t in (temperature,) if isinstance(t, Tensor)]
    _require_device(logits, drafts, uniform, noise, cu_seqlens, draft_logits, *given)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits [rows, vocab] expected, got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits float32 or bfloat16 expected, not {logits.dtype}")
    if draft_logits is not None and (draft_logits.shape != logits.shape or draft_logits.dtype != logits.dtype):
        raise ValueError(f"draft_logits {tuple(draft_logits.shape)} {draft_logits.dtype} must be as logits "
                         f"{tuple(logits.shape)} {logits.dtype}")
    if drafts.dtype != torch.int32 or tuple(drafts.shape) != (rows,):
        raise ValueError(f"drafts must be int32 [{rows}]")
    if uniform.dtype != torch.float32 or tuple(uniform.shape) != (rows,):
        raise ValueError(f"uniform must be float32 [{rows}]")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be int32 [sequences + 1]")
    S = cu_seqlens.shape[0] - 1
    if noise.dtype != torch.float32 or tuple(noise.shape) != (S, vocab):
        raise ValueError(f"noise must be float32 [{S}, {vocab}]")
    heat, heat_all = _setting("temperature", temperature, 1.0, S, torch.float32)
    return _registry.launch(verify_op, logits, drafts, uniform, noise, cu_seqlens, draft_logits, heat, heat_all)


@_registry.device_op(
    "verify_tokens(Tensor logits, Tensor drafts, Tensor uniform, Tensor noise, Tensor cu_seqlens, Tensor? draft_logits, "
    "Tensor? temperature, float temperature_all) -> (Tensor, Tensor)")
def verify_op(
    logits: Tensor, drafts: Tensor, uniform: Tensor, noise: Tensor, cu_seqlens: Tensor, draft_logits: Tensor | None,
    temperature: Tensor | None, temperature_all: float,
) -> tuple[Tensor, Tensor]:
    """The verification's launches (arguments checked by :func:`verify_tokens`)."""
    device = _require_cuda(logits, drafts, uniform, noise, cu_seqlens, draft_logits, temperature)
    logits, noise = _rows(logits), _rows(noise)
    draft_logits = None if draft_logits is None else _rows(draft_logits)
    drafts, uniform, cu_seqlens = _ints(drafts), _ints(uniform), _ints(cu_seqlens)
    temperature = None if temperature is None else temperature.contiguous()
    rows, vocab = logits.shape
    seqs = cu_seqlens.shape[0] - 1
    tokens = torch.empty(rows, dtype=torch.int32, device=device)
    accepted = torch.empty(seqs, dtype=torch.int32, device=device)
    args = _lib.VerifyArgs(
        dtype=_dtype_code(logits), rows=rows, vocab=vocab, num_seqs=seqs, logits=_ptr(logits),
        logits_stride=logits.stride(0), draft_logits=_ptr(draft_logits),
        draft_stride=0 if draft_logits is None else draft_logits.stride(0), drafts=_ptr(drafts), uniform=_ptr(uniform),
        noise=_ptr(noise), noise_stride=noise.stride(0), cu_seqlens=_ptr(cu_seqlens), temperature=_ptr(temperature),
        temperature_all=temperature_all, tokens=_ptr(tokens), accepted=_ptr(accepted),
    )
    args.struct_size = ctypes.sizeof(args)
    floats = _lib.lib().pkda_verify_workspace(ctypes.byref(args))
    workspace = torch.empty(floats, dtype=torch.float32, device=device) if floats > 0 else None
    args.workspace = _ptr(workspace)
    with _on(device):
        _lib.call("pkda_verify", args, _stream(device))
    return tokens, accepted


def _verify_fake(logits, drafts, uniform, noise, cu_seqlens, *rest):
    return (logits.new_empty(logits.shape[:1], dtype=torch.int32),
            logits.new_empty((cu_seqlens.shape[0] - 1,), dtype=torch.int32))


_registry.register_fake(verify_op, _verify_fake)
