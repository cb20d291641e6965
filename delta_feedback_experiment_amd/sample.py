"""The next token of every row of logits: temperature, top-k, top-p and min-p,
from random numbers the caller gives."""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib, _registry
from .pkda import _dtype_code, _on, _ptr, _require_cuda, _require_device, _stream


def _setting(name: str, value, off, rows: int, dtype: torch.dtype) -> tuple[Tensor | None, float | int]:
    """One of the settings as a tensor of one value a row, or as one number."""
    if not isinstance(value, Tensor):
        return None, off if value is None else type(off)(value)
    if value.dtype != dtype or tuple(value.shape) != (rows,):
        raise ValueError(f"{name} must be {dtype} [{rows}] or a number")
    return value, off


def sample_tokens(
    logits: Tensor,
    noise: Tensor,
    *,
    temperature: float | Tensor | None = None,
    top_k: int | Tensor | None = None,
    top_p: float | Tensor | None = None,
    min_p: float | Tensor | None = None,
) -> tuple[Tensor, Tensor]:
    """Draw one token from every row; returns ``(token, logprob)``.

    ``logits [rows, vocab]`` FP32 or BF16 and ``noise [rows, vocab]`` FP32
    Gumbel numbers (``torch.empty(...).exponential_().log_().neg_()``), rows
    any distance apart; each setting a number or a tensor of one value a row
    (FP32; ``top_k`` int32).  Per row, with tokens in order of their logits
    (falling, ties by index), ``z = (logits - max) / temperature`` and ``w =
    exp(z)``:

    * ``top_k``: the first ``top_k`` tokens (all of them for ``top_k <= 0``);
    * ``top_p``: of those, the tokens before which they hold less than
      ``top_p`` of their ``w`` (all for ``top_p >= 1``; always the first);
    * ``min_p``: the tokens with ``w >= min_p``, the most likely one's being 1.

    The token is the lowest index that maximises ``z + noise`` over what is
    left: a draw from the softmax over it.  ``temperature <= 0`` takes the
    first token, an infinite one makes every ``z`` 0.  ``token [rows]`` int32;
    ``logprob [rows]`` FP32 is its ``log_softmax(logits)``, before any setting.

    Logits of NaN or -inf are never taken, +inf counts as the largest finite
    number; a row that holds nothing else gives token -1 and logprob -inf.
    """
    _require_device(logits, noise, *(t for t in (temperature, top_k, top_p, min_p) if isinstance(t, Tensor)))
    if logits.dim() != 2 or noise.shape != logits.shape or logits.shape[1] < 1:
        raise ValueError(f"logits and noise [rows, vocab] expected, got {tuple(logits.shape)} and "
                         f"{tuple(noise.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16) or noise.dtype != torch.float32:
        raise ValueError(f"logits float32 or bfloat16 and noise float32 expected, not {logits.dtype}, {noise.dtype}")
    rows = logits.shape[0]
    settings = (_setting("temperature", temperature, 1.0, rows, torch.float32),
                _setting("top_k", top_k, 0, rows, torch.int32), _setting("top_p", top_p, 1.0, rows, torch.float32),
                _setting("min_p", min_p, 0.0, rows, torch.float32))
    return _registry.launch(sample_op, logits, noise, *(s[0] for s in settings), *(s[1] for s in settings))


def _rows(t: Tensor) -> Tensor:
    return t if t.stride(1) == 1 and t.stride(0) >= 0 else t.contiguous()


@_registry.device_op(
    "sample_tokens(Tensor logits, Tensor noise, Tensor? temperature, Tensor? top_k, Tensor? top_p, Tensor? min_p, "
    "float temperature_all, SymInt top_k_all, float top_p_all, float min_p_all) -> (Tensor, Tensor)")
def sample_op(
    logits: Tensor, noise: Tensor, temperature: Tensor | None, top_k: Tensor | None, top_p: Tensor | None,
    min_p: Tensor | None, temperature_all: float, top_k_all: int, top_p_all: float, min_p_all: float,
) -> tuple[Tensor, Tensor]:
    """The sampling's launch (arguments checked by :func:`sample_tokens`)."""
    device = _require_cuda(logits, noise, temperature, top_k, top_p, min_p)
    logits, noise = _rows(logits), _rows(noise)
    rows, vocab = logits.shape
    settings = [None if t is None else t.contiguous() for t in (temperature, top_k, top_p, min_p)]
    token = torch.empty(rows, dtype=torch.int32, device=device)
    logprob = torch.empty(rows, dtype=torch.float32, device=device)
    args = _lib.SampleArgs(
        dtype=_dtype_code(logits), rows=rows, vocab=vocab, logits=_ptr(logits), logits_stride=logits.stride(0),
        noise=_ptr(noise), noise_stride=noise.stride(0), temperature=_ptr(settings[0]), top_k=_ptr(settings[1]),
        top_p=_ptr(settings[2]), min_p=_ptr(settings[3]), temperature_all=temperature_all,
        top_k_all=max(0, min(int(top_k_all), vocab)), top_p_all=top_p_all, min_p_all=min_p_all, token=_ptr(token),
        logprob=_ptr(logprob),
    )
    with _on(device):
        _lib.call("pkda_sample", args, _stream(device))
    return token, logprob


def _sample_fake(logits, *args):
    return tuple(logits.new_empty(logits.shape[:1], dtype=t) for t in (torch.int32, torch.float32))


_registry.register_fake(sample_op, _sample_fake)
