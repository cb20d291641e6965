"""A paged key/value cache of 8-bit floats, half the bytes of a BF16 one: what a
server holds twice the positions in, and a decode step reads in half the time.

The pools are those of :mod:`.paged` with E4M3 codes (``float8_e4m3fn``) for
numbers, and a scale for every 32 channels of a row (``float8_e8m0fnu``, a power
of two, 2^-117 .. 2^119): a key or value is ``code * scale``, which BF16 holds exactly.
:func:`paged_append_fp8_` quantises the new tokens' keys and values as it stores
them; :func:`paged_attention_fp8` is :func:`.paged.paged_attention` over the
numbers that the cache stands for.  Tables, lengths and what they may say wrong
are as there.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from . import _lib, _registry
from .paged import SCALE_BLOCK, _attend, _check_append, _check_cache, store_op, validate_pages
from .pkda import _require_cuda, _require_device


@dataclass
class PagedKVFP8:
    """The keys and values of one attention layer as 8-bit floats."""

    k: Tensor        # float8_e4m3fn [num_pages, page_size, kv_heads, head_dim]
    v: Tensor
    k_scale: Tensor  # float8_e8m0fnu [num_pages, page_size, kv_heads, head_dim / 32]
    v_scale: Tensor

    @staticmethod
    def zeros(pages: int, page_size: int, kv_heads: int, head_dim: int, *,
              device: torch.device | str = "cuda") -> "PagedKVFP8":
        shape = (pages, page_size, kv_heads)
        k, v = (torch.zeros(*shape, head_dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
                for _ in range(2))
        one = 127  # the byte of the scale 1
        k_scale, v_scale = (torch.full((*shape, head_dim // SCALE_BLOCK), one, dtype=torch.uint8, device=device).view(
            torch.float8_e8m0fnu) for _ in range(2))
        return PagedKVFP8(k, v, k_scale, v_scale)


def paged_append_fp8_(
    k: Tensor,
    v: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    k_scales: Tensor,
    v_scales: Tensor,
    page_table: Tensor,
    seq_lens: Tensor,
    *,
    cu_seqlens: Tensor | None = None,
    q: Tensor | None = None,
    cos: Tensor | None = None,
    sin: Tensor | None = None,
    interleaved: bool = False,
    q_norm: Tensor | None = None,
    k_norm: Tensor | None = None,
    eps: float = 1e-6,
    check_pages: bool = False,
) -> Tensor | None:
    """:func:`.paged.paged_append_` into a cache of 8-bit floats; returns the
    queries in their own dtype (``None`` without ``q``).

    ``k_pages, v_pages`` float8_e4m3fn ``[P, page_size, kv_heads, head_dim]``
    with ``head_dim`` 64 or 128, ``k_scales, v_scales`` float8_e8m0fnu ``[P,
    page_size, kv_heads, head_dim / 32]``, all updated in place (pages of the
    codes any whole 16 bytes apart, of the scales any whole ``head_dim / 32``).
    Norms and rotation are FP32; a block of 32 channels takes the smallest scale
    of 2^-117 .. 2^119 by which its largest finite magnitude is at most 448, the
    largest code, and every number the code nearest to it over the scale, ties to
    even (past +-448, at the largest scale, +-448).  What is not finite is stored
    as NaN.
    """
    _require_device(k, v, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_seqlens, q, cos, sin, q_norm,
                    k_norm)
    _check_cache("k", k, k_pages, v_pages, page_table, seq_lens, cu_seqlens, (k_scales, v_scales))
    _check_append(k, v, k_pages, page_table, q, cos, sin, q_norm, k_norm)
    if check_pages:
        validate_pages(page_table, seq_lens, cu_seqlens, k.shape[0], k_pages.shape[0], k_pages.shape[1],
                       appended=True)
    if torch.compiler.is_compiling():
        # as the bytes they are: the compiler's default backend cannot have float8_e8m0fnu written in place
        k_scales, v_scales = k_scales.view(torch.uint8), v_scales.view(torch.uint8)
    out = _registry.launch(store_op, k, v, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_seqlens, q,
                           cos, sin, bool(interleaved), q_norm, k_norm, float(eps))
    return None if q is None else out


def paged_attention_fp8(
    q: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    k_scales: Tensor,
    v_scales: Tensor,
    page_table: Tensor,
    seq_lens: Tensor,
    *,
    cu_seqlens: Tensor | None = None,
    scale: float | None = None,
    check_pages: bool = False,
) -> tuple[Tensor, Tensor]:
    """:func:`.paged.paged_attention` over a cache of 8-bit floats; returns ``(o,
    lse)``, ``o`` in ``q.dtype`` (FP32 or BF16).  Keys and values are the numbers
    the cache stands for, exactly; nothing is rounded but what that operator
    rounds."""
    _require_device(q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_seqlens)
    _check_cache("q", q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, (k_scales, v_scales))
    if q.shape[1] < 1 or q.shape[1] % k_pages.shape[2]:
        raise ValueError(f"{q.shape[1]} query heads cannot share {k_pages.shape[2]} key/value heads")
    if check_pages:
        validate_pages(page_table, seq_lens, cu_seqlens, q.shape[0], k_pages.shape[0], k_pages.shape[1],
                       appended=False)
    return _registry.launch(attention_fp8_op, q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_seqlens,
                            q.shape[2] ** -0.5 if scale is None else float(scale))


@_registry.device_op(
    "paged_attention_fp8(Tensor q, Tensor k_pages, Tensor v_pages, Tensor k_scales, Tensor v_scales, Tensor page_table, "
    "Tensor seq_lens, Tensor? cu_seqlens, float scale) -> (Tensor, Tensor)")
def attention_fp8_op(
    q: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor, page_table: Tensor,
    seq_lens: Tensor, cu_seqlens: Tensor | None, scale: float,
) -> tuple[Tensor, Tensor]:
    """The attention's launches (arguments checked by :func:`paged_attention_fp8`)."""
    device = _require_cuda(q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_seqlens)
    return _attend(_lib.PagedAttentionFP8Args, "pkda_paged_attention_fp8", "pkda_paged_attention_fp8_workspace", device, q,
                   k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_seqlens, scale)


def _attention_fp8_fake(q, *rest):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


_registry.register_fake(attention_fp8_op, _attention_fp8_fake)
