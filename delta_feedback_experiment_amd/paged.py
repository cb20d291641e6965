"""A paged key/value cache and the attention of new tokens over it: what the
attention layers of a trunk keep between calls, where the PKDA layers keep
:class:`.serve.DecodePool`.

The cache is two pools of pages, ``[num_pages, page_size, kv_heads, head_dim]``
in the activation dtype.  Position ``p`` of sequence ``n`` is row ``p %
page_size`` of page ``page_table[n, p // page_size]``; which page is whose is
the caller's to say.  ``seq_lens[n]`` counts the sequence's positions with its
new tokens, which are its last ones.

:func:`paged_append_` stores the new tokens' keys and values, turning keys and
queries by their position on the way; :func:`paged_attention` is causal
attention of the new tokens over everything their sequence holds.  Tokens are
packed ``[N_tok, heads, head_dim]`` with ``cu_seqlens`` as elsewhere, or one a
sequence without: the decode step.  Neither records autograd history.

Device data that names what does not exist stays inside the buffers: a length
past the table's row is cut to it, ``cu_seqlens`` is clamped to the packed
length and begins at 0, a page number outside the pool holds nothing, a token of
no sequence (padding past ``cu_seqlens[-1]``) is stored nowhere and attends to
nothing.  ``cu_seqlens`` that falls names no sequences: what the tokens' outputs
and their sequences' rows then hold is undefined.  ``check_pages=True`` raises
instead, at the price of a copy to the host.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch
from torch import Tensor

from . import _lib, _registry
from .pkda import _dtype_code, _on, _ptr, _require_cuda, _require_device, _stream

HEAD_DIMS = (32, 64, 128)


@dataclass
class PagedKV:
    """The keys and values of one attention layer."""

    k: Tensor  # [num_pages, page_size, kv_heads, head_dim]
    v: Tensor

    @staticmethod
    def zeros(pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda") -> "PagedKV":
        shape = (pages, page_size, kv_heads, head_dim)
        return PagedKV(*(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)))


def _check_cache(name: str, x: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seq_lens: Tensor,
                 cu_seqlens: Tensor | None) -> None:
    """The checks the two operators share; ``x`` is a token tensor."""
    shape, pages, dtype, lens = x.shape, k_pages.shape, x.dtype, seq_lens.shape
    if len(shape) != 3:
        raise ValueError(f"{name} [tokens, heads, head_dim] expected, got {tuple(shape)}")
    if len(pages) != 4 or pages != v_pages.shape:
        raise ValueError(f"k_pages {tuple(pages)} and v_pages {tuple(v_pages.shape)} must be one "
                         "[pages, page_size, kv_heads, head_dim] shape")
    if dtype != k_pages.dtype or dtype != v_pages.dtype:
        raise ValueError(f"{name} {dtype} and the pages {k_pages.dtype}, {v_pages.dtype} must share one dtype")
    if dtype != torch.bfloat16 and dtype != torch.float32:
        raise ValueError(f"float32 or bfloat16 expected, not {dtype}")
    _, R, H, D = pages
    if shape[2] != D or D not in HEAD_DIMS:
        raise ValueError(f"head_dim {shape[2]} of {name} and {D} of the pages: one of {HEAD_DIMS} expected")
    if R < 1 or H < 1:
        raise ValueError(f"pages {tuple(pages)} hold nothing")
    if seq_lens.dtype != torch.int32 or len(lens) != 1:
        raise ValueError("seq_lens must be int32 [sequences]")
    S, table = lens[0], page_table.shape
    if page_table.dtype != torch.int32 or len(table) != 2 or table[0] != S:
        raise ValueError(f"page_table must be int32 [{S}, pages of a sequence]")
    if cu_seqlens is None:
        if shape[0] != S:
            raise ValueError(f"{shape[0]} tokens of {S} sequences need cu_seqlens")
    elif cu_seqlens.dtype != torch.int32 or tuple(cu_seqlens.shape) != (S + 1,):
        raise ValueError(f"cu_seqlens must be int32 [{S + 1}]")
    for t in (k_pages, v_pages):
        stride = t.stride()
        if (stride[3] != 1 or (stride[2] != D and H > 1) or (stride[1] != H * D and R > 1)
                or not _aligned(t, stride[0])) and t.numel():
            raise ValueError("every page must be dense, in whole 16 bytes")


def _aligned(t: Tensor, stride: int) -> bool:
    # fake tensors have no address: the offset is what a view adds to its storage (a
    # compiler's trace has no offset either; the launch checks the address)
    offset = 0 if torch.compiler.is_compiling() else t.storage_offset()
    return (stride | offset) * t.element_size() % 16 == 0


def _rows(t: Tensor) -> Tensor:
    """Tokens as the kernels read them: heads dense, tokens any whole 16 bytes apart."""
    _, H, D = t.shape
    token, head, channel = t.stride()
    if channel == 1 and (head == D or H == 1) and token >= 0 and _aligned(t, token):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _ints(t: Tensor) -> Tensor:
    stride = t.stride()
    return t if stride[-1] == 1 and stride[0] >= 0 else t.contiguous()


def validate_pages(page_table: Tensor, seq_lens: Tensor, cu_seqlens: Tensor | None, num_tokens: int, num_pages: int,
                   page_size: int, *, appended: bool) -> None:
    """Host-side check of a cache's tables (synchronises): lengths, document
    bounds and page numbers in range, and, where new tokens are stored, no row
    of the pools stored twice."""
    lens, table = seq_lens.cpu().tolist(), page_table.cpu().tolist()
    cu = list(range(len(lens) + 1)) if cu_seqlens is None else cu_seqlens.cpu().tolist()
    if cu[0] != 0 or any(a > b for a, b in zip(cu, cu[1:])) or cu[-1] > num_tokens:
        raise ValueError(f"cu_seqlens must rise from 0 to at most {num_tokens}, got {cu}")
    stored = set()
    for n, length in enumerate(lens):
        new = cu[n + 1] - cu[n]
        if length < new or length > len(table[n]) * page_size:
            raise ValueError(f"seq_lens[{n}] = {length} must hold its {new} new tokens and fit "
                             f"{len(table[n])} pages of {page_size}")
        for i in range(-(-length // page_size)):
            if not 0 <= table[n][i] < num_pages:
                raise IndexError(f"page_table[{n}, {i}] = {table[n][i]} is out of range [0, {num_pages})")
        for p in range(length - new, length) if appended else ():
            row = (table[n][p // page_size], p % page_size)
            if row in stored:
                raise ValueError(f"position {p} of sequence {n} is stored over another new token (page, row {row})")
            stored.add(row)


def paged_append_(
    k: Tensor,
    v: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    page_table: Tensor,
    seq_lens: Tensor,
    *,
    cu_seqlens: Tensor | None = None,
    q: Tensor | None = None,
    cos: Tensor | None = None,
    sin: Tensor | None = None,
    interleaved: bool = False,
    check_pages: bool = False,
) -> Tensor | None:
    """Store new keys and values in the cache; returns the rotated queries
    (``None`` without ``q``).

    ``k, v [N_tok, kv_heads, head_dim]`` and ``q [N_tok, q_heads, head_dim]``
    (slices of one packed projection are taken as they are); ``k_pages,
    v_pages [P, page_size, kv_heads, head_dim]``, updated in place (pages may
    be any distance apart, as in one pool of both); ``page_table`` int32
    ``[S, pages]``, ``seq_lens`` int32 ``[S]`` with the new tokens,
    ``cu_seqlens`` int32 ``[S + 1]`` (``None``: one token a sequence).

    With ``cos, sin`` (FP32 ``[positions, rotary / 2]``, one row for every
    position of a table row) the first ``rotary`` channels (a multiple of 16)
    of ``q`` and ``k`` turn by their position's angles: pairs ``(c, c + rotary
    / 2)``, or ``(2c, 2c + 1)`` when ``interleaved``.  Without, they are
    copied.  Rows of the result whose token has no position are zeros.
    """
    _require_device(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, q, cos, sin)
    _check_cache("k", k, k_pages, v_pages, page_table, seq_lens, cu_seqlens)
    if v.shape != k.shape or v.dtype != k.dtype or k.shape[1] != k_pages.shape[2]:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} and pages of {k_pages.shape[2]} heads must match")
    if q is not None and (q.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.dtype != k.dtype
                          or q.shape[1] < 1):
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} does not match k {tuple(k.shape)} {k.dtype}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        capacity = page_table.shape[1] * k_pages.shape[1]
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise ValueError("cos and sin must be float32 [positions, rotary / 2]")
        if cos.shape[1] % 8 or not 0 < 2 * cos.shape[1] <= k.shape[2]:
            raise ValueError(f"rotary dim {2 * cos.shape[1]}: a multiple of 16 up to {k.shape[2]} expected")
        if cos.shape[0] < capacity:
            raise ValueError(f"cos and sin hold {cos.shape[0]} positions, a row of page_table {capacity}")
    if check_pages:
        validate_pages(page_table, seq_lens, cu_seqlens, k.shape[0], k_pages.shape[0], k_pages.shape[1],
                       appended=True)
    out = _registry.launch(append_op, k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, q, cos, sin,
                           bool(interleaved))
    return None if q is None else out


@_registry.device_op(
    "paged_append_(Tensor k, Tensor v, Tensor(a2!) k_pages, Tensor(a3!) v_pages, Tensor page_table, Tensor seq_lens, "
    "Tensor? cu_seqlens, Tensor? q, Tensor? cos, Tensor? sin, bool interleaved) -> Tensor")
def append_op(
    k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seq_lens: Tensor,
    cu_seqlens: Tensor | None, q: Tensor | None, cos: Tensor | None, sin: Tensor | None, interleaved: bool,
) -> Tensor:
    """The append's launch (arguments checked by :func:`paged_append_`):
    writes the cache's rows and returns the rotated queries (without ``q``,
    an empty tensor)."""
    _require_cuda(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, q, cos, sin)
    k, v = _rows(k), _rows(v)
    q = None if q is None else _rows(q)
    q_out = k.new_empty((0,) if q is None else q.shape)
    if cos is not None:
        cos, sin = (t if t.is_contiguous() and _aligned(t, 0) else t.clone(memory_format=torch.contiguous_format)
                    for t in (cos, sin))
    page_table, seq_lens = _ints(page_table), _ints(seq_lens)
    cu_seqlens = None if cu_seqlens is None else _ints(cu_seqlens)
    args = _lib.PagedAppendArgs(
        dtype=_dtype_code(k), num_seqs=seq_lens.shape[0], num_tokens=k.shape[0],
        q_heads=0 if q is None else q.shape[1], kv_heads=k.shape[1], head_dim=k.shape[2],
        page_size=k_pages.shape[1], max_pages=page_table.shape[1], num_pages=k_pages.shape[0],
        table_stride=page_table.stride(0), cu_seqlens=_ptr(cu_seqlens), seq_lens=_ptr(seq_lens),
        page_table=_ptr(page_table), q=_ptr(q), k=_ptr(k), v=_ptr(v),
        q_stride=0 if q is None else q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0),
        q_out=_ptr(q_out), k_pages=_ptr(k_pages), v_pages=_ptr(v_pages),
        k_page_stride=k_pages.stride(0), v_page_stride=v_pages.stride(0), cos=_ptr(cos), sin=_ptr(sin),
        rotary_dim=0 if cos is None else 2 * cos.shape[1], interleaved=int(interleaved),
        rope_rows=0 if cos is None else cos.shape[0],
    )
    with _on(k.device):
        _lib.call("pkda_paged_append", args, _stream(k.device))
    return q_out


def _append_fake(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, q, cos, sin, interleaved):
    return k.new_empty((0,) if q is None else q.shape)


_registry.register_fake(append_op, _append_fake)


def paged_attention(
    q: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    page_table: Tensor,
    seq_lens: Tensor,
    *,
    cu_seqlens: Tensor | None = None,
    scale: float | None = None,
    check_pages: bool = False,
) -> tuple[Tensor, Tensor]:
    """Causal attention of new tokens over the cache; returns ``(o, lse)``.

    ``q [N_tok, q_heads, head_dim]`` (tokens may be strided); the cache as
    :func:`paged_append_` left it, the new tokens' keys and values in it;
    query head ``h`` reads key/value head ``h // (q_heads / kv_heads)``.  A
    sequence of ``n`` new tokens and length ``L`` has them at positions ``L -
    n .. L - 1``; each sees its own and every earlier position.  ``o [N_tok,
    q_heads, head_dim]`` in ``q.dtype``; ``lse [N_tok, q_heads]`` FP32 is the
    natural log of the softmax's sum, by which attention over other keys can
    be joined to this one.  A token without keys has ``o = 0``, ``lse =
    -inf``.  ``scale`` defaults to ``head_dim ** -0.5``.
    """
    _require_device(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens)
    _check_cache("q", q, k_pages, v_pages, page_table, seq_lens, cu_seqlens)
    if q.shape[1] < 1 or q.shape[1] % k_pages.shape[2]:
        raise ValueError(f"{q.shape[1]} query heads cannot share {k_pages.shape[2]} key/value heads")
    if check_pages:
        validate_pages(page_table, seq_lens, cu_seqlens, q.shape[0], k_pages.shape[0], k_pages.shape[1],
                       appended=False)
    return _registry.launch(attention_op, q, k_pages, v_pages, page_table, seq_lens, cu_seqlens,
                            q.shape[2] ** -0.5 if scale is None else float(scale))


@_registry.device_op(
    "paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor seq_lens, "
    "Tensor? cu_seqlens, float scale) -> (Tensor, Tensor)")
def attention_op(
    q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seq_lens: Tensor, cu_seqlens: Tensor | None,
    scale: float,
) -> tuple[Tensor, Tensor]:
    """The attention's launches (arguments checked by :func:`paged_attention`)."""
    device = _require_cuda(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens)
    q = _rows(q)
    page_table, seq_lens = _ints(page_table), _ints(seq_lens)
    cu_seqlens = None if cu_seqlens is None else _ints(cu_seqlens)
    N, Hq, D = q.shape
    o = torch.empty(N, Hq, D, dtype=q.dtype, device=device)
    lse = torch.empty(N, Hq, dtype=torch.float32, device=device)
    args = _lib.PagedAttentionArgs(
        dtype=_dtype_code(q), num_seqs=seq_lens.shape[0], num_tokens=N, q_heads=Hq, kv_heads=k_pages.shape[2],
        head_dim=D, page_size=k_pages.shape[1], max_pages=page_table.shape[1], num_pages=k_pages.shape[0],
        table_stride=page_table.stride(0), cu_seqlens=_ptr(cu_seqlens), seq_lens=_ptr(seq_lens),
        page_table=_ptr(page_table), q=_ptr(q), q_stride=q.stride(0), k_pages=_ptr(k_pages), v_pages=_ptr(v_pages),
        k_page_stride=k_pages.stride(0), v_page_stride=v_pages.stride(0), scale=scale, o=_ptr(o), lse=_ptr(lse),
    )
    args.struct_size = ctypes.sizeof(args)
    floats = _lib.lib().pkda_paged_attention_workspace(ctypes.byref(args))
    workspace = torch.empty(floats, dtype=torch.float32, device=device) if floats > 0 else None
    args.workspace = _ptr(workspace)
    with _on(device):
        _lib.call("pkda_paged_attention", args, _stream(device))
    return o, lse


def _attention_fake(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


_registry.register_fake(attention_op, _attention_fake)
