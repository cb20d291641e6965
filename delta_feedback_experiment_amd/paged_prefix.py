"""Attention of a batch whose sequences share long prefixes: a common instruction,
a document that many ask about, the samples of one prompt.  The shared positions
are read once for all of a group's rows, not once a sequence."""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib, _registry
from .paged import _attend, _check_cache, _ints, validate_pages
from .pkda import _ptr, _require_cuda, _require_device


def validate_groups(cu_groups: Tensor, prefix_lens: Tensor, seq_lens: Tensor) -> None:
    """Host-side check of a batch's groups (synchronises): bounds that rise from 0
    over the sequences, prefixes that every sequence of their group holds."""
    cu, prefix, lens = cu_groups.cpu().tolist(), prefix_lens.cpu().tolist(), seq_lens.cpu().tolist()
    if cu[0] != 0 or any(a > b for a, b in zip(cu, cu[1:])) or cu[-1] > len(lens):
        raise ValueError(f"cu_groups must rise from 0 to at most {len(lens)}, got {cu}")
    for g, length in enumerate(prefix):
        held = min(lens[cu[g]:cu[g + 1]], default=length)
        if not 0 <= length <= held:
            raise ValueError(f"prefix_lens[{g}] = {length} must be positions of all its sequences, the shortest of "
                             f"which holds {held}")


def paged_prefix_attention(
    q: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    page_table: Tensor,
    seq_lens: Tensor,
    cu_groups: Tensor,
    prefix_lens: Tensor,
    *,
    k_scales: Tensor | None = None,
    v_scales: Tensor | None = None,
    cu_seqlens: Tensor | None = None,
    scale: float | None = None,
    check_pages: bool = False,
) -> tuple[Tensor, Tensor]:
    """:func:`.paged.paged_attention` of a batch in groups; returns ``(o, lse)``.

    Sequences ``cu_groups[g] .. cu_groups[g + 1] - 1`` (int32 ``[groups + 1]``)
    share their first ``prefix_lens[g]`` positions (int32 ``[groups]``, any number
    of them, zero too): the same keys and values, in the same pages or in copies.
    Every sequence's row of ``page_table`` names the pages of all its positions,
    the shared ones too; from which of a group's rows those are read is not said.
    One that holds fewer positions than the prefix (a finished slot, of length 0) sees
    what it holds of it and takes nothing from the others, whatever its row says past
    its length; ``check_pages`` refuses it.  Sequences past ``cu_groups[-1]`` share nothing.  Otherwise arguments and result
    are those of :func:`.paged.paged_attention`, or with ``k_scales, v_scales`` of
    :func:`.paged_fp8.paged_attention_fp8`; both read the groups on the device, so
    that a captured step follows them.

    What is saved is the reading of the prefix.  A batch of chunks alone that fill the
    card reads it often enough to be bound by products, and takes up to a fifth less
    time by those operators (16 sequences of 512 new tokens behind 4,096, 32/8 heads:
    689 us, and 874 by this one).
    """
    _require_device(q, k_pages, v_pages, page_table, seq_lens, cu_groups, prefix_lens, k_scales, v_scales, cu_seqlens)
    if (k_scales is None) != (v_scales is None):
        raise ValueError("k_scales and v_scales go together")
    _check_cache("q", q, k_pages, v_pages, page_table, seq_lens, cu_seqlens,
                 None if k_scales is None else (k_scales, v_scales))
    if q.shape[1] < 1 or q.shape[1] % k_pages.shape[2]:
        raise ValueError(f"{q.shape[1]} query heads cannot share {k_pages.shape[2]} key/value heads")
    if prefix_lens.dtype != torch.int32 or prefix_lens.dim() != 1:
        raise ValueError("prefix_lens must be int32 [groups]")
    if cu_groups.dtype != torch.int32 or tuple(cu_groups.shape) != (prefix_lens.shape[0] + 1,):
        raise ValueError(f"cu_groups must be int32 [{prefix_lens.shape[0] + 1}]")
    if check_pages:
        validate_pages(page_table, seq_lens, cu_seqlens, q.shape[0], k_pages.shape[0], k_pages.shape[1],
                       appended=False)
        validate_groups(cu_groups, prefix_lens, seq_lens)
    return _registry.launch(prefix_op, q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_groups,
                            prefix_lens, cu_seqlens, q.shape[2] ** -0.5 if scale is None else float(scale))


@_registry.device_op(
    "paged_prefix_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor? k_scales, Tensor? v_scales, "
    "Tensor page_table, Tensor seq_lens, Tensor cu_groups, Tensor prefix_lens, Tensor? cu_seqlens, float scale) "
    "-> (Tensor, Tensor)")
def prefix_op(
    q: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor | None, v_scales: Tensor | None, page_table: Tensor,
    seq_lens: Tensor, cu_groups: Tensor, prefix_lens: Tensor, cu_seqlens: Tensor | None, scale: float,
) -> tuple[Tensor, Tensor]:
    """The attention's launches (arguments checked by :func:`paged_prefix_attention`)."""
    device = _require_cuda(q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_groups, prefix_lens,
                           cu_seqlens)
    cu_groups, prefix_lens = _ints(cu_groups), _ints(prefix_lens)
    return _attend(_lib.PagedPrefixArgs, "pkda_paged_prefix_attention", "pkda_paged_prefix_workspace", device, q,
                   k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_seqlens, scale,
                   cu_groups=_ptr(cu_groups), prefix_lens=_ptr(prefix_lens), num_groups=prefix_lens.shape[0])


def _prefix_fake(q, *rest):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


_registry.register_fake(prefix_op, _prefix_fake)
