"""A paged key/value cache and attention over it, in 64 bits on the CPU, one
token at a time."""

from __future__ import annotations

import torch
from torch import Tensor


def spans(seq_lens, cu_seqlens, num_tokens: int):
    """(sequence, position) of every token, or None for a token of none."""
    lens = seq_lens.tolist()
    cu = list(range(len(lens) + 1)) if cu_seqlens is None else cu_seqlens.tolist()
    out = [None] * num_tokens
    for n, length in enumerate(lens):
        new = cu[n + 1] - cu[n]
        for j in range(new):
            pos = length - new + j
            out[cu[n] + j] = (n, pos) if pos >= 0 else None
    return out


def rotate(x: Tensor, pos: int, cos: Tensor, sin: Tensor, interleaved: bool) -> Tensor:
    """One token's heads ``[H, D]`` turned by the angles of row ``pos``, in 64 bits."""
    x = x.double().clone()
    r = 2 * cos.shape[1]
    c, s = cos[pos].double(), sin[pos].double()
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[:, first].clone(), x[:, second].clone()
    x[:, first], x[:, second] = a * c - b * s, b * c + a * s
    return x


def append_reference(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens=None, q=None, cos=None, sin=None,
                     interleaved=False):
    """``(q_out, k_pages, v_pages)`` in 64 bits; the inputs stay as they are."""
    kp, vp = k_pages.double().clone(), v_pages.double().clone()
    P, R = kp.shape[:2]
    q_out = None if q is None else torch.zeros(q.shape, dtype=torch.float64)
    for t, at in enumerate(spans(seq_lens, cu_seqlens, k.shape[0])):
        if at is None:
            continue
        n, pos = at
        turn = (lambda x: x.double()) if cos is None else (lambda x: rotate(x, pos, cos, sin, interleaved))
        if q is not None:
            q_out[t] = turn(q[t])
        page = int(page_table[n, pos // R])
        if 0 <= page < P:
            kp[page, pos % R], vp[page, pos % R] = turn(k[t]), v[t].double()
    return q_out, kp, vp


def attention_reference(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens=None, scale=None):
    """``(o, lse)`` in 64 bits."""
    N, Hq, D = q.shape
    P, R, Hkv = k_pages.shape[:3]
    scale = D ** -0.5 if scale is None else scale
    o, lse = torch.zeros(N, Hq, D, dtype=torch.float64), torch.full((N, Hq), -torch.inf, dtype=torch.float64)
    for t, at in enumerate(spans(seq_lens, cu_seqlens, N)):
        if at is None:
            continue
        n, pos = at
        rows = [(int(page_table[n, p // R]), p % R) for p in range(pos + 1)]
        rows = [r for r in rows if 0 <= r[0] < P]
        if not rows:
            continue
        page, row = (torch.tensor(x) for x in zip(*rows))
        k, v = k_pages[page, row].double(), v_pages[page, row].double()  # [L, Hkv, D]
        for h in range(Hq):
            s = scale * (k[:, h // (Hq // Hkv)] @ q[t, h].double())
            lse[t, h] = torch.logsumexp(s, 0)
            o[t, h] = torch.softmax(s, 0) @ v[:, h // (Hq // Hkv)]
    return o, lse


def attention_of_sequences(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale=None):
    """``attention_reference`` a sequence at a time, for longer ones."""
    N, Hq, D = q.shape
    P, R, Hkv = k_pages.shape[:3]
    scale = D ** -0.5 if scale is None else scale
    o, lse = torch.zeros(N, Hq, D, dtype=torch.float64), torch.full((N, Hq), -torch.inf, dtype=torch.float64)
    for n, length in enumerate(seq_lens.tolist()):
        first, new = int(cu_seqlens[n]), int(cu_seqlens[n + 1] - cu_seqlens[n])
        if new == 0 or length <= 0:
            continue
        at = torch.arange(length)
        page = page_table[n, at // R].long()
        there = (page >= 0) & (page < P)
        page, row = page.clamp(0, P - 1), at % R
        sees = (at <= (length - new + torch.arange(new))[:, None]) & there  # [new, length]
        for h in range(Hkv):
            k, v = k_pages[page, row, h].double(), v_pages[page, row, h].double()
            k, v = (torch.where(there[:, None], x, 0.0) for x in (k, v))
            heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            s = scale * (q[first:first + new, heads].double() @ k.T)  # [new, group, length]
            s = s.masked_fill(~sees[:, None], -torch.inf)
            top = torch.logsumexp(s, -1)
            lse[first:first + new, heads] = top
            pr = torch.exp(s - top.clamp(min=torch.finfo(torch.float64).min)[..., None])
            o[first:first + new, heads] = pr @ v
    return o, lse
