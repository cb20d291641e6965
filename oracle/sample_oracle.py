"""One token of a row of logits with temperature, top-k, top-p and min-p, from
given Gumbel numbers: the definition in 64 bits on the CPU."""

from __future__ import annotations

import math

import torch
from torch import Tensor


def kept_tokens(logits: Tensor, temperature: float, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0):
    """The tokens (in order) that a row's settings leave, and their z."""
    l = logits.double()
    usable = ~(torch.isnan(l) | (l == -math.inf))
    index = usable.nonzero()[:, 0]
    if not len(index):
        return index, l[index]
    x = l[index].clamp(max=float(torch.finfo(torch.float32).max))
    order = torch.sort(x, descending=True, stable=True).indices
    index, x = index[order], x[order]
    if temperature <= 0:
        return index[:1], torch.zeros(1, dtype=torch.float64)
    z = (x - x[0]) / temperature
    w = z.exp()
    n = min(top_k, len(w)) if top_k > 0 else len(w)
    if top_p < 1:
        before = torch.cat((torch.zeros(1, dtype=torch.float64), w[:n].cumsum(0)[:-1]))
        n = max(1, int((before < top_p * w[:n].sum()).sum()))
    keep = torch.arange(len(w)) < n
    keep &= w >= min_p
    keep[0] = True
    return index[keep], z[keep]


def sample_reference(logits: Tensor, noise: Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``(token, logprob)`` of one row."""
    index, z = kept_tokens(logits, temperature, top_k, top_p, min_p)
    if not len(index):
        return -1, -math.inf
    score = z + noise.double()[index]
    token = int(index[score == score.max()].min())
    l = torch.nan_to_num(logits.double(), nan=-math.inf, posinf=float(torch.finfo(torch.float32).max), neginf=-math.inf)
    return token, float(l[token] - l.max() - torch.exp(l - l.max()).sum().log())
