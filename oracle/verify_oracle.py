"""Verification of drafted tokens in 64 bits on the CPU, one row at a time."""

from __future__ import annotations

import torch
from torch import Tensor


def probabilities(logits: Tensor, temperature: float) -> Tensor:
    """softmax(logits / temperature) of one row; zeros where nothing can be taken."""
    x = logits.float().double()
    big = torch.finfo(logits.dtype).max
    x = torch.where(torch.isnan(x), -torch.inf, x).clamp(max=big)
    top = x.max()
    if top == -torch.inf:
        return torch.zeros_like(x)
    z = x - top
    z = torch.where(x == -torch.inf, -torch.inf, z / temperature if temperature < torch.inf else z * 0)
    return torch.softmax(z, 0)


def first_largest(logits: Tensor) -> int:
    x = logits.float()
    x = torch.where(torch.isnan(x), -torch.inf, x).clamp(max=torch.finfo(logits.dtype).max)
    top = x.max()
    return -1 if top == -torch.inf else int((x == top).nonzero()[0])


def check(tokens: Tensor, accepted: Tensor, logits, drafts, uniform, noise, cu, draft_logits=None, temperature=1.0,
          slack: float = 2.0 ** -16) -> int:
    """Assert that the outputs are those of the definition, where a probability may
    be off by ``slack`` of its size; returns how many rows were decided by less."""
    temperature = temperature.tolist() if isinstance(temperature, Tensor) else [temperature] * (len(cu) - 1)
    near, seen = 0, torch.full((logits.shape[0],), -1, dtype=torch.int32)
    for n, t in enumerate(temperature):
        first, end = int(cu[n]), int(cu[n + 1])
        a = int(accepted[n])
        if first == end:
            assert a == 0
            continue
        assert 0 <= a < end - first, (n, a)
        for j in range(a + 1):
            row, last = first + j, first + j == end - 1
            d = int(drafts[row])
            stands = j < a
            if t <= 0:
                best = first_largest(logits[row])
                assert last or stands == (best >= 0 and d == best), (n, j)
                if not stands:
                    assert int(tokens[row]) == best, (n, j)
                else:
                    seen[row] = d
                continue
            p = probabilities(logits[row], t)
            inside = 0 <= d < p.numel()
            if draft_logits is not None:
                q = probabilities(draft_logits[row], t)
            else:
                q = torch.zeros_like(p)
                if inside:
                    q[d] = 1
            if not last:
                u = float(uniform[row])
                lhs, rhs = (u * float(q[d]), float(p[d])) if inside else (1.0, 0.0)
                assert lhs < rhs * (1 + slack) if stands else lhs >= rhs * (1 - slack), (n, j, lhs, rhs, stands)
                near += abs(lhs - rhs) <= slack * rhs
            if stands:
                seen[row] = d
                continue
            token = int(tokens[row])
            # (without a draft nothing was drawn from q)
            rest = p if last or not inside else (p - q).clamp(min=0)
            if not (rest > 0).any():
                rest = p
            if not (rest > 0).any():
                assert token == -1, (n, j, token)
                continue
            score = rest.log() + noise[n].double()
            off = slack * (1 + (p + (0 if last or not inside else q)) / rest.clamp(min=1e-300))
            off = torch.where(rest > 0, off, 0.0)
            assert 0 <= token < p.numel() and rest[token] > 0, (n, j, token)
            assert score[token] + off[token] >= (score - off)[rest > 0].max(), (n, j, token, int(score.argmax()))
            near += int(score.argmax()) != token
        row = first + a
        seen[row] = tokens[row]
    assert torch.equal(tokens.cpu(), seen)
    return near
