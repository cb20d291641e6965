"""Verification where a row has no draft though draft logits are given, and at
temperatures whose reciprocal is past FP32, on the GPU.

The oracle's bars are those of ``test_gpu_verify.py``; the rest is exact.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_verify import RAGGED, Drafts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_a_draft_the_token_is_the_target_s(dev, dtype):
    """p is even over two tokens and q all on the first: nothing was drawn from q, so
    the noise alone decides, and equal noise takes the lower index."""
    print(f"[gpu] verify, no draft {dtype}", flush=True)
    for none in (-1, 2, 2 ** 31 - 1, -2 ** 31):
        d = Drafts([2] * 3, 2, dtype, seed=1)
        d.logits[:] = 1.0
        d.draft_logits[:, 0], d.draft_logits[:, 1] = 9.0, -math.inf
        d.drafts[:] = none
        d.uniform[:] = 0.0
        d.noise[:] = torch.tensor([[0.5, 0.5], [0.6, 0.5], [0.5, 0.6]])
        tokens, accepted = d.check(dev)
        assert accepted.tolist() == [0] * 3 and tokens[::2].tolist() == [0, 0, 1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [7, 4096, 100001])
def test_rows_without_drafts_among_others(dev, dtype, vocab):
    """A step of fixed shape whose sequences have fewer drafts each: up to the first
    place without one as ever, there what the same rows give without draft logits."""
    print(f"[gpu] verify, fewer drafts {dtype} vocab {vocab}", flush=True)
    d = Drafts(RAGGED, vocab, dtype, seed=vocab, near=0.2)
    d.temperature = 0.8
    first = d.cu[:-1].tolist()
    for n, r in enumerate(RAGGED):
        if r > 1:
            d.drafts[first[n] + (n * 5) % (r - 1):first[n] + r] = -1
    got = d.check(dev)
    d.drafts[:] = -1
    tokens, accepted = d.check(dev)
    assert (accepted == 0).all()
    d.draft_logits = None
    assert torch.equal(d.check(dev)[0], tokens)
    assert got[1].sum() > 0


def test_draws_of_sequences_with_and_without_drafts(dev):
    """The next tokens are distributed as the target where half the sequences have no
    draft: 40,000 sequences, a chi-square over 12 tokens (11 degrees of freedom: over
    40 has probability under 4e-5)."""
    from delta_feedback_experiment_amd import verify_tokens

    gen = torch.Generator(device=dev).manual_seed(20)
    S, V = 40000, 12
    l, ld = (1.5 * torch.randn(V, generator=gen, device=dev) for _ in range(2))
    gumbel = lambda *s: -torch.empty(*s, device=dev).exponential_(generator=gen).log()  # noqa: E731
    drafts = (ld + gumbel(S, V)).argmax(-1).int()
    drafts[::2] = -1
    logits, draft_logits = (t.expand(2 * S, V).contiguous() for t in (l, ld))
    cu = torch.arange(0, 2 * S + 1, 2, dtype=torch.int32, device=dev)
    uniform = torch.rand(2 * S, generator=gen, device=dev)
    tokens, accepted = verify_tokens(logits, drafts.repeat_interleave(2), uniform, gumbel(S, V), cu,
                                     draft_logits=draft_logits)
    assert (accepted[::2] == 0).all()
    for part in (tokens[::4], tokens[2::4]):
        want = torch.softmax(l.double(), 0) * part.numel()
        chi = float(((torch.bincount(part.long(), minlength=V) - want) ** 2 / want).sum())
        print(f"[gpu] verify draws with and without drafts: chi-square {chi:.1f}", flush=True)
        assert chi < 40


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-6, 1e-38, 1e-45])
def test_cold_drafts_stand_where_they_are_the_largest(dev, dtype, temperature):
    """At the smallest temperatures p is 1 at the largest logit: a draft there stands
    whatever the number (q <= 1), any other falls."""
    for draft in (True, False):
        print(f"[gpu] verify, cold {temperature} {dtype} draft logits {draft}", flush=True)
        d = Drafts([3] * 9, 700, dtype, seed=40, draft=draft)
        d.temperature = temperature
        top = d.logits.float().sort(-1)
        d.logits[torch.arange(27), top.indices[:, -1]] += 1  # (BF16 rows may tie at the top)
        best = top.indices[:, -1].int()
        d.drafts = best.clone()
        d.uniform[:] = 1 - 2.0 ** -24
        tokens, accepted = d.check(dev)
        assert (accepted == 2).all() and torch.equal(tokens.cpu(), best)
        wrong = torch.tensor([3 * n + n % 3 for n in range(9)])
        d.drafts[wrong] = (best[wrong] + 1) % 700
        if draft:  # the draft's own largest
            d.draft_logits[wrong, d.drafts[wrong].long()] = 50.0
        tokens, accepted = d.check(dev)
        assert accepted.tolist() == [n % 3 for n in range(9)]
        assert torch.equal(tokens.cpu()[wrong], best[wrong])
