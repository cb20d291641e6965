"""Sampling on the GPU against the 64-bit oracle: tokens are equal, logprobs
within FP32's 1e-5 (1 + |logprob|)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import sample_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


def gumbel(*shape, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.empty(*shape).exponential_(generator=gen).log_().neg_()


def check(dev, logits, noise, settings):
    """One call whose rows have their own settings; every row against the oracle."""
    from delta_feedback_experiment_amd import sample_tokens

    rows = logits.shape[0]
    cols = [[s.get(n, off) for s in settings] for n, off in
            (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))]
    t, k, p, m = (torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32) for i, c in enumerate(cols))
    token, logprob = sample_tokens(logits.to(dev), noise.to(dev), temperature=t.to(dev), top_k=k.to(dev),
                                   top_p=p.to(dev), min_p=m.to(dev))
    torch.cuda.synchronize()
    for r in range(rows):
        want, lp = oracle.sample_reference(logits[r], noise[r], float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        assert int(token[r]) == want, (r, settings[r], int(token[r]), want)
        got = float(logprob[r])
        assert got == lp or abs(got - lp) <= 1e-5 * (1 + abs(lp)), (r, got, lp)
    return token


SETTINGS = [
    {}, {"temperature": 0.0}, {"temperature": -1.0}, {"temperature": 0.3}, {"temperature": 5.0},
    {"top_k": 1}, {"top_k": 2}, {"top_k": 50}, {"top_k": 1000}, {"top_k": 10 ** 9}, {"top_k": -3},
    {"top_p": 0.9}, {"top_p": 0.5}, {"top_p": 0.999}, {"top_p": 1e-6}, {"top_p": 0.0}, {"top_p": 2.0},
    {"min_p": 0.1}, {"min_p": 1.0}, {"min_p": 1e-4},
    {"top_k": 40, "top_p": 0.9}, {"top_k": 40, "min_p": 0.05}, {"top_p": 0.95, "min_p": 0.02},
    {"temperature": 0.7, "top_k": 100, "top_p": 0.8, "min_p": 0.01}, {"temperature": 1.5, "top_k": 3, "top_p": 0.99},
    {"temperature": 2.0, "top_p": 0.97}, {"temperature": 1e-3, "top_p": 0.9},
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 5003, 50304, 131072])
def test_every_setting(dev, dtype, vocab):
    print(f"[gpu] sample {dtype} {vocab}", flush=True)
    gen = torch.Generator().manual_seed(vocab)
    logits = (3 * torch.randn(len(SETTINGS), vocab, generator=gen)).to(dtype)
    check(dev, logits, gumbel(*logits.shape, seed=vocab), SETTINGS)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.0, 1e-3, 0.3, 30.0])
def test_flat_and_peaked_rows(dev, dtype, scale):
    """All logits equal (0), nearly so, and rows one token wins: the cut falls
    among thousands of ties, or after the first token."""
    print(f"[gpu] sample {dtype} spread {scale}", flush=True)
    gen = torch.Generator().manual_seed(1)
    logits = (scale * torch.randn(len(SETTINGS), 20011, generator=gen)).to(dtype)
    check(dev, logits, gumbel(*logits.shape, seed=2), SETTINGS)


def test_ties_go_to_the_lowest_index(dev):
    """A few values only, and a noise that ties too."""
    print("[gpu] sample ties", flush=True)
    gen = torch.Generator().manual_seed(3)
    logits = torch.randint(-3, 4, (len(SETTINGS), 9001), generator=gen).float() * 0.5
    noise = torch.randint(-1, 2, logits.shape, generator=gen).float()
    check(dev, logits, noise, SETTINGS)
    check(dev, logits.bfloat16(), torch.zeros_like(noise), SETTINGS)
    zeros = torch.zeros(len(SETTINGS), 40)
    zeros[:, ::2] = -0.0  # one value
    check(dev, zeros, torch.zeros_like(zeros), SETTINGS)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_logits(dev, dtype):
    """-inf, NaN and the type's lowest value among the logits; rows of nothing else."""
    print(f"[gpu] sample masks {dtype}", flush=True)
    gen = torch.Generator().manual_seed(4)
    n = len(SETTINGS)
    logits = 2 * torch.randn(n, 3001, generator=gen)
    logits[:, ::3] = -math.inf
    logits[:, 1::7] = math.nan
    check(dev, logits.to(dtype), gumbel(n, 3001, seed=5), SETTINGS)
    lowest = float(torch.finfo(dtype).min)
    logits = torch.full((n, 700), lowest)
    check(dev, logits.to(dtype), gumbel(n, 700, seed=6), SETTINGS)
    logits[:, 333] = 1.0
    check(dev, logits.to(dtype), gumbel(n, 700, seed=7), SETTINGS)
    for bad in (-math.inf, math.nan):
        logits = torch.full((n, 700), bad)
        token = check(dev, logits.to(dtype), gumbel(n, 700, seed=8), SETTINGS)
        assert (token == -1).all()
        logits[:, 699] = lowest
        token = check(dev, logits.to(dtype), gumbel(n, 700, seed=8), SETTINGS)
        assert (token == 699).all()


def test_infinite_logits_and_noise(dev):
    """+inf counts as the largest finite number; noise of -inf or NaN does not win."""
    from delta_feedback_experiment_amd import sample_tokens

    print("[gpu] sample infinities", flush=True)
    logits = torch.randn(len(SETTINGS), 500)
    logits[:, [7, 400]] = math.inf
    check(dev, logits, gumbel(len(SETTINGS), 500, seed=9), SETTINGS)
    logits = torch.randn(2, 500)
    noise = torch.full((2, 500), -math.inf)
    noise[1] = math.nan
    token, _ = sample_tokens(logits.to(dev), noise.to(dev))
    assert torch.equal(token.cpu().long(), logits.argmax(-1))  # nothing else to go by
    noise[:, 123] = -50.0
    token, _ = sample_tokens(logits.to(dev), noise.to(dev))
    assert (token.cpu() == 123).all()


def test_numbers_strides_and_repeats(dev):
    """Settings as numbers, rows of a wider tensor, every other column, a
    transposed one, another stream, a graph: the same tokens."""
    from delta_feedback_experiment_amd import sample_tokens

    print("[gpu] sample strides", flush=True)
    gen = torch.Generator(device=dev).manual_seed(10)
    R, V = 9, 4099
    logits = 2 * torch.randn(R, V, generator=gen, device=dev)
    noise = gumbel(R, V, seed=11).to(dev)
    put = dict(temperature=0.8, top_k=50, top_p=0.9, min_p=0.01)
    want, lp = sample_tokens(logits, noise, **put)
    as_rows = {n: torch.full((R,), x, dtype=torch.int32 if n == "top_k" else torch.float32, device=dev)
               for n, x in put.items()}
    got, lp2 = sample_tokens(logits, noise, **as_rows)
    assert torch.equal(got, want) and torch.equal(lp, lp2)
    wide = torch.randn(R, V + 13, device=dev)
    wide[:, 5:5 + V] = logits
    apart = torch.randn(R, V, 2, device=dev)
    apart[..., 1] = logits
    turned = logits.t().contiguous().t()
    for x in (wide[:, 5:5 + V], apart[..., 1], turned):
        got, lp2 = sample_tokens(x, noise, **put)
        assert torch.equal(got, want) and torch.equal(lp, lp2)
    one = logits[:1].expand(R, V)  # rows that are one row
    got, _ = sample_tokens(one, noise, **put)
    assert torch.equal(got, sample_tokens(one.contiguous(), noise, **put)[0])
    half = logits.bfloat16()
    odd = torch.empty(R * V + 1, dtype=torch.bfloat16, device=dev)[1:].view(R, V)
    odd.copy_(half)
    assert torch.equal(sample_tokens(odd, noise, **put)[0], sample_tokens(half, noise, **put)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = sample_tokens(logits, noise, **put)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(logits, noise, **put)
    for _ in range(4):
        logits.normal_(generator=gen)
        eager = [t.clone() for t in sample_tokens(logits, noise, **put)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_no_rows(dev):
    from delta_feedback_experiment_amd import sample_tokens

    token, logprob = sample_tokens(torch.zeros(0, 7, device=dev), torch.zeros(0, 7, device=dev))
    assert token.shape == logprob.shape == (0,)


def test_draws_follow_the_distribution(dev):
    """Frequencies over 200,000 draws of one row: each within 5 standard
    deviations of its probability (20 tokens: 1e-5 that a right kernel fails)."""
    from delta_feedback_experiment_amd import sample_tokens

    print("[gpu] sample distribution", flush=True)
    n, V = 200_000, 20
    gen = torch.Generator(device=dev).manual_seed(12)
    row = torch.randn(V, generator=gen, device=dev)
    noise = torch.empty(n, V, device=dev).exponential_(generator=gen).log_().neg_()
    token, _ = sample_tokens(row.expand(n, V), noise, temperature=0.9, top_k=12)
    kept, z = oracle.kept_tokens(row.cpu(), float(torch.tensor(0.9)), 12)
    p = torch.zeros(V, dtype=torch.float64)
    p[kept] = torch.softmax(z, 0)
    freq = torch.bincount(token.long().cpu(), minlength=V).double() / n
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lists_in_any_order(dev, dtype):
    """Prefixes of a few thousand near-equal tokens, which a list holds in
    whatever order it was filled: the same token every time, the oracle's."""
    from delta_feedback_experiment_amd import sample_tokens

    print(f"[gpu] sample, lists {dtype}", flush=True)
    gen = torch.Generator().manual_seed(15)
    logits = (0.05 * torch.randn(48, 20011, generator=gen)).to(dtype)
    logits[:, :4000] += 4
    noise = gumbel(48, 20011, seed=16)
    settings = [{"top_p": 0.05 + 0.9 * r / 48, "temperature": 0.5 + r % 3} for r in range(48)]
    want = check(dev, logits, noise, settings)
    t, p = (torch.tensor([s[n] for s in settings], device=dev) for n in ("temperature", "top_p"))
    x, g = logits.to(dev), noise.to(dev)
    for _ in range(10):
        assert torch.equal(sample_tokens(x, g, temperature=t, top_p=p)[0], want)
