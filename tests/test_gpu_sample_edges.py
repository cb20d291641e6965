"""Sampling on the GPU at its edges, against the 64-bit oracle: bars as in test_gpu_sample.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_sample import SETTINGS, check, dev, gumbel  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("large", [1e6, 1e9, 6e9, 1e10, 1e11, 1e12, 3e12, 1e30])
def test_large_finite_logits(dev, dtype, large):  # noqa: F811
    """Most of a row, and whole waves of it, masked with a large negative number;
    and rows whose every logit is large, of either sign."""
    print(f"[gpu] sample, logits of {large:g} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(17)
    n, V = len(SETTINGS), 40011
    noise = gumbel(n, V, seed=18)
    logits = torch.full((n, V), -large)
    logits[:, 30000:30300] = 3 * torch.randn(n, 300, generator=gen)
    logits[:, V - 1] = 0.5
    check(dev, logits.to(dtype), noise, SETTINGS)
    for sign in (-1, 1):
        logits = sign * large * (1 + torch.randint(0, 3, (n, 9001), generator=gen) * 2.0 ** -6)
        check(dev, logits.to(dtype), noise[:, :9001].contiguous(), SETTINGS)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5003, 50304])
def test_infinite_noise_ties_at_the_lowest_index(dev, dtype, vocab):  # noqa: F811
    """Noise of +inf at two tokens: of one load, of one thread, of two threads."""
    print(f"[gpu] sample, infinite noise {dtype} {vocab}", flush=True)
    gen = torch.Generator().manual_seed(19)
    logits = torch.randn(len(SETTINGS), vocab, generator=gen).to(dtype)
    for pair in ([8, 9], [8, 11], [8, 8 + 4096], [700, 9]):
        noise = gumbel(len(SETTINGS), vocab, seed=20)
        noise[:, pair] = math.inf
        check(dev, logits, noise, SETTINGS)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [math.inf, 3e38, 1e30])
@pytest.mark.parametrize("vocab", [4099, 50303])
def test_temperatures_without_bound(dev, dtype, temperature, vocab):  # noqa: F811
    """z is 0, or nearly, for every finite logit: a uniform draw over what the
    settings leave.  Rows with -inf, with the type's lowest value, and without."""
    print(f"[gpu] sample, temperature {temperature:g} {dtype} {vocab}", flush=True)
    gen = torch.Generator().manual_seed(21)
    settings = [{**s, "temperature": temperature} for s in SETTINGS]
    for other in (None, -math.inf, float(torch.finfo(dtype).min)):
        logits = 3 * torch.randn(len(settings), vocab, generator=gen)
        if other is not None:
            logits[:, 1::2] = other
        check(dev, logits.to(dtype), gumbel(*logits.shape, seed=22), settings)
