"""Attention over the paged cache with enough rows that 128 of them share a
workgroup's tiles of keys: at least 256 such tiles over the key/value heads,
in the sequences of more than 32 rows (a row: a token's query head of one
key/value head).  Shorter sequences of the same calls run with their keys over
the waves.  Bars as in test_gpu_paged.py.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import rel_l2
from oracle import paged_oracle as oracle
from test_gpu_paged import TOL, Cache, dev  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


def tiles(c, Hkv):
    """The 128-row tiles that the host counts, over the heads."""
    group = c.q.shape[1] // Hkv
    return (c.q.shape[0] * group // 128 + len(c.lens) + 1) * Hkv


def check(c, dev, Hkv, **kw):
    assert tiles(c, Hkv) >= 256
    o, lse = c.attend(dev, **kw)
    ro, rl = oracle.attention_of_sequences(c.q, c.k_pages, c.v_pages, c.table, c.lens, c.cu, **kw)
    assert torch.isfinite(o).all()
    empty = torch.isneginf(rl)
    assert torch.equal(torch.isneginf(lse.cpu()), empty) and (o.cpu()[empty] == 0).all()
    err = rel_l2(o.float(), ro)
    gap = float(((lse.cpu().double() - rl).abs() / (1 + rl.abs()))[~empty].max())
    print(f"  o {err:.2e} lse {gap:.2e}", flush=True)
    assert err < TOL[c.dtype] and gap < 1e-5
    return o, lse


# single tokens, short and long chunks, sequences without and with a past, a page's and a tile's edges
MIXED = ([300, 0, 1, 77, 33, 64, 129, 130, 256, 40], [1, 0, 1, 5, 33, 64, 129, 100, 128, 40])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(32, 32, 128, 16), (32, 32, 128, 1), (64, 32, 64, 24), (96, 32, 32, 8),
                                           (32, 32, 64, 3), (160, 32, 64, 128), (64, 64, 32, 5)])
def test_chunks_of_many_rows(dev, dtype, Hq, Hkv, D, page):  # noqa: F811
    """Pages that hold what a wave stages at a time whole, and pages that do not."""
    print(f"[gpu] paged attention, many rows {dtype} {Hq}/{Hkv} x {D}, pages of {page}", flush=True)
    check(Cache(*MIXED, Hq, Hkv, D, page, dtype, seed=D + page), dev, Hkv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,new,Hq,Hkv,page", [
    ([2600], [780], 32, 32, 16),  # 256 tiles: two splits
    ([1900, 2000, 900], [1, 250, 49], 64, 64, 24),  # under 128 rows a sequence: more splits, single tokens too
    ([1300, 50, 2100, 0], [20, 50, 300, 0], 128, 64, 16)])
def test_split_chunks_of_many_rows(dev, dtype, lens, new, Hq, Hkv, page):  # noqa: F811
    print(f"[gpu] paged attention, many rows, split {dtype} {lens} {Hq}/{Hkv}", flush=True)
    check(Cache(lens, new, Hq, Hkv, 32, page, dtype, seed=page), dev, Hkv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 5])
def test_many_rows_without_keys(dev, dtype, page):  # noqa: F811
    """Padding, more new tokens than positions, holes at a tile's start, end and all through."""
    print(f"[gpu] paged attention, many rows without keys {dtype} pages of {page}", flush=True)
    c = Cache([40, 200, 150], [140, 200, 90], 64, 64, 64, page, dtype, seed=21, tail=70)
    check(c, dev, 64)
    c.table[1, 0], c.table[1, 64 // page], c.table[1, 199 // page] = -1, c.pages, 2 ** 31 - 1
    check(c, dev, 64)
    c.table[2] = -1
    check(c, dev, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_later_tokens_of_many_rows(dev, dtype, bad):  # noqa: F811
    """A later token's key and value, whatever they are, change no earlier token."""
    print(f"[gpu] paged attention, many rows, later tokens {dtype} {bad}", flush=True)
    for Hq, Hkv, page in ((128, 128, 16), (128, 64, 3)):
        c = Cache([200, 40], [150, 40], Hq, Hkv, 32, page, dtype, seed=22)
        assert tiles(c, Hkv) >= 256
        clean, lse0 = c.attend(dev)
        for back in (1, 30, 100):
            at, first = 200 - back, 150 - back
            where = int(c.table[0, at // page]), at % page, 1
            kept = c.k_pages[where].clone(), c.v_pages[where].clone()
            c.k_pages[where][7] = c.v_pages[where][5] = bad
            o, _ = c.attend(dev)
            g = Hq // Hkv
            rest = [h for h in range(Hq) if not g <= h < 2 * g]
            assert torch.equal(o[:first], clean[:first]) and torch.equal(o[150:], clean[150:])
            assert torch.equal(o[:, rest], clean[:, rest])
            if math.isnan(bad):
                assert torch.isnan(o[first:150, g:2 * g]).all()
            # the value alone: its channel only, and lse as it was
            c.k_pages[where] = kept[0]
            o, lse = c.attend(dev)
            assert torch.equal(lse, lse0)
            hit = o[first:150, g:2 * g, 5]
            assert (torch.isnan(hit) if math.isnan(bad) else hit == bad).all()
            o[first:150, g:2 * g, 5] = clean[first:150, g:2 * g, 5]
            assert torch.equal(o, clean)
            c.v_pages[where] = kept[1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scales_of_many_rows(dev, dtype):  # noqa: F811
    """Scores past exp's range, a negative scale, equal scores."""
    print(f"[gpu] paged attention, many rows, scales {dtype}", flush=True)
    c = Cache([300, 65], [150, 65], 64, 64, 64, 16, dtype, seed=23)
    check(c, dev, 64, scale=4.0)
    check(c, dev, 64, scale=-0.2)
    c.q.zero_()
    check(c, dev, 64)


def test_many_rows_repeat(dev):  # noqa: F811
    """The same bits again, also where keys are split."""
    print("[gpu] paged attention, many rows, repeats", flush=True)
    for lens, new, Hq, Hkv in ((*MIXED, 64, 32), ([1900, 2000, 900], [1, 250, 49], 64, 64)):
        c = Cache(lens, new, Hq, Hkv, 32, 16, torch.bfloat16, seed=24)
        first = c.attend(dev)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, c.attend(dev)))
