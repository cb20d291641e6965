"""Attention with 128 rows a workgroup where there are 64 sequences and more: a
tile's sequence is then found by a search over cu_seqlens, not by the sequences'
lengths.  Bars as in test_gpu_paged.py.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import Cache, dev  # noqa: F401  (dev is a fixture)
from test_gpu_paged_rows import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,longest,Hq,Hkv,page", [
    (64, 90, 4, 4, 16),     # whole sequences
    (70, 1500, 4, 4, 16),   # split: fewer tiles than workgroups the card holds
    (70, 1500, 8, 4, 5),    # pages that end inside what a wave stages
    (130, 1300, 8, 4, 16),  # a full card: whole up to 1,024 positions, longer ones split
])
def test_many_sequences_of_many_rows(dev, dtype, S, longest, Hq, Hkv, page):  # noqa: F811
    """Chunks of 0 to 150 rows, some with no past, some of no tokens, and padding."""
    print(f"[gpu] paged attention, {S} sequences of many rows {dtype} up to {longest}", flush=True)
    gen = torch.Generator().manual_seed(S + page)
    new = torch.randint(20, 90, (S,), generator=gen)
    lens = new + torch.randint(0, longest, (S,), generator=gen)
    new[3], new[S // 2], lens[S // 2], lens[7] = 0, 0, 0, new[7]
    lens[11] = new[11] - 5  # more new tokens than positions
    check(Cache(lens.tolist(), new.tolist(), Hq, Hkv, 32, page, dtype, seed=S, tail=70), dev, Hkv)


def test_many_sequences_repeat_alone_and_together(dev):  # noqa: F811
    """A sequence's rows have the same bits whichever others are in the call, as
    long as none is split."""
    print("[gpu] paged attention, many sequences, together and apart", flush=True)
    gen = torch.Generator().manual_seed(41)
    new = torch.randint(33, 90, (66,), generator=gen).tolist()
    c = Cache(new, new, 32, 32, 32, 16, torch.bfloat16, seed=42)
    o, lse = c.attend(dev)
    starts = c.cu.tolist()
    c.table, c.lens, c.cu = c.table[:60], c.lens[:60], c.cu[:61]
    n = starts[60]
    c.q = c.q[:n]
    few, few_lse = c.attend(dev)
    assert torch.equal(few, o[:n]) and torch.equal(few_lse, lse[:n])
