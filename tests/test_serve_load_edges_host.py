"""What the loaded server's operators promise at their edges, without a device."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import verify_oracle


def test_oracle_takes_the_target_where_there_is_no_draft():
    """Nothing was drawn from q in a row without a draft: the next token is p's."""
    even, first = torch.zeros(2, 2), torch.tensor([[9.0, -torch.inf]] * 2)
    noise, cu = torch.tensor([[0.5, 0.5]]), torch.tensor([0, 2])
    for none in (-1, 2, 2 ** 31 - 1):
        drafts = torch.tensor([none, 0], dtype=torch.int32)
        args = (even, drafts, torch.zeros(2), noise, cu, first)
        verify_oracle.check(torch.tensor([0, -1], dtype=torch.int32), torch.tensor([0]), *args)
        with pytest.raises(AssertionError):
            verify_oracle.check(torch.tensor([1, -1], dtype=torch.int32), torch.tensor([0]),
                                even, drafts, torch.zeros(2), noise + torch.tensor([[1.0, 0.0]]), cu, first)


@pytest.mark.parametrize("seqs,tokens", [(61, 4156), (251, 8442), (2, 5000), (16, 8192)])
def test_groups_are_shared_whatever_the_mean(seqs, tokens):
    """One long chunk among sequences that decode does not turn the sharing off: a
    shared part and one of its own of every row, by the sizes alone."""
    from delta_feedback_experiment_amd import _lib

    args = _lib.PagedPrefixArgs(dtype=1, num_seqs=seqs, num_tokens=tokens, q_heads=32, kv_heads=8, head_dim=128,
                                page_size=64, max_pages=400, num_pages=9, num_groups=1, cu_seqlens=16)
    args.struct_size = ctypes.sizeof(args)
    assert _lib.lib().pkda_paged_prefix_workspace(ctypes.byref(args)) >= 2 * tokens * 32 * 130
