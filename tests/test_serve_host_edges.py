"""The serving operators without a device, at their edges."""

from __future__ import annotations

import ctypes
import re

import pytest

from conftest import ROOT

CSRC = ROOT / "delta_feedback_experiment_amd" / "csrc"


def test_lane_reads_are_widened_without_their_sign():
    """The lane reads return int: in a 64-bit mask a word with its top bit set
    would fill the upper word, and name keys past the sequence."""
    found = 0
    for path in sorted((CSRC / "serve").glob("*")):
        for statement in path.read_text().split(";"):
            if "uint64_t" not in statement or "<< 32" not in statement:
                continue
            for m in re.finditer(r"__builtin_amdgcn_read(?:first)?lane\(", statement):
                found += 1
                assert statement[:m.start()].endswith("(uint32_t)"), (path.name, statement.strip())
    assert found


@pytest.mark.parametrize("tokens,seqs,heads,kv_heads,positions", [
    (200, 1, 4, 1, 1024), (300, 1, 8, 2, 2048), (1, 1, 32, 8, 131072), (64, 64, 32, 8, 4096), (5, 5, 64, 64, 4096),
    (320, 64, 32, 4, 4096), (2048, 1, 32, 8, 16384), (500, 500, 96, 32, 65536), (300, 300, 96, 3, 4096)])
def test_workspace_follows_from_the_sizes(tokens, seqs, heads, kv_heads, positions):
    """The same length whether cu_seqlens is there yet or not, and enough for
    the form that takes more."""
    from delta_feedback_experiment_amd import _lib

    handle = _lib.lib()

    def floats(**kw):
        args = _lib.PagedAttentionArgs(dtype=1, num_seqs=seqs, num_tokens=tokens, q_heads=heads, kv_heads=kv_heads,
                                       head_dim=128, page_size=64, max_pages=positions // 64, num_pages=9, **kw)
        args.struct_size = ctypes.sizeof(args)
        return handle.pkda_paged_attention_workspace(ctypes.byref(args))

    assert floats() == floats(cu_seqlens=16) >= 0
    assert floats() % (tokens * heads * 130) == 0  # so many rows' sums and outputs a split
