"""The serving operators without a device, at their edges."""

from __future__ import annotations

import ctypes
import re
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from test_serve_host import _append, _attention, _case, _fake

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


def _meta_case():
    def z(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="meta")

    i32 = dict(dtype=torch.int32)
    return z(4, 4, 64), z(4, 2, 64), z(3, 16, 2, 64), z(2, 3, **i32), z(2, **i32), z(3, **i32), z(48, 32)


def test_meta_tensors_get_their_shapes():
    """On the meta device, as the operators themselves and the decode step take it."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention, sample_tokens

    q, kv, pages, table, lens, cu, angle = _meta_case()
    out = paged_append_(kv, kv, pages, pages, table, lens, cu_seqlens=cu, q=q, cos=angle, sin=angle)
    assert out.is_meta and out.shape == q.shape and out.dtype == q.dtype
    assert paged_append_(kv, kv, pages, pages, table, lens, cu_seqlens=cu) is None
    o, lse = paged_attention(q, pages, pages, table, lens, cu_seqlens=cu)
    assert o.is_meta and o.shape == q.shape and lse.shape == (4, 4) and lse.dtype == torch.float32
    logits = torch.empty(3, 10, dtype=torch.bfloat16, device="meta")
    token, logprob = sample_tokens(logits, logits.float(), top_k=5)
    assert token.is_meta and token.shape == logprob.shape == (3,)
    assert token.dtype == torch.int32 and logprob.dtype == torch.float32
    with pytest.raises(ValueError, match="share"):
        paged_attention(q[:, :3], pages, pages, table, lens, cu_seqlens=cu)


@pytest.mark.parametrize("pages", [torch.zeros(3, 1, 16, 64).transpose(1, 2), torch.zeros(3, 64)[:, None, None],
                                   torch.zeros(1, 3, 64).permute(1, 0, 2)[:, None]])
def test_dense_pages_of_one_head_or_one_row(pages):
    """The stride of an axis of length one says nothing."""
    assert pages.is_contiguous() and pages.shape[2] == 1
    page = pages.shape[1]
    x, mode = _fake(_case(k=torch.zeros(4, 1, 64), v=torch.zeros(4, 1, 64), k_pages=pages, v_pages=pages,
                          page_table=torch.zeros(2, 48 // page, dtype=torch.int32)))
    with mode:
        assert _append(x).shape == x["q"].shape
        assert _attention(x)[0].shape == x["q"].shape


@pytest.mark.parametrize("seqs", [0, 1, 7])
def test_no_tokens_of_some_sequences(seqs):
    """Nothing to do is no error, and no division by the rows a sequence has; in
    a process of its own, which a division by zero would end."""
    code = f"""
import ctypes
from delta_feedback_experiment_amd import _lib
common = dict(dtype=1, num_seqs={seqs}, num_tokens=0, q_heads=4, kv_heads=2, head_dim=64, page_size=16, max_pages=3,
              num_pages=5, table_stride=3, cu_seqlens=16, seq_lens=16, page_table=16, k_pages=16, v_pages=16)
args = _lib.PagedAttentionArgs(**common)
args.struct_size = ctypes.sizeof(args)
assert _lib.lib().pkda_paged_attention_workspace(ctypes.byref(args)) == 0
_lib.call("pkda_paged_attention", args, 0)
_lib.call("pkda_paged_append", _lib.PagedAppendArgs(**common), 0)
print("done")
"""
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "done" in got.stdout, (got.returncode, got.stderr[-500:])
