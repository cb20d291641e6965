"""The serving operators without a device: C ABI, refusals, fake tensors, and
the paged oracle against textbook attention."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from conftest import ROOT
from oracle import paged_oracle, sample_oracle

HEADER = ROOT / "include" / "serve" / "pkda_serve_gfx950.h"


def test_library_exports_the_serving_entry_points():
    from delta_feedback_experiment_amd import _lib

    handle = _lib.lib()  # checks both ABI versions and every struct size
    names = set(re.findall(r"^\w[\w\s\*]*?\b(pkda_\w+)\s*\(", HEADER.read_text(), re.M))
    assert {"pkda_paged_append", "pkda_paged_attention", "pkda_sample"} <= names
    for name in names:
        assert hasattr(handle, name), name
    for kind, struct in _lib._SERVE_ARG_KINDS.items():
        assert handle.pkda_serve_args_size(kind) == ctypes.sizeof(struct)


def _paged(cls, **kw):
    base = dict(dtype=1, num_seqs=2, num_tokens=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16, max_pages=3,
                num_pages=5, table_stride=3, seq_lens=16, page_table=32, q=48, k_pages=64, v_pages=80, q_stride=256,
                k_page_stride=2048, v_page_stride=2048)
    return cls(**{**base, **kw})


@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=48), "head_dim 48"), (dict(dtype=3), "dtype 3"), (dict(page_size=0), "page_size"),
    (dict(page_size=2 ** 20, max_pages=2 ** 12), "page_size"), (dict(num_tokens=3), "cu_seqlens"),
    (dict(k_pages=72), "aligned"), (dict(k_page_stride=2052), "aligned"), (dict(seq_lens=None), "seq_lens"),
    (dict(kv_heads=0), "kv_heads"), (dict(page_table=None), "page_table"), (dict(num_seqs=-1), "num_seqs"),
])
def test_entry_points_refuse_before_any_launch(kw, match):
    """Every refusal comes before a HIP call; the pointers are stand-ins and never read."""
    from delta_feedback_experiment_amd import _lib

    for cls, name, more in ((_lib.PagedAppendArgs, "pkda_paged_append",
                             dict(k=96, v=112, k_stride=128, v_stride=128, q_out=128)),
                            (_lib.PagedAttentionArgs, "pkda_paged_attention", dict(o=96, lse=112))):
        with pytest.raises(ValueError, match=match):
            _lib.call(name, _paged(cls, **more, **kw), 0)


def test_more_refusals_before_any_launch():
    from delta_feedback_experiment_amd import _lib

    with pytest.raises(ValueError, match="q_heads 5"):
        _lib.call("pkda_paged_attention", _paged(_lib.PagedAttentionArgs, q_heads=5, o=96, lse=112), 0)
    append = dict(k=96, v=112, k_stride=128, v_stride=128, q_out=128)
    for kw, match in ((dict(cos=16), "cos"), (dict(cos=16, sin=32, rotary_dim=24), "rotary_dim"),
                      (dict(cos=16, sin=32, rotary_dim=80), "rotary_dim"),
                      (dict(cos=16, sin=32, rotary_dim=64, rope_rows=47), "positions"), (dict(q_stride=250), "aligned")):
        with pytest.raises(ValueError, match=match):
            _lib.call("pkda_paged_append", _paged(_lib.PagedAppendArgs, **{**append, **kw}), 0)
    for kw, match in ((dict(vocab=0), "vocab"), (dict(vocab=2 ** 25), "vocab"), (dict(dtype=5), "dtype"),
                      (dict(logits=None), "null"), (dict(rows=-1), "rows")):
        args = _lib.SampleArgs(**{**dict(dtype=0, rows=2, vocab=9, logits=16, noise=16, token=16, logprob=16), **kw})
        with pytest.raises(ValueError, match=match):
            _lib.call("pkda_sample", args, 0)


@pytest.mark.parametrize("kw,match", [
    (dict(page_size=2 ** 20, max_pages=2 ** 10 + 1), "page_size"), (dict(page_size=2 ** 31 - 1, max_pages=1), "page_size"),
    (dict(num_tokens=2 ** 29 + 1, cu_seqlens=16), "tokens of")])
def test_positions_and_rows_stay_clear_of_32_bits(kw, match):
    """The kernels add up to a tile to a position or a row: none may wrap."""
    from delta_feedback_experiment_amd import _lib

    with pytest.raises(ValueError, match=match):
        _lib.call("pkda_paged_attention", _paged(_lib.PagedAttentionArgs, o=96, lse=112, **kw), 0)


def test_operators_refuse_cpu_tensors():
    from delta_feedback_experiment_amd import paged_append_, paged_attention, sample_tokens

    kv, pages = torch.zeros(2, 2, 64), torch.zeros(3, 16, 2, 64)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_append_(kv, kv, pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention(kv, pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        sample_tokens(torch.zeros(2, 5), torch.zeros(2, 5))


def _case(**kw):
    z = dict(q=torch.zeros(4, 4, 64), k=torch.zeros(4, 2, 64), v=torch.zeros(4, 2, 64),
             k_pages=torch.zeros(3, 16, 2, 64), v_pages=torch.zeros(3, 16, 2, 64),
             page_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32),
             cu_seqlens=torch.tensor([0, 2, 4], dtype=torch.int32), cos=None, sin=None)
    return {**z, **kw}


BAD = [
    (dict(k_pages=torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)), "dtype"),
    (dict(v_pages=torch.zeros(3, 8, 2, 64)), "one"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int64)), "seq_lens"),
    (dict(page_table=torch.zeros(3, 3, dtype=torch.int32)), "page_table"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), "cu_seqlens"),
    (dict(cu_seqlens=None), "cu_seqlens"),
    (dict(k_pages=torch.zeros(3, 2, 16, 64).transpose(1, 2), v_pages=torch.zeros(3, 2, 16, 64).transpose(1, 2)),
     "dense"),
    (dict(k_pages=torch.zeros(3, 16, 2, 48), v_pages=torch.zeros(3, 16, 2, 48)), "head_dim"),
]
BAD_APPEND = [
    (dict(v=torch.zeros(4, 3, 64)), "match"), (dict(k=torch.zeros(4, 1, 64), v=torch.zeros(4, 1, 64)), "match"),
    (dict(q=torch.zeros(3, 4, 64)), "match"), (dict(cos=torch.zeros(48, 32)), "together"),
    (dict(cos=torch.zeros(47, 32), sin=torch.zeros(47, 32)), "positions"),
    (dict(cos=torch.zeros(48, 12), sin=torch.zeros(48, 12)), "rotary"),
    (dict(cos=torch.zeros(48, 40), sin=torch.zeros(48, 40)), "rotary"),
    (dict(cos=torch.zeros(48, 32).double(), sin=torch.zeros(48, 32).double()), "float32"),
]


def _fake(kw):
    """The tensors as fake ones of a HIP device, keeping their strides."""
    mode = FakeTensorMode()
    with mode:
        return {n: None if t is None else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
                for n, t in kw.items()}, mode


def _append(x):
    from delta_feedback_experiment_amd import paged_append_

    return paged_append_(x["k"], x["v"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"],
                         cu_seqlens=x["cu_seqlens"], q=x["q"], cos=x["cos"], sin=x["sin"])


def _attention(x):
    from delta_feedback_experiment_amd import paged_attention

    return paged_attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"],
                           cu_seqlens=x["cu_seqlens"])


@pytest.mark.parametrize("kw,match", BAD + BAD_APPEND)
def test_append_checks_its_arguments(kw, match):
    x, mode = _fake(_case(**kw))
    with mode, pytest.raises(ValueError, match=match):
        _append(x)


@pytest.mark.parametrize("kw,match", BAD + [(dict(q=torch.zeros(4, 5, 64)), "share"),
                                            (dict(q=torch.zeros(4, 256)), "head_dim")])
def test_attention_checks_its_arguments(kw, match):
    x, mode = _fake(_case(**kw))
    with mode, pytest.raises(ValueError, match=match):
        _attention(x)


def test_sample_checks_its_arguments():
    from delta_feedback_experiment_amd import sample_tokens

    with FakeTensorMode():
        l, n = (torch.empty(3, 10, device="cuda") for _ in range(2))
        for args, kw, match in (
                ((l, n[:, :9]), {}, "noise"), ((l[0], n[0]), {}, "rows"), ((l.double(), n), {}, "float32"),
                ((l, n.bfloat16()), {}, "float32"), ((l, n), dict(top_k=torch.zeros(3, device="cuda")), "top_k"),
                ((l, n), dict(temperature=torch.zeros(2, device="cuda")), "temperature"),
                ((l[:, :0], n[:, :0]), {}, "vocab")):
            with pytest.raises(ValueError, match=match):
                sample_tokens(*args, **kw)


def test_shapes_of_fake_tensors():
    from delta_feedback_experiment_amd import sample_tokens

    x, mode = _fake(_case(cos=torch.zeros(48, 32), sin=torch.zeros(48, 32)))
    with mode:
        q = _append(x)
        assert q.shape == x["q"].shape and q.dtype == x["q"].dtype
        o, lse = _attention(x)
        assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (4, 4) and lse.dtype == torch.float32
        token, logprob = sample_tokens(torch.empty(3, 10, device="cuda", dtype=torch.bfloat16),
                                       torch.empty(3, 10, device="cuda"), top_k=5, top_p=0.9)
        assert token.shape == logprob.shape == (3,) and token.dtype == torch.int32


def test_host_check_of_a_cache():
    from delta_feedback_experiment_amd.paged import validate_pages

    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ok = dict(num_tokens=5, num_pages=4, page_size=4, appended=True)
    validate_pages(table, i32(7, 3), i32(0, 2, 5), **ok)
    for tab, lens, cu, kind in ((table, i32(9, 3), i32(0, 2, 5), ValueError), (table, i32(1, 3), i32(0, 2, 5), ValueError),
                                (table, i32(7, 3), i32(0, 4, 2), ValueError), (table, i32(7, 3), i32(1, 2, 5), ValueError),
                                (table + 1, i32(7, 8), i32(0, 2, 5), IndexError), (table - 1, i32(7, 3), i32(0, 2, 5), IndexError),
                                (torch.tensor([[0, 1], [0, 1]]).int(), i32(3, 3), i32(0, 2, 5), ValueError)):
        with pytest.raises(kind):
            validate_pages(tab, lens, cu, **ok)
    # a shared prefix is read by both
    validate_pages(torch.tensor([[0, 1], [0, 1]]).int(), i32(3, 3), i32(0, 2, 5), **{**ok, "appended": False})


def test_paged_oracle_is_causal_attention():
    gen = torch.Generator().manual_seed(0)
    L, Hq, Hkv, D, page = 13, 4, 2, 32, 4
    q, k, v = (torch.randn(L, h, D, generator=gen) for h in (Hq, Hkv, Hkv))
    table = torch.tensor([[3, 0, 2, 1]], dtype=torch.int32)
    pages = torch.zeros(4, page, Hkv, D)
    lens, cu = torch.tensor([L], dtype=torch.int32), torch.tensor([0, L], dtype=torch.int32)
    _, kp, vp = paged_oracle.append_reference(k, v, pages, pages, table, lens, cu)
    o, lse = paged_oracle.attention_reference(q, kp, vp, table, lens, cu)
    kk, vv = (t.double().repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q.double(), kk) * D ** -0.5
    s = s.masked_fill(torch.ones(L, L).triu(1).bool(), -torch.inf)
    assert torch.allclose(o, torch.einsum("hij,jhd->ihd", s.softmax(-1), vv), atol=1e-12)
    assert torch.allclose(lse, s.logsumexp(-1).t(), atol=1e-12)


def test_paged_oracle_by_sequence_equals_by_token():
    gen = torch.Generator().manual_seed(3)
    lens, new = [7, 0, 12, 5], [3, 0, 12, 9]
    cu = torch.tensor([0, 3, 3, 15, 24], dtype=torch.int32)
    table = torch.randperm(16, generator=gen).int().view(4, 4)
    table[2, 1], table[0, 0] = -1, 99
    q = torch.randn(26, 4, 8, generator=gen)
    k, v = (torch.randn(16, 4, 2, 8, generator=gen) for _ in range(2))
    args = (q, k, v, table, torch.tensor(lens, dtype=torch.int32), cu, 0.7)
    for a, b in zip(paged_oracle.attention_reference(*args), paged_oracle.attention_of_sequences(*args)):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)



def test_sample_oracle_settings():
    l = torch.tensor([1.0, 3.0, 2.0, 3.0, 0.0])
    assert sample_oracle.kept_tokens(l, 1.0)[0].tolist() == [1, 3, 2, 0, 4]
    assert sample_oracle.kept_tokens(l, 1.0, top_k=1)[0].tolist() == [1]
    assert sample_oracle.kept_tokens(l, 1.0, top_p=0.5)[0].tolist() == [1, 3]
    assert sample_oracle.kept_tokens(l, 1.0, min_p=0.3)[0].tolist() == [1, 3, 2]
    assert sample_oracle.kept_tokens(l, 0.0)[0].tolist() == [1]
    token, logprob = sample_oracle.sample_reference(l, torch.tensor([0.0, 0.0, 9.0, 0.0, 0.0]))
    assert token == 2 and abs(logprob - float(torch.log_softmax(l, 0)[2])) < 1e-6
