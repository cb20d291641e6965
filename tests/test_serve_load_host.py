"""The operators of a loaded server (8-bit cache, heads' norms, shared prefixes,
verification) without a device: C ABI, refusals, fake and meta tensors, oracles."""

from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from conftest import ROOT
from oracle import paged_fp8_oracle as fp8
from oracle import verify_oracle

CODES, POWERS = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _paged(cls, **kw):
    base = dict(dtype=1, num_seqs=2, num_tokens=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16, max_pages=3,
                num_pages=5, table_stride=3, seq_lens=16, page_table=32, q=48, k_pages=64, v_pages=80, q_stride=256,
                k_page_stride=2048, v_page_stride=2048, k_scales=96, v_scales=112, k_scale_stride=64, v_scale_stride=64)
    return cls(**{**base, **kw})


def _entries():
    from delta_feedback_experiment_amd import _lib

    attend = dict(o=96, lse=112, workspace=128, scale=1.0)
    return (
        (_lib.PagedStoreArgs, "pkda_paged_store", dict(k=96, v=112, k_stride=128, v_stride=128, q_out=128,
                                                       cache_dtype=_lib.PKDA_CACHE_FP8, q_norm=16, k_norm=32)),
        (_lib.PagedAttentionFP8Args, "pkda_paged_attention_fp8", attend),
        (_lib.PagedPrefixArgs, "pkda_paged_prefix_attention", dict(attend, cu_groups=16, prefix_lens=32, num_groups=1)),
    )


@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=48), "head_dim 48"), (dict(head_dim=32), "head_dim 32"), (dict(dtype=3), "dtype 3"),
    (dict(page_size=0), "page_size"), (dict(page_size=2 ** 20, max_pages=2 ** 12), "page_size"),
    (dict(num_tokens=3), "cu_seqlens"), (dict(k_pages=72), "aligned"), (dict(k_page_stride=2056), "aligned"),
    (dict(seq_lens=None), "seq_lens"), (dict(kv_heads=0), "kv_heads"), (dict(page_table=None), "page_table"),
    (dict(num_seqs=-1), "num_seqs"), (dict(k_scales=None), "scales"), (dict(v_scales=113), "scales"),
    (dict(v_scale_stride=63), "scales"), (dict(q_stride=250), "aligned"),
])
def test_entry_points_refuse_before_any_launch(kw, match):
    """Every refusal comes before a HIP call; the pointers are stand-ins and never read."""
    from delta_feedback_experiment_amd import _lib

    for cls, name, more in _entries():
        with pytest.raises(ValueError, match=match):
            _lib.call(name, _paged(cls, **{**more, **kw}), 0)


def test_more_refusals_before_any_launch():
    from delta_feedback_experiment_amd import _lib

    (store, store_name, more), (_, attend_name, attend), (prefix, prefix_name, groups) = _entries()
    for kw, match in ((dict(cos=16), "cos"), (dict(cos=16, sin=32, rotary_dim=24), "rotary_dim"),
                      (dict(cos=16, sin=32, rotary_dim=64, rope_rows=47), "positions"), (dict(cache_dtype=0), "cache_dtype"),
                      (dict(cache_dtype=3), "cache_dtype"), (dict(norm_dtype=2), "norm_dtype"), (dict(q_norm=8), "aligned"),
                      (dict(k=None), "null")):
        with pytest.raises(ValueError, match=match):
            _lib.call(store_name, _paged(store, **{**more, **kw}), 0)
    for kw, match in ((dict(q_heads=5), "q_heads 5"), (dict(o=None), "null"), (dict(scale=float("inf")), "scale"),
                      (dict(num_tokens=2 ** 29 + 1, cu_seqlens=16), "tokens of")):
        for name, cls, base in ((attend_name, _lib.PagedAttentionFP8Args, attend), (prefix_name, prefix, groups)):
            with pytest.raises(ValueError, match=match):
                _lib.call(name, _paged(cls, **{**base, **kw}), 0)
    for kw, match in ((dict(cu_groups=None), "groups"), (dict(prefix_lens=None), "groups"), (dict(num_groups=-1), "num_groups"),
                      (dict(workspace=None), "workspace"), (dict(workspace=24), "workspace")):
        with pytest.raises(ValueError, match=match):
            _lib.call(prefix_name, _paged(prefix, **{**groups, **kw}), 0)
    ok = dict(dtype=0, rows=4, vocab=9, num_seqs=2, logits=16, drafts=16, uniform=16, noise=16, cu_seqlens=16, tokens=16,
              accepted=16, workspace=16)
    for kw, match in ((dict(vocab=0), "vocab"), (dict(vocab=2 ** 24 + 1), "vocab"), (dict(dtype=5), "dtype"),
                      (dict(logits=None), "null"), (dict(rows=-1), "rows"), (dict(num_seqs=-1), "num_seqs"),
                      (dict(cu_seqlens=None), "cu_seqlens"), (dict(accepted=None), "null"), (dict(workspace=None), "workspace"),
                      (dict(logits=18), "aligned"), (dict(draft_logits=17), "aligned")):
        with pytest.raises(ValueError, match=match):
            _lib.call("pkda_verify", _lib.VerifyArgs(**{**ok, **kw}), 0)


@pytest.mark.parametrize("tokens,seqs,groups,heads,kv_heads,positions", [
    (200, 1, 1, 4, 1, 1024), (64, 64, 1, 32, 8, 32768), (96, 96, 6, 16, 4, 4096), (5, 5, 0, 64, 64, 4096),
    (320, 64, 3, 32, 4, 4096), (2048, 8, 2, 32, 8, 16384), (500, 500, 500, 96, 32, 65536), (7, 9, 2, 8, 2, 0)])
def test_workspace_follows_from_the_sizes(tokens, seqs, groups, heads, kv_heads, positions):
    from delta_feedback_experiment_amd import _lib

    handle = _lib.lib()

    def floats(cls, name, **kw):
        args = cls(dtype=1, num_seqs=seqs, num_tokens=tokens, q_heads=heads, kv_heads=kv_heads, head_dim=128, page_size=64,
                   max_pages=positions // 64, num_pages=9, **kw)
        args.struct_size = ctypes.sizeof(args)
        return getattr(handle, name)(ctypes.byref(args))

    row = tokens * heads * 130
    for cls, name, more in ((_lib.PagedAttentionFP8Args, "pkda_paged_attention_fp8_workspace", {}),
                            (_lib.PagedPrefixArgs, "pkda_paged_prefix_workspace", dict(num_groups=groups))):
        some = floats(cls, name, **more)
        assert some == floats(cls, name, cu_seqlens=16, **more) >= 0 and some % row == 0
    # a shared part and one of its own at least, 128 of each at most; but for sequences
    # that fill the card with tiles of their own
    alone = tokens * heads // kv_heads > 128 * seqs and tokens * heads >= 128 * 256
    assert some <= 256 * row and (alone or some >= 2 * row)


@pytest.mark.parametrize("seqs", [0, 1, 7])
def test_no_tokens_of_some_sequences(seqs):
    """Nothing to do is no error, and no division by what there is none of; in a
    process of its own, which a division by zero would end."""
    code = f"""
import ctypes
from delta_feedback_experiment_amd import _lib
common = dict(dtype=1, num_seqs={seqs}, num_tokens=0, q_heads=4, kv_heads=2, head_dim=64, page_size=16, max_pages=3,
              num_pages=5, table_stride=3, cu_seqlens=16, seq_lens=16, page_table=16, k_pages=16, v_pages=16,
              k_scales=16, v_scales=16)
for cls, name, sizes, more in (
        (_lib.PagedStoreArgs, "pkda_paged_store", None, dict(cache_dtype=2)),
        (_lib.PagedAttentionFP8Args, "pkda_paged_attention_fp8", "pkda_paged_attention_fp8_workspace", {{}}),
        (_lib.PagedPrefixArgs, "pkda_paged_prefix_attention", "pkda_paged_prefix_workspace", {{}}),
        (_lib.PagedPrefixArgs, "pkda_paged_prefix_attention", "pkda_paged_prefix_workspace",
         dict(num_groups={seqs}, cu_groups=16, prefix_lens=16))):
    args = cls(**common, **more)
    args.struct_size = ctypes.sizeof(args)
    assert sizes is None or getattr(_lib.lib(), sizes)(ctypes.byref(args)) == 0
    _lib.call(name, args, 0)
args = _lib.VerifyArgs(vocab=5, cu_seqlens=16)
args.struct_size = ctypes.sizeof(args)
assert _lib.lib().pkda_verify_workspace(ctypes.byref(args)) == 0
_lib.call("pkda_verify", args, 0)
print("done")
"""
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "done" in got.stdout, (got.returncode, got.stderr[-500:])


def _codes(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(CODES)


def _powers(*shape):
    return torch.full(shape, 127, dtype=torch.uint8).view(POWERS)


def _case(**kw):
    z = dict(q=torch.zeros(4, 4, 64), k=torch.zeros(4, 2, 64), v=torch.zeros(4, 2, 64), k_pages=_codes(3, 16, 2, 64),
             v_pages=_codes(3, 16, 2, 64), k_scales=_powers(3, 16, 2, 2), v_scales=_powers(3, 16, 2, 2),
             page_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32),
             cu_seqlens=torch.tensor([0, 2, 4], dtype=torch.int32), cos=None, sin=None, q_norm=None, k_norm=None,
             cu_groups=torch.tensor([0, 2], dtype=torch.int32), prefix_lens=torch.zeros(1, dtype=torch.int32))
    return {**z, **kw}


def _on(device, kw):
    return {n: None if t is None else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device)
            for n, t in kw.items()}


def _append(x):
    from delta_feedback_experiment_amd import paged_append_fp8_

    return paged_append_fp8_(x["k"], x["v"], x["k_pages"], x["v_pages"], x["k_scales"], x["v_scales"], x["page_table"],
                             x["seq_lens"], cu_seqlens=x["cu_seqlens"], q=x["q"], cos=x["cos"], sin=x["sin"],
                             q_norm=x["q_norm"], k_norm=x["k_norm"])


def _attend(x):
    from delta_feedback_experiment_amd import paged_attention_fp8

    return paged_attention_fp8(x["q"], x["k_pages"], x["v_pages"], x["k_scales"], x["v_scales"], x["page_table"],
                               x["seq_lens"], cu_seqlens=x["cu_seqlens"])


def _prefix(x):
    from delta_feedback_experiment_amd import paged_prefix_attention

    return paged_prefix_attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["cu_groups"],
                                  x["prefix_lens"], k_scales=x["k_scales"], v_scales=x["v_scales"],
                                  cu_seqlens=x["cu_seqlens"])


BAD = [
    (dict(k_pages=torch.zeros(3, 16, 2, 64)), "float8_e4m3fn"),
    (dict(v_pages=_codes(3, 8, 2, 64)), "one"),
    (dict(k_scales=_powers(3, 16, 2, 4)), "scales"), (dict(v_scales=torch.zeros(3, 16, 2, 2)), "scales"),
    (dict(k_scales=_powers(3, 2, 16, 2).transpose(1, 2)), "scales"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int64)), "seq_lens"),
    (dict(page_table=torch.zeros(3, 3, dtype=torch.int32)), "page_table"),
    (dict(cu_seqlens=None), "cu_seqlens"),
    (dict(k_pages=_codes(3, 2, 16, 64).transpose(1, 2), v_pages=_codes(3, 2, 16, 64).transpose(1, 2)), "dense"),
    (dict(k_pages=_codes(3, 16, 2, 32), v_pages=_codes(3, 16, 2, 32), q=torch.zeros(4, 4, 32), k=torch.zeros(4, 2, 32),
          v=torch.zeros(4, 2, 32)), "head_dim"),
    (dict(q=torch.zeros(4, 4, 64).half(), k=torch.zeros(4, 2, 64).half(), v=torch.zeros(4, 2, 64).half()), "float32 or"),
]
BAD_APPEND = [
    (dict(v=torch.zeros(4, 3, 64)), "match"), (dict(q=torch.zeros(3, 4, 64)), "match"),
    (dict(cos=torch.zeros(48, 32)), "together"), (dict(cos=torch.zeros(47, 32), sin=torch.zeros(47, 32)), "positions"),
    (dict(q_norm=torch.ones(32)), "q_norm"), (dict(k_norm=torch.ones(64).half()), "k_norm"),
    (dict(q_norm=torch.ones(64), q=None), "without q"), (dict(q_norm=torch.ones(64), k_norm=torch.ones(64).bfloat16()), "one dtype"),
]


@pytest.mark.parametrize("kw,match", BAD + BAD_APPEND)
def test_append_checks_its_arguments(kw, match):
    mode = FakeTensorMode()
    with mode, pytest.raises(ValueError, match=match):
        _append(_on("cuda", _case(**kw)))


@pytest.mark.parametrize("kw,match", BAD + [(dict(q=torch.zeros(4, 5, 64)), "share"), (dict(q=torch.zeros(4, 256)), "head_dim")])
def test_attention_checks_its_arguments(kw, match):
    mode = FakeTensorMode()
    with mode, pytest.raises(ValueError, match=match):
        _attend(_on("cuda", _case(**kw)))
    with mode, pytest.raises(ValueError, match=match):
        _prefix(_on("cuda", _case(**kw)))


@pytest.mark.parametrize("kw,match", [
    (dict(k_scales=None), "together"), (dict(k_scales=None, v_scales=None), "dtype"),
    (dict(cu_groups=torch.zeros(3, dtype=torch.int32)), "cu_groups"), (dict(cu_groups=torch.zeros(2)), "cu_groups"),
    (dict(prefix_lens=torch.zeros(1, dtype=torch.int64)), "prefix_lens"),
    (dict(prefix_lens=torch.zeros(1, 1, dtype=torch.int32)), "prefix_lens")])
def test_prefix_checks_its_groups(kw, match):
    with FakeTensorMode(), pytest.raises(ValueError, match=match):
        _prefix(_on("cuda", _case(**kw)))


def _rows(device="cuda", **kw):
    i32 = torch.int32
    z = dict(logits=torch.zeros(5, 10), drafts=torch.zeros(5, dtype=i32), uniform=torch.zeros(5), noise=torch.zeros(2, 10),
             cu_seqlens=torch.zeros(3, dtype=i32), draft_logits=torch.zeros(5, 10), temperature=torch.ones(2))
    return _on(device, {**z, **kw})


def _verify(x):
    from delta_feedback_experiment_amd import verify_tokens

    return verify_tokens(x["logits"], x["drafts"], x["uniform"], x["noise"], x["cu_seqlens"],
                         draft_logits=x["draft_logits"], temperature=x["temperature"])


@pytest.mark.parametrize("kw,match", [
    (dict(logits=torch.zeros(5)), "logits"), (dict(logits=torch.zeros(5, 0)), "logits"),
    (dict(logits=torch.zeros(5, 10).double()), "float32"), (dict(draft_logits=torch.zeros(4, 10)), "draft_logits"),
    (dict(draft_logits=torch.zeros(5, 10).bfloat16()), "draft_logits"), (dict(drafts=torch.zeros(5).long()), "drafts"),
    (dict(drafts=torch.zeros(4).int()), "drafts"), (dict(uniform=torch.zeros(5).double()), "uniform"),
    (dict(noise=torch.zeros(5, 10)), "noise"), (dict(noise=torch.zeros(2, 10).bfloat16()), "noise"),
    (dict(cu_seqlens=torch.zeros(0).int()), "cu_seqlens"), (dict(cu_seqlens=torch.zeros(3).long()), "cu_seqlens"),
    (dict(temperature=torch.ones(5)), "temperature")])
def test_verify_checks_its_arguments(kw, match):
    with FakeTensorMode(), pytest.raises(ValueError, match=match):
        _verify(_rows(**kw))


@pytest.mark.parametrize("device", ["cuda", "meta"])
def test_shapes_of_fake_and_meta_tensors(device):
    from contextlib import nullcontext

    from delta_feedback_experiment_amd import paged_append_

    with FakeTensorMode() if device == "cuda" else nullcontext():
        x = _on(device, _case(cos=torch.zeros(48, 32), sin=torch.zeros(48, 32), q_norm=torch.ones(64), k_norm=torch.ones(64)))
        q = _append(x)
        assert q.shape == x["q"].shape and q.dtype == x["q"].dtype
        for o, lse in (_attend(x), _prefix(x)):
            assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (4, 4) and lse.dtype == torch.float32
        plain = torch.empty(3, 16, 2, 64, device=device)
        q = paged_append_(x["k"], x["v"], plain, plain, x["page_table"], x["seq_lens"], cu_seqlens=x["cu_seqlens"], q=x["q"],
                          k_norm=x["k_norm"])
        assert q.shape == x["q"].shape
        tokens, accepted = _verify(_rows(device))
        assert tokens.shape == (5,) and accepted.shape == (2,) and tokens.dtype == accepted.dtype == torch.int32


def test_operators_refuse_cpu_tensors():
    for call, x in ((_append, _case()), (_attend, _case()), (_prefix, _case()), (_verify, _rows("cpu"))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call(x)


def test_a_new_cache_is_zeros():
    from delta_feedback_experiment_amd import PagedKVFP8

    kv = PagedKVFP8.zeros(3, 4, 2, 64, device="cpu")
    assert kv.k.dtype == kv.v.dtype == CODES and kv.k_scale.dtype == kv.v_scale.dtype == POWERS
    assert (kv.k.float() == 0).all() and (kv.v_scale.float() == 1).all() and kv.k_scale.shape == (3, 4, 2, 2)


def test_host_check_of_groups():
    from delta_feedback_experiment_amd.paged_prefix import validate_groups

    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    validate_groups(i32(0, 2, 2, 3), i32(5, 99, 0), i32(5, 9, 1, 7))
    for cu, prefix in ((i32(0, 2, 5), i32(1, 1)), (i32(0, 2, 1), i32(1, 1)), (i32(1, 2, 3), i32(1, 1)),
                       (i32(0, 2, 3), i32(6, 1)), (i32(0, 2, 3), i32(5, -1))):
        with pytest.raises(ValueError):
            validate_groups(cu, prefix, i32(5, 9, 1, 7))


def test_oracle_s_codes_are_the_type_s():
    """Its rounding against torch's, on every code, every middle and what is beside it."""
    every = torch.arange(256, dtype=torch.uint8).view(CODES).float()
    every = every[torch.isfinite(every)].sort().values.unique()
    mid = (every[1:] + every[:-1]) / 2
    x = torch.cat((every, mid, mid.nextafter(torch.tensor(1e9)), mid.nextafter(torch.tensor(-1e9))))
    assert torch.equal(fp8.rounded_to_e4m3(x), x.to(CODES).double())
    blocks = torch.randn(50, 64, generator=torch.Generator().manual_seed(0)) * torch.logspace(-44, 38, 50)[:, None]
    codes, scales = fp8.quantised(blocks)
    top = blocks.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    held = top <= 448 * scales  # (all but what the largest scale does not reach)
    assert (held | (scales == 2.0 ** 119)).all() and ((top > 224 * scales) | (scales == 2.0 ** -117)).all()
    value = codes * scales.repeat_interleave(32, -1)
    assert torch.equal(value, value.bfloat16().double())
    # a rounding is off by half a step of eight an octave, or of 2^-9 under 2^-6
    off = (value - blocks.double()).abs()
    half = torch.maximum(blocks.double().abs() * 2.0 ** -4, scales.repeat_interleave(32, -1) * 2.0 ** -10)
    assert ((off <= half) | ~held.repeat_interleave(32, -1)).all() and held.sum() > 90


def test_oracle_of_verification_finds_mistakes():
    gen = torch.Generator().manual_seed(1)
    V, cu = 50, torch.tensor([0, 3])
    l, ld = torch.randn(3, V, generator=gen), torch.randn(3, V, generator=gen)
    d = torch.tensor([4, 9, 0], dtype=torch.int32)
    u, noise = torch.tensor([0.0, 1.0, 0.5]), torch.randn(1, V, generator=gen)
    p, q = torch.softmax(l.double(), -1), torch.softmax(ld.double(), -1)
    u[1] = min(1.0, float(p[1, 9] / q[1, 9]) * 1.01)
    if q[1, 9] * u[1] < p[1, 9]:
        ld[1, 9] += 9
        q = torch.softmax(ld.double(), -1)
        u[1] = 0.999
    token = int(((p[1] - q[1]).clamp(min=0).log() + noise[0]).argmax())
    good = torch.tensor([4, token, -1], dtype=torch.int32)
    args = (l, d, u, noise, cu, ld)
    verify_oracle.check(good, torch.tensor([1]), *args)
    for tokens, accepted in (([4, (token + 1) % V, -1], 1), ([4, 9, token], 2), ([token, -1, -1], 0), ([4, token, 0], 1)):
        with pytest.raises(AssertionError):
            verify_oracle.check(torch.tensor(tokens, dtype=torch.int32), torch.tensor([accepted]), *args)
