"""The paged cache at its edges: bounds and lengths that cannot be, between
guarded buffers, and tables without an entry to spare.  Bars as in
test_gpu_paged.py.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from conftest import rel_l2
from oracle import paged_oracle as oracle
from test_gpu_paged import TOL, Cache, dev  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu

GUARD = 4096  # elements on either side


class Guarded:
    """A device tensor between two stretches of a pattern."""

    def __init__(self, shape, dtype, dev, value=None):
        n = 1
        for d in shape:
            n *= d
        self.whole = torch.full((n + 2 * GUARD,), 77.0, dtype=dtype, device=dev)
        self.t = self.whole[GUARD:GUARD + n].view(shape)
        if value is not None:
            self.t.copy_(value)

    def intact(self):
        return bool((self.whole[:GUARD] == 77).all() and (self.whole[-GUARD:] == 77).all())


def guarded_step(c, dev, lens, cu):
    """Append and attention through the C ABI, every buffer they write guarded;
    returns (q, k_pages, v_pages, o, lse)."""
    from delta_feedback_experiment_amd import _lib

    N, Hq, D = c.q.shape
    P, page, Hkv, _ = c.k_pages.shape
    table, q, k, v = (t.to(dev) for t in (c.table, c.q, c.k, c.v))
    kp, vp = (Guarded(t.shape, c.dtype, dev, t) for t in (c.k_pages, c.v_pages))
    q_out, o = (Guarded(q.shape, c.dtype, dev) for _ in range(2))
    lse = Guarded((N, Hq), torch.float32, dev)
    at = lambda t: t.data_ptr()  # noqa: E731
    common = dict(dtype=_lib.PKDA_BF16 if c.dtype == torch.bfloat16 else _lib.PKDA_F32, num_seqs=len(lens),
                  num_tokens=N, q_heads=Hq, kv_heads=Hkv, head_dim=D, page_size=page, max_pages=table.shape[1],
                  num_pages=P, table_stride=table.stride(0), cu_seqlens=at(cu), seq_lens=at(lens), page_table=at(table),
                  k_pages=at(kp.t), v_pages=at(vp.t), k_page_stride=kp.t.stride(0), v_page_stride=vp.t.stride(0),
                  q_stride=q.stride(0))
    stream = torch.cuda.current_stream().cuda_stream
    _lib.call("pkda_paged_append", _lib.PagedAppendArgs(q=at(q), k=at(k), v=at(v), k_stride=k.stride(0),
                                                        v_stride=v.stride(0), q_out=at(q_out.t), **common), stream)
    args = _lib.PagedAttentionArgs(q=at(q_out.t), scale=D ** -0.5, o=at(o.t), lse=at(lse.t), **common)
    args.struct_size = ctypes.sizeof(args)
    floats = _lib.lib().pkda_paged_attention_workspace(ctypes.byref(args))
    work = Guarded((max(floats, 4),), torch.float32, dev)
    args.workspace = at(work.t)
    _lib.call("pkda_paged_attention", args, stream)
    torch.cuda.synchronize()
    assert all(x.intact() for x in (kp, vp, q_out, o, lse, work))
    return q_out.t.cpu(), kp.t.cpu(), vp.t.cpu(), o.t.cpu(), lse.t.cpu()


def untouched(c, kp, vp):
    """Pages that no sequence owns are as they were."""
    used = torch.zeros(c.pages, dtype=torch.bool)
    used[c.table[(c.table >= 0) & (c.table < c.pages)].long()] = True
    return torch.equal(kp[~used], c.k_pages[~used]) and torch.equal(vp[~used], c.v_pages[~used])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clamped_bounds_and_lengths(dev, dtype):  # noqa: F811
    """Bounds that rise once they are clamped to the packed length (the first one
    counts as 0), and lengths clamped to the table's row, give the clamped ones' result."""
    print(f"[gpu] paged cache, clamped bounds {dtype}", flush=True)
    c = Cache([20, 30, 9], [4, 5, 6], 4, 2, 64, 8, dtype, seed=10, garbage=0.0, tail_pages=0)
    room = c.table.shape[1] * 8
    c.table[0], c.table[1], c.table[2] = torch.tensor([1, 0, 3, 2]), torch.tensor([7, 5, 4, 6]), -1
    for cu in ([0, 4, 9, 900], [3, 4, 9, 15], [-5, -4, 2 ** 31 - 1, 15], [0, 4, 9, 11]):
        for lens in ([20, 30, 9], [2 ** 31 - 1, -3, 9]):
            got = guarded_step(c, dev, *(torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, cu)))
            inside = torch.tensor([0, *(min(max(x, 0), 15) for x in cu[1:])])
            short = torch.tensor([min(max(x, 0), room) for x in lens])
            rq, rk, rv = oracle.append_reference(c.k, c.v, c.k_pages, c.v_pages, c.table, short, inside, c.q)
            assert all(torch.equal(a.double(), b) for a, b in zip(got[:3], (rq, rk, rv))), (cu, lens)
            assert untouched(c, got[1], got[2])
            ro, rl = oracle.attention_reference(rq.to(dtype), got[1], got[2], c.table, short, inside)
            assert rel_l2(got[3].float(), ro) < TOL[dtype], (cu, lens)
            assert torch.equal(torch.isneginf(got[4]), torch.isneginf(rl))


@pytest.mark.parametrize("S,N,Hq,Hkv", [(3, 60, 64, 4), (70, 300, 64, 4), (70, 300, 64, 64), (200, 3000, 16, 2),
                                        (5, 3000, 64, 16)])
def test_falling_bounds_stay_inside(dev, S, N, Hq, Hkv):  # noqa: F811
    """Bounds that fall name no sequences: nothing past a buffer is read or
    written, nothing in a page that no sequence has."""
    print(f"[gpu] paged cache, falling bounds {S} sequences {N} tokens", flush=True)
    gen = torch.Generator().manual_seed(S + N)
    new = [N // S] * S
    c = Cache([n + 5 for n in new], new, Hq, Hkv, 32, 8, torch.bfloat16, seed=31, garbage=0.0, tail=N - sum(new))
    lens = c.lens.to(dev)
    for _ in range(4):
        cu = torch.randint(-5, N + 5, (S + 1,), generator=gen, dtype=torch.int32).to(dev)
        _, kp, vp, _, _ = guarded_step(c, dev, lens, cu)
        assert untouched(c, kp, vp)
    falls = torch.arange(S, -1, -1, dtype=torch.int32).mul(N // S).to(dev)
    _, kp, vp, _, _ = guarded_step(c, dev, lens, falls)
    assert untouched(c, kp, vp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_a_bad_value_at_the_middle_of_the_last_tile(dev, dtype, page):  # noqa: F811
    """The last position is key 31 of a tile of 64, its value is not finite and
    the table ends there: the keys after it, which do not exist, are not looked
    up (the table is a view, with entries of the pool's behind each row)."""
    from delta_feedback_experiment_amd import paged_attention

    print(f"[gpu] paged attention, bad value at key 31 {dtype} pages of {page}", flush=True)
    c = Cache([160, 160], [100, 100], 128, 128, 32, page, dtype, seed=34, tail_pages=0, garbage=0.0)
    assert c.table.shape[1] * page == 160
    wide = torch.zeros(2, c.table.shape[1] + 64, dtype=torch.int32, device=dev)
    wide[:, :c.table.shape[1]] = c.table.to(dev)
    table, lens, cu = wide[:, :c.table.shape[1]], c.lens.to(dev), c.cu.to(dev)

    def attend():
        return paged_attention(c.q.to(dev), c.k_pages.to(dev), c.v_pages.to(dev), table, lens, cu_seqlens=cu)

    clean, lse0 = attend()
    c.v_pages[int(c.table[1, 159 // page]), 159 % page, :, 5] = math.nan
    o, lse = attend()
    assert torch.equal(lse, lse0) and torch.isnan(o[199, :, 5]).all()
    o[199, :, 5] = clean[199, :, 5]
    assert torch.equal(o, clean)


@pytest.mark.parametrize("lens,new,Hq,Hkv", [([300, 65], [150, 65], 64, 64), ([300], [1], 8, 2),
                                             ([300, 9], [40, 9], 4, 2)])
def test_the_likeliest_key_is_not_rounded(dev, lens, new, Hq, Hkv):  # noqa: F811
    """One key of the second tile has a larger score than the others, by less
    than 2^8 for most rows, and the only value: its probability against the row's
    maximum is 1, so the output is rounded once (FP32 sums: 1e-5 before that)."""
    print(f"[gpu] paged attention, likeliest key {lens} {Hq}/{Hkv}", flush=True)
    c = Cache(lens, new, Hq, Hkv, 64, 16, torch.bfloat16, seed=33, garbage=0.0)
    kept = c.v_pages.clone()
    c.k_pages.zero_()
    c.v_pages.zero_()
    for n, length in enumerate(lens):
        at = 70 if length > 70 else 3
        where = int(c.table[n, at // 16]), at % 16
        c.k_pages[where][:, 0] = 1.0
        c.v_pages[where] = kept[where]
    c.q.abs_()
    o, _ = c.attend(dev, scale=1.0)
    ro, _ = oracle.attention_of_sequences(c.q, c.k_pages, c.v_pages, c.table, c.lens, c.cu, 1.0)
    slack = 1e-5 * ro.abs()
    assert ((o.cpu() >= (ro - slack).bfloat16()) & (o.cpu() <= (ro + slack).bfloat16())).all()


def test_function_modes_and_lazy_negations(dev):  # noqa: F811
    """A function mode sees the operators, and a lazily negated view is negated."""
    from torch.overrides import TorchFunctionMode

    from delta_feedback_experiment_amd import paged_append_, paged_attention, sample_tokens

    print("[gpu] paged cache, function modes", flush=True)
    c = Cache([3, 9], [1, 1], 4, 2, 64, 8, torch.float32, seed=35, cu=False, garbage=0.0)
    table, lens, _ = c.tables(dev)
    q, k, v = (t.to(dev) for t in (c.q, c.k, c.v))
    logits, noise = torch.randn(2, 100, device=dev), torch.randn(2, 100, device=dev)

    def run(q, k, logits):
        kp, vp = c.k_pages.to(dev), c.v_pages.to(dev)
        out = paged_append_(k, v, kp, vp, table, lens, q=q)
        return (out, kp, vp, *paged_attention(q, kp, vp, table, lens), *sample_tokens(logits, noise))

    class Watch(TorchFunctionMode):
        def __init__(self):
            super().__init__()
            self.seen = set()

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.seen.add(str(func))
            return func(*args, **(kwargs or {}))

    with Watch() as watch:
        watched = run(q, k, logits)
    for name in ("paged_append_", "paged_attention", "sample_tokens"):
        assert any(name in f for f in watch.seen), name
    assert all(torch.equal(a, b) for a, b in zip(watched, run(q, k, logits)))
    negated = run(*(torch._neg_view(t) for t in (q, k, logits)))
    assert all(torch.equal(a, b) for a, b in zip(negated, run(-q, -k, -logits)))


def test_pages_of_one_head_kept_by_head(dev):  # noqa: F811
    """Pools [pages, 1, page_size, head_dim], turned: dense all the same."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention

    print("[gpu] paged cache, one head", flush=True)
    c = Cache([3, 30], [2, 30], 4, 1, 64, 8, torch.bfloat16, seed=36, garbage=0.0)
    table, lens, cu = c.tables(dev)
    q, k, v = (t.to(dev) for t in (c.q, c.k, c.v))
    runs = []
    for turned in (False, True):
        kp, vp = (t.to(dev) for t in (c.k_pages, c.v_pages))
        if turned:
            kp, vp = (t.view(c.pages, 1, 8, 64).transpose(1, 2) for t in (kp, vp))
        out = paged_append_(k, v, kp, vp, table, lens, cu_seqlens=cu, q=q)
        runs.append((out, kp, vp, *paged_attention(out, kp, vp, table, lens, cu_seqlens=cu)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_step_without_tokens(dev):  # noqa: F811
    """Live sequences, none of which has a new token."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention

    print("[gpu] paged cache, no tokens", flush=True)
    c = Cache([20, 3], [0, 0], 4, 2, 64, 8, torch.bfloat16, seed=37, garbage=0.0)
    table, lens, cu = c.tables(dev)
    q, k, v, kp, vp = (t.to(dev) for t in (c.q, c.k, c.v, c.k_pages, c.v_pages))
    out = paged_append_(k, v, kp, vp, table, lens, cu_seqlens=cu, q=q)
    o, lse = paged_attention(q, kp, vp, table, lens, cu_seqlens=cu)
    torch.cuda.synchronize()
    assert out.shape == o.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert torch.equal(kp.cpu(), c.k_pages) and torch.equal(vp.cpu(), c.v_pages)
