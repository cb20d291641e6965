"""The paged key/value cache on the GPU: append with rotation, and attention
over the cache, against the 64-bit oracle.

Bars, from the arithmetic:

* append: rotated values are FP32 sums of two products, off by at most 2^-21
  of the largest input, then rounded once to the type: between the roundings
  of the exact value less and plus that; copied values are equal;
* attention, FP32: the framework's FP32 bar 1e-5 (relative L2);
* attention, BF16: the probabilities and the output are each rounded once to
  eight bits: a root mean square error of 2^-8 / sqrt(6) of their own size
  (uniform over the mantissas), independent of each other; both together are
  0.58 of 2^-8 (relative L2), and the bar is 2^-8;
* lse: scores of up to a few tens, FP32 sums: 1e-5 (1 + |lse|).
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import rel_l2
from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


class Cache:
    """A used cache on the CPU: pages in random order, garbage in what no sequence holds."""

    def __init__(self, lens, new, Hq, Hkv, D, page, dtype, *, seed=0, garbage=math.nan, spare=3, tail_pages=2, tail=0,
                 cu=True):
        gen = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=gen).tolist()
        # past a sequence's pages the table holds what the caller left there
        self.table = torch.full((len(lens), max([*need, 0]) + tail_pages), -7, dtype=torch.int32)
        self.table[:, -1:] = self.pages + 99
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.cu = torch.tensor(starts, dtype=torch.int32) if cu else None
        N = starts[-1] + tail
        self.k_pages = torch.full((self.pages, page, Hkv, D), garbage)
        self.v_pages = torch.full((self.pages, page, Hkv, D), garbage)
        for i, n in enumerate(lens):
            for p in range(n):
                row = int(self.table[i, p // page])
                self.k_pages[row, p % page] = torch.randn(Hkv, D, generator=gen)
                self.v_pages[row, p % page] = torch.randn(Hkv, D, generator=gen)
        self.k_pages, self.v_pages = self.k_pages.to(dtype), self.v_pages.to(dtype)
        self.q = (2 * torch.randn(N, Hq, D, generator=gen)).to(dtype)
        self.k, self.v = (torch.randn(N, Hkv, D, generator=gen).to(dtype) for _ in range(2))
        self.dtype = dtype

    def tables(self, dev):
        return self.table.to(dev), self.lens.to(dev), None if self.cu is None else self.cu.to(dev)

    def attend(self, dev, **kw):
        from delta_feedback_experiment_amd import paged_attention

        table, lens, cu = self.tables(dev)
        o, lse = paged_attention(self.q.to(dev), self.k_pages.to(dev), self.v_pages.to(dev), table, lens,
                                 cu_seqlens=cu, **kw)
        torch.cuda.synchronize()
        return o, lse

    def check(self, dev, **kw):
        o, lse = self.attend(dev, **kw)
        ro, rl = oracle.attention_reference(self.q, self.k_pages, self.v_pages, self.table, self.lens, self.cu, **kw)
        assert torch.isfinite(o).all()
        empty = torch.isinf(rl)
        assert torch.equal(torch.isinf(lse.cpu()) & (lse.cpu() < 0), empty)
        assert (o.cpu()[empty] == 0).all()
        err = rel_l2(o.float(), ro) if ro.abs().max() > 0 else 0.0
        gap = ((lse.cpu().double() - rl).abs() / (1 + rl.abs()))[~empty]
        gap = float(gap.max()) if gap.numel() else 0.0
        print(f"  o {err:.2e} lse {gap:.2e}", flush=True)
        assert err < TOL[self.dtype] and gap < 1e-5
        return o, lse


# lens and new tokens of each sequence: nothing, one, a page's edge, inside and past tiles
RAGGED = ([0, 1, 16, 33, 64, 65, 130, 257], [0, 1, 1, 33, 2, 5, 64, 130])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 4, 32, 16), (8, 2, 64, 24), (5, 1, 128, 8), (16, 2, 128, 64),
                                           (3, 3, 64, 1), (40, 1, 64, 128)])
def test_attention_of_ragged_chunks(dev, dtype, Hq, Hkv, D, page):
    print(f"[gpu] paged attention {dtype} {Hq}/{Hkv} x {D}, pages of {page}", flush=True)
    Cache(*RAGGED, Hq, Hkv, D, page, dtype, seed=D + page).check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 128, 16), (12, 2, 64, 24), (2, 2, 32, 64), (64, 1, 128, 64)])
def test_attention_of_single_tokens(dev, dtype, Hq, Hkv, D, page):
    """The decode form: no cu_seqlens; empty, short and longer sequences."""
    print(f"[gpu] paged decode {dtype} {Hq}/{Hkv} x {D}, pages of {page}", flush=True)
    lens = [0, 1, 2, 63, 64, 65, 511, 700, 1031]
    Cache(lens, [1] * len(lens), Hq, Hkv, D, page, dtype, seed=D, cu=False).check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_one_long_sequence(dev, dtype):
    """One sequence whose positions are split over the card, and a chunk at its end."""
    print(f"[gpu] paged attention, long {dtype}", flush=True)
    Cache([4999], [1], 4, 1, 64, 16, dtype, seed=1, cu=False).check(dev)
    Cache([4999], [37], 4, 2, 64, 16, dtype, seed=2).check(dev)
    Cache([700, 3000], [1, 300], 2, 1, 128, 16, dtype, seed=3).check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_tokens_without_keys(dev, dtype):
    """Padding past cu_seqlens[-1], more new tokens than positions, missing pages."""
    print(f"[gpu] paged attention without keys {dtype}", flush=True)
    c = Cache([7, 40, 3], [3, 40, 9], 8, 2, 64, 8, dtype, seed=4, tail=6)
    c.check(dev)
    c.table[1, 0], c.table[1, 2] = -1, c.pages  # holes: nothing there
    c.check(dev)
    c.table[0, 0] = 2 ** 31 - 1
    c.check(dev)


def test_no_sequences_and_no_pages(dev):
    from delta_feedback_experiment_amd import paged_append_, paged_attention

    i32 = dict(dtype=torch.int32, device=dev)
    pages = torch.zeros(0, 16, 2, 64, device=dev)
    empty = torch.zeros(0, 4, 64, device=dev)
    o, lse = paged_attention(empty, pages, pages, torch.zeros(0, 0, **i32), torch.zeros(0, **i32))
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.randn(3, 4, 64, device=dev)
    kv = torch.randn(3, 2, 64, device=dev)
    table, lens = torch.zeros(3, 0, **i32), torch.tensor([0, 5, 1], **i32)
    o, lse = paged_attention(q, pages, pages, table, lens)
    assert (o == 0).all() and torch.isneginf(lse).all()
    out = paged_append_(kv, kv, pages, pages, table, lens, q=q)
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_later_tokens_do_not_reach_earlier_ones(dev, dtype, bad):
    """A later token's keys and values, whatever they are, change no earlier
    token of its chunk; the row's own do."""
    print(f"[gpu] paged attention, later tokens {dtype} {bad}", flush=True)
    for lens, new, Hq, Hkv in (([90], [60], 4, 2), ([200], [150], 16, 1), ([70, 33], [5, 33], 4, 4)):
        c = Cache(lens, new, Hq, Hkv, 64, 16, dtype, seed=5)
        clean, _ = c.attend(dev)
        at = lens[0] - 3  # the third token from the end
        page, row = int(c.table[0, at // 16]), at % 16
        c.v_pages[page, row, 0, 5] = bad
        c.k_pages[page, row, 0, 7] = bad
        o, _ = c.attend(dev)
        first = new[0] - 3  # that token's row
        assert torch.equal(o[:first], clean[:first])
        assert torch.equal(o[new[0]:], clean[new[0]:])
        hit = o[first:new[0], :Hq // Hkv]
        if math.isnan(bad):
            assert torch.isnan(hit).all()
        assert torch.equal(o[first:new[0], Hq // Hkv:], clean[first:new[0], Hq // Hkv:])


def test_value_of_a_later_token_alone(dev):
    """The value rows only: the masked probability is zero, not zero times the value."""
    for dtype in (torch.float32, torch.bfloat16):
        c = Cache([130], [130], 8, 1, 128, 16, dtype, seed=6)
        clean, lse0 = c.attend(dev)
        for at in (1, 63, 64, 100, 129):
            c2 = Cache([130], [130], 8, 1, 128, 16, dtype, seed=6)
            c2.v_pages[int(c.table[0, at // 16]), at % 16, 0, 3] = math.inf
            o, lse = c2.attend(dev)
            assert torch.equal(o[:at], clean[:at]) and torch.equal(lse, lse0), at
            keep = [i for i in range(128) if i != 3]
            assert torch.equal(o[at:][..., keep], clean[at:][..., keep]), at
            assert torch.isposinf(o[at:, :, 3]).all(), at


def test_large_scores_and_equal_scores(dev):
    """Scores past exp's range (the running maximum holds them), and rows of equal scores."""
    print("[gpu] paged attention, large and equal scores", flush=True)
    for dtype in (torch.float32, torch.bfloat16):
        c = Cache([300, 65], [20, 65], 4, 2, 64, 16, dtype, seed=7)
        c.q *= 40
        c.check(dev, scale=1.0) if dtype == torch.float32 else c.check(dev, scale=0.25)
        c.q.zero_()
        c.check(dev)


def test_strided_queries_pools_and_tables(dev):
    """Queries as a slice of a projection, K and V in one pool, a table that is a
    view of a wider one; scale given."""
    from delta_feedback_experiment_amd import paged_attention

    print("[gpu] paged attention, strides", flush=True)
    for dtype in (torch.float32, torch.bfloat16):
        c = Cache(*RAGGED, 8, 2, 64, 16, dtype, seed=8)
        plain, plain_lse = c.attend(dev, scale=0.3)
        N = c.q.shape[0]
        wide = torch.randn(N, 13 * 64, device=dev).to(dtype)
        q = wide[:, 64:9 * 64].unflatten(-1, (8, 64))
        q.copy_(c.q)
        pool = torch.stack((c.k_pages, c.v_pages), 1).to(dev)  # [P, 2, page, H, D]
        table = torch.full((len(c.lens), c.table.shape[1] + 5), 3, dtype=torch.int32, device=dev)
        table[:, 2:-3] = c.table.to(dev)
        o, lse = paged_attention(q, pool[:, 0], pool[:, 1], table[:, 2:-3], c.lens.to(dev), cu_seqlens=c.cu.to(dev),
                                 scale=0.3)
        assert torch.equal(o, plain) and torch.equal(lse, plain_lse)
        # heads apart, and an odd offset: copied to what the kernels read
        odd = torch.randn(N * 8 * 64 + 1, device=dev).to(dtype)[1:].view(N, 8, 64)
        odd.copy_(c.q)
        turned = c.q.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
        for x in (odd, turned):
            o, lse = paged_attention(x, pool[:, 0], pool[:, 1], c.table.to(dev), c.lens.to(dev),
                                     cu_seqlens=c.cu.to(dev), scale=0.3)
            assert torch.equal(o, plain) and torch.equal(lse, plain_lse)


def test_offsets_past_32_bits(dev):
    """Pages more than 2^32 bytes into the pool, in append and attention."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention

    print("[gpu] paged cache past 2^32 bytes", flush=True)
    H, D, page = 2, 64, 16
    stride = 2 ** 31 + 2 ** 20  # elements: page 1 begins past 2^32 bytes
    pools = [torch.empty(stride + page * H * D, dtype=torch.bfloat16, device=dev).as_strided(
        (2, page, H, D), (stride, H * D, D, 1)) for _ in range(2)]
    gen = torch.Generator().manual_seed(9)
    k, v = (torch.randn(16, H, D, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn(16, 4, D, generator=gen).bfloat16()
    table = torch.tensor([[1]], dtype=torch.int32)
    lens, cu = torch.tensor([16], dtype=torch.int32), torch.tensor([0, 16], dtype=torch.int32)
    pools[0][0].zero_(), pools[1][0].zero_()
    paged_append_(k.to(dev), v.to(dev), *pools, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev))
    assert torch.equal(pools[0][1].cpu(), k) and torch.equal(pools[1][1].cpu(), v)
    assert (pools[0][0] == 0).all()
    o, _ = paged_attention(q.to(dev), *pools, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev))
    ref, _ = oracle.attention_reference(q, torch.stack((k, k)), torch.stack((v, v)), table, lens, cu)
    assert rel_l2(o.float(), ref) < TOL[torch.bfloat16]


def test_malformed_bounds_stay_inside(dev):
    """cu_seqlens and lengths that cannot be: clamped, nothing read or written past the buffers."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention

    print("[gpu] paged cache, malformed bounds", flush=True)
    c = Cache([20, 30, 9], [4, 5, 6], 4, 2, 64, 8, torch.bfloat16, seed=10, garbage=0.0)
    table = c.table.to(dev)
    for cu in ([0, 4, 9, 900], [0, 12, 3, 15], [3, 4, 9, 15], [-5, -4, 2 ** 31 - 1, 15]):
        for lens in ([20, 30, 9], [2 ** 31 - 1, -3, 9]):
            cu_t, lens_t = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (cu, lens))
            kp, vp = c.k_pages.to(dev), c.v_pages.to(dev)
            q = paged_append_(c.k.to(dev), c.v.to(dev), kp, vp, table, lens_t, cu_seqlens=cu_t, q=c.q.to(dev))
            paged_attention(q, kp, vp, table, lens_t, cu_seqlens=cu_t)
            torch.cuda.synchronize()


def test_repeats_streams_and_graph(dev):
    """The same bits every time: repeated, on another stream, and replayed from
    a graph with other work between the replays."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention

    print("[gpu] paged cache, repeats", flush=True)
    for lens, new, cu in ((RAGGED[0], RAGGED[1], True), ([5, 900, 2000], [1, 1, 1], False)):
        c = Cache(lens, new, 8, 2, 128, 16, torch.bfloat16, seed=11)
        table, lens_t, cu_t = c.tables(dev)
        cu_t = cu_t if cu else None
        q, k, v, kp, vp = (t.to(dev) for t in (c.q, c.k, c.v, c.k_pages, c.v_pages))

        def step():
            qr = paged_append_(k, v, kp, vp, table, lens_t, cu_seqlens=cu_t, q=q)
            return paged_attention(qr, kp, vp, table, lens_t, cu_seqlens=cu_t)

        first = [t.clone() for t in step()]
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, step()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i in range(4):
            q.normal_()
            eager = [t.clone() for t in step()]
            out[0].fill_(float(i))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,page,rotary,interleaved", [
    (8, 2, 128, 16, 128, False), (8, 2, 128, 16, 128, True), (5, 5, 64, 24, 32, False), (3, 1, 64, 8, 16, True),
    (40, 8, 128, 64, 64, False), (2, 2, 32, 1, 32, True), (9, 3, 32, 16, 0, False)])
def test_append_against_the_oracle(dev, dtype, Hq, Hkv, D, page, rotary, interleaved):
    from delta_feedback_experiment_amd import paged_append_

    print(f"[gpu] append {dtype} {Hq}/{Hkv} x {D} rotary {rotary}", flush=True)
    c = Cache([0, 1, 16, 33, 64, 65, 130, 3], [0, 1, 1, 33, 2, 5, 64, 5], Hq, Hkv, D, page, dtype, seed=12, garbage=0.5,
              tail=3)
    c.table[5, 0] = -1 if page > 60 else c.table[5, 0]
    cos = sin = None
    if rotary:
        angle = torch.rand(c.table.shape[1] * page, rotary // 2) * 6.28
        cos, sin = angle.cos(), angle.sin()
    # k, v, q as slices of one projection
    packed = torch.cat((c.q, c.k, c.v), 1).flatten(1).to(dev)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in packed.split((Hq * D, Hkv * D, Hkv * D), -1))
    kp, vp = c.k_pages.to(dev), c.v_pages.to(dev)
    table, lens, cu = c.tables(dev)
    put = dict(cos=None if cos is None else cos.to(dev), sin=None if sin is None else sin.to(dev),
               interleaved=interleaved)
    out = paged_append_(k, v, kp, vp, table, lens, cu_seqlens=cu, q=q, **put)
    torch.cuda.synchronize()
    rq, rk, rv = oracle.append_reference(c.k, c.v, c.k_pages, c.v_pages, c.table, c.lens, c.cu, c.q, cos, sin,
                                         interleaved)
    assert torch.equal(vp.cpu().double(), rv)
    for got, ref, src in ((out, rq, c.q), (kp, rk, c.k)):
        eps = 2 ** -22 * float(src.abs().max()) * 2
        assert ((got.cpu() >= (ref - eps).to(dtype)) & (got.cpu() <= (ref + eps).to(dtype))).all()
        if not rotary:
            assert torch.equal(got.cpu().double(), ref)
    # without queries: the same cache
    kp2, vp2 = c.k_pages.to(dev), c.v_pages.to(dev)
    assert paged_append_(k, v, kp2, vp2, table, lens, cu_seqlens=cu, **put) is None
    assert torch.equal(kp, kp2) and torch.equal(vp, vp2)


def test_append_of_many_sequences(dev):
    """More sequences than a search step's 64 candidates, empty ones among them; single tokens too."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention

    print("[gpu] append, 5000 sequences", flush=True)
    gen = torch.Generator().manual_seed(13)
    S = 5000
    new = torch.randint(0, 4, (S,), generator=gen)
    lens = (new + torch.randint(0, 5, (S,), generator=gen)).int()
    cu = torch.cat((torch.zeros(1), new.cumsum(0))).int()
    N = int(cu[-1])
    table = torch.randperm(S, generator=gen).int()[:, None]
    k, v = (torch.randn(N, 1, 32, generator=gen) for _ in range(2))
    kp, vp = (torch.randn(S, 8, 1, 32, generator=gen) for _ in range(2))
    q = torch.randn(N, 2, 32, generator=gen)
    dk, dvp = kp.to(dev), vp.to(dev)
    out = paged_append_(k.to(dev), v.to(dev), dk, dvp, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev), q=q.to(dev),
                        check_pages=True)
    _, rk, rv = oracle.append_reference(k, v, kp, vp, table, lens, cu)
    assert torch.equal(out.cpu(), q) and torch.equal(dk.cpu().double(), rk) and torch.equal(dvp.cpu().double(), rv)
    o, lse = paged_attention(out, dk, dvp, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev))
    ro, rl = oracle.attention_reference(q, dk.cpu(), dvp.cpu(), table, lens, cu)
    assert rel_l2(o, ro) < TOL[torch.float32] and float((lse.cpu() - rl).abs().max()) < 1e-5


def test_chunks_then_tokens_equal_one_prompt(dev):
    """A prompt appended and attended in pieces, then token by token, gives what
    one call over the whole prompt gives."""
    from delta_feedback_experiment_amd import PagedKV, paged_append_, paged_attention

    print("[gpu] chunks then tokens", flush=True)
    gen = torch.Generator().manual_seed(14)
    L, Hq, Hkv, D, page = 150, 8, 2, 64, 16
    q, k, v = (torch.randn(L, h, D, generator=gen).to(dev) for h in (Hq, Hkv, Hkv))
    angle = torch.rand(160, D // 2, generator=gen).to(dev) * 6.28
    rope = dict(cos=angle.cos(), sin=angle.sin())
    table = torch.randperm(10, generator=gen).int()[None].to(dev)

    def run(pieces):
        kv = PagedKV.zeros(10, page, Hkv, D, dtype=torch.float32)
        outs, at = [], 0
        for n in pieces:
            sl = slice(at, at + n)
            at += n
            lens = torch.tensor([at], dtype=torch.int32, device=dev)
            cu = None if n == 1 else torch.tensor([0, n], dtype=torch.int32, device=dev)
            qr = paged_append_(k[sl], v[sl], kv.k, kv.v, table, lens, cu_seqlens=cu, q=q[sl], **rope)
            outs.append(paged_attention(qr, kv.k, kv.v, table, lens, cu_seqlens=cu)[0])
        return torch.cat(outs)

    whole = run([L])
    assert rel_l2(run([64, 33, 40] + [1] * 13), whole) < 2 * TOL[torch.float32]


def test_modes_and_profilers_see_the_operators(dev):
    """Called past the dispatcher when nothing watches, through it otherwise:
    the same results, version counters raised either way."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from delta_feedback_experiment_amd import paged_append_, paged_attention, sample_tokens

    print("[gpu] paged cache, dispatch", flush=True)
    c = Cache([3, 9], [1, 1], 4, 2, 64, 8, torch.bfloat16, seed=15, cu=False)
    table, lens, _ = c.tables(dev)
    q, k, v = (t.to(dev) for t in (c.q, c.k, c.v))
    logits, noise = torch.randn(2, 100, device=dev), torch.randn(2, 100, device=dev)

    def run(q=q):
        kp, vp = c.k_pages.to(dev), c.v_pages.to(dev)
        version = kp._version
        out = paged_append_(k, v, kp, vp, table, lens, q=q)
        assert kp._version == vp._version == version + 1
        return (out, kp, *paged_attention(out, kp, vp, table, lens), *sample_tokens(logits, noise))

    class Watch(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(func._schema.name.split("::")[-1])
            return func(*args, **(kwargs or {}))

    names = {"paged_append_", "paged_attention", "sample_tokens"}
    plain = run()
    with Watch() as watch:
        watched = run()
    assert names <= set(watch.seen)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        profiled = run()
    assert names <= {e.name.split("::")[-1] for e in prof.events()}
    for other in (watched, profiled, run(q.requires_grad_())):
        assert all(torch.equal(a.detach().nan_to_num(9), b.nan_to_num(9)) for a, b in zip(other, plain))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_full_card_splits_long_sequences_only(dev, dtype):
    """512 (sequence, head) pairs: those of up to 1,024 positions stay whole, the
    others are split; none where the table holds no more than 2,048."""
    print(f"[gpu] paged attention, whole and split {dtype}", flush=True)
    for lens in ([1024, 1025, 2600, 7], [1024, 1500, 2000, 0]):
        c = Cache(lens, [1] * 4, 128, 128, 32, 16, dtype, seed=17, cu=False, tail_pages=1)
        o, lse = c.attend(dev)
        cu = torch.arange(5, dtype=torch.int32)
        ro, rl = oracle.attention_of_sequences(c.q, c.k_pages, c.v_pages, c.table, c.lens, cu)
        assert rel_l2(o.float(), ro) < TOL[dtype]
        some = c.lens > 0
        gap = (lse.cpu().double() - rl).abs() / (1 + rl.abs())
        assert float(gap[some].max()) < 1e-5 and torch.isneginf(lse.cpu()[~some]).all()


def test_opcheck_and_compile(dev):
    """The schemas' marks match what the kernels write, the fake forms agree in
    shape and dtype, and a compiled step gives the eager bits."""
    from delta_feedback_experiment_amd import paged_append_, paged_attention, sample_tokens

    print("[gpu] paged cache, opcheck and compile", flush=True)
    c = Cache([3, 9, 20], [2, 1, 20], 4, 2, 64, 8, torch.bfloat16, seed=18)
    table, lens, cu = c.tables(dev)
    q, k, v, kp, vp = (t.to(dev) for t in (c.q, c.k, c.v, c.k_pages.nan_to_num(0.5), c.v_pages.nan_to_num(0.5)))
    angle = torch.rand(table.shape[1] * 8, 32, device=dev)
    logits, noise = torch.randn(3, 100, device=dev), torch.randn(3, 100, device=dev)
    ops, utils = torch.ops.pkda_mi355x, ("test_schema", "test_faketensor")
    for query in (q, None):
        torch.library.opcheck(ops.paged_append_.default,
                              (k, v, kp, vp, table, lens, cu, query, angle.cos(), angle.sin(), False), test_utils=utils)
    torch.library.opcheck(ops.paged_attention.default, (q, kp, vp, table, lens, cu, 0.125), test_utils=utils)
    torch.library.opcheck(ops.sample_tokens.default, (logits, noise, None, None, None, None, 0.7, 5, 0.9, 0.01),
                          test_utils=utils)

    def step(q, k, v, kp, vp):
        q = paged_append_(k, v, kp, vp, table, lens, cu_seqlens=cu, q=q, cos=angle.cos(), sin=angle.sin())
        o, lse = paged_attention(q * 1.0, kp, vp, table, lens, cu_seqlens=cu)
        return (o, lse, *sample_tokens(logits + o.float().mean() * 0, noise, top_k=5))

    pools = [(kp.clone(), vp.clone()) for _ in range(2)]
    eager = step(q, k, v, *pools[0])
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, *pools[1])
    for a, b in zip((*eager, *pools[0]), (*compiled, *pools[1])):
        assert torch.equal(a, b)
