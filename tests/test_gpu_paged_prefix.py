"""Attention of a batch in groups that share their first positions, on the GPU,
against the 64-bit oracle of plain paged attention (which the groups do not
change).

Bars: those of paged attention (FP32 1e-5, BF16 2^-8, relative L2; lse
1e-5 (1 + |lse|)): the parts of a row are FP32, each probability is rounded once
as an operand whatever part it is in, and joining them adds a few roundings of
2^-24.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import rel_l2
from oracle import paged_fp8_oracle as fp8
from oracle import paged_oracle as oracle
from test_gpu_paged import TOL

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


class Batch:
    """Sequences of ``own[n]`` positions behind the prefix of their group; whole pages
    of it shared, one that it fills in part copied; groups (prefix, sequences)."""

    def __init__(self, groups, own, new, Hq, Hkv, D, page, dtype, *, fp8_cache=False, seed=0, garbage=math.nan, tail=0,
                 cu=True, loose=0):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.page = dtype, page
        self.prefix = torch.tensor([p for p, _ in groups], dtype=torch.int32)
        bounds = [0]
        for _, n in groups:
            bounds.append(bounds[-1] + n)
        self.groups = torch.tensor(bounds, dtype=torch.int32)
        assert len(own) == bounds[-1] + loose
        of = [p for p, n in groups for _ in range(n)] + [0] * loose
        lens = [p + o for p, o in zip(of, own)]
        self.lens = torch.tensor(lens, dtype=torch.int32)
        width = max([-(-n // page) for n in lens] + [0]) + 2
        self.table = torch.full((len(own), width), -7, dtype=torch.int32)
        need, shared = 0, []
        for g, (p, n) in enumerate(groups):
            shared.append(range(need, need + p // page))
            need += p // page
        for i, n in enumerate(lens):
            g = next((g for g in range(len(groups)) if bounds[g] <= i < bounds[g + 1]), None)
            pages = list(shared[g]) if g is not None else []
            more = max(0, -(-n // page) - len(pages))
            pages += range(need, need + more)
            need += more
            self.table[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        order = torch.randperm(need + 3, generator=gen)
        self.pages = need + 3
        self.table = torch.where((self.table >= 0), order[self.table.clamp(min=0).long()].int(), self.table)
        k, v = (torch.full((self.pages, page, Hkv, D), garbage) for _ in range(2))
        for g, (p, n) in enumerate(groups):
            content = [torch.randn(p, Hkv, D, generator=gen) for _ in range(2)]
            for i in range(bounds[g], bounds[g + 1]):
                self._put(k, v, i, 0, content)
        for i, (p, o) in enumerate(zip(of, own)):
            self._put(k, v, i, p, [torch.randn(max(o, 0), Hkv, D, generator=gen) for _ in range(2)])
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.cu = torch.tensor(starts, dtype=torch.int32) if cu else None
        self.q = (2 * torch.randn(starts[-1] + tail, Hq, D, generator=gen)).to(dtype)
        self.scales = (None, None)
        if fp8_cache:
            (kc, ks), (vc, vs) = (fp8.quantised(x) for x in (k, v))
            self.k, self.v = (x.float().to(torch.float8_e4m3fn) for x in (kc, vc))
            self.scales = tuple(x.float().to(torch.float8_e8m0fnu) for x in (ks, vs))
        else:
            self.k, self.v = k.to(dtype), v.to(dtype)

    def _put(self, k, v, n, first, content):
        at = first + torch.arange(content[0].shape[0])
        page, row = self.table[n, at // self.page].long(), at % self.page
        k[page, row], v[page, row] = content

    def values(self):
        if self.scales[0] is None:
            return self.k.double(), self.v.double()
        return tuple(fp8.values(c, s) for c, s in zip((self.k, self.v), self.scales))

    def args(self, dev):
        on = lambda t: None if t is None else t.to(dev)  # noqa: E731
        return ([on(t) for t in (self.q, self.k, self.v, self.table, self.lens, self.groups, self.prefix)],
                dict(k_scales=on(self.scales[0]), v_scales=on(self.scales[1]), cu_seqlens=on(self.cu)))

    def attend(self, dev, **kw):
        from delta_feedback_experiment_amd import paged_prefix_attention

        args, more = self.args(dev)
        out = paged_prefix_attention(*args, **more, **kw)
        torch.cuda.synchronize()
        return out

    def reference(self, **kw):
        cu = torch.arange(len(self.lens) + 1, dtype=torch.int32) if self.cu is None else self.cu
        k, v = (x.nan_to_num(0.0) for x in self.values())
        return oracle.attention_of_sequences(self.q, k, v, self.table, self.lens, cu, **kw)

    def check(self, dev, **kw):
        o, lse = self.attend(dev, **kw)
        ro, rl = self.reference(**{k: v for k, v in kw.items() if k == "scale"})
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


KINDS = [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, True)]


@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 64, 16), (16, 4, 128, 64), (5, 1, 128, 24), (12, 12, 64, 7)])
def test_single_tokens_of_groups(dev, dtype, eight, Hq, Hkv, D, page):
    """Prefixes of nothing, less than a tile, a tile, odd and long; groups of one and many."""
    print(f"[gpu] prefix decode {dtype} fp8 {eight} {Hq}/{Hkv} x {D}, pages of {page}", flush=True)
    groups = [(0, 2), (1, 3), (63, 1), (64, 4), (65, 2), (700, 9), (1000, 1), (129, 0)]
    own = [1, 9, 1, 2, 130, 5, 1, 64, 65, 300, 77, 1, 1, 2, 3, 40, 50, 60, 70, 80, 500, 33]
    Batch(groups, own, [1] * len(own), Hq, Hkv, D, page, dtype, fp8_cache=eight, seed=D + page, cu=False).check(dev)


@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 64, 16), (4, 1, 128, 13)])
def test_drafts_and_chunks_of_groups(dev, dtype, eight, Hq, Hkv, D, page):
    """Several new tokens a sequence, sequences without any, padding, loose sequences."""
    print(f"[gpu] prefix chunks {dtype} fp8 {eight} {Hq}/{Hkv} x {D}, pages of {page}", flush=True)
    groups = [(200, 5), (64, 1), (515, 4), (10, 2)]
    new = [1, 5, 0, 3, 7, 40, 2, 0, 33, 1, 9, 4, 6, 20]
    own = [n + x for n, x in zip(new, [0, 3, 5, 60, 1, 0, 100, 2, 7, 200, 0, 0, 11, 90])]
    Batch(groups, own, new, Hq, Hkv, D, page, dtype, fp8_cache=eight, seed=3, tail=5, loose=2).check(dev)


@pytest.mark.parametrize("dtype,eight", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
@pytest.mark.parametrize("page", [16, 11])
def test_large_groups_of_many_rows(dev, dtype, eight, page):
    """Groups whose rows are tiles of 128, over a card that takes them; more than 64 sequences."""
    print(f"[gpu] prefix, many rows {dtype} fp8 {eight}", flush=True)
    own = [1 + (7 * i) % 90 for i in range(150)]
    Batch([(900, 150)], own, [1] * 150, 32, 8, 64, page, dtype, fp8_cache=eight, seed=4, cu=False).check(dev)
    new = [1 + i % 6 for i in range(90)]
    own = [n + (5 * i) % 40 for i, n in enumerate(new)]
    Batch([(333, 40), (700, 50)], own, new, 32, 8, 64, page, dtype, fp8_cache=eight, seed=5).check(dev)
    # rows enough that sequences' own part is tiles of 128 too
    new = [8 + i for i in range(40)]
    Batch([(450, 30), (77, 10)], [n + 3 * (i % 9) for i, n in enumerate(new)], new, 32, 8, 64, page, dtype,
          fp8_cache=eight, seed=6).check(dev)
    # and so many that every sequence is attended whole
    new = [64 + i for i in range(20)]
    Batch([(450, 20)], [n + 3 * i for i, n in enumerate(new)], new, 32, 8, 64, page, dtype, fp8_cache=eight,
          seed=6).check(dev)


@pytest.mark.parametrize("groups", [62, 63, 64, 65, 130])
def test_as_many_groups_as_lanes_and_more(dev, groups):
    print(f"[gpu] prefix, {groups} groups", flush=True)
    sizes = [(64 * (i % 4) + i % 7, 1 + i % 3) for i in range(groups)]
    n = sum(c for _, c in sizes) + 3
    own = [1 + i % 11 for i in range(n)]
    for cu in (False, True):
        new = [1 + i % 3 if cu else 1 for i in range(n)]
        Batch(sizes, [o + x for o, x in zip(own, new)], new, 4, 2, 64, 16, torch.bfloat16, seed=groups, cu=cu, loose=3).check(dev)


def test_heads_of_32_channels(dev):
    for dtype in (torch.float32, torch.bfloat16):
        Batch([(150, 3), (64, 2)], [4, 5, 1, 70, 2], [1, 2, 1, 5, 1], 6, 2, 32, 8, dtype, seed=7).check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_inside_the_prefix(dev, dtype):
    """A sequence shorter than its group's prefix sees what it holds, as without the
    group; in both forms of the shared part."""
    print(f"[gpu] prefix, inside {dtype}", flush=True)
    for seqs, heads in ((6, (8, 2)), (80, (32, 8))):
        own = [[-100, 3, -650, 1, -699, 20][i % 6] for i in range(seqs)]
        b = Batch([(700, seqs)], own, [[5, 1, 3, 1, 1, 2][i % 6] for i in range(seqs)], *heads, 64, 16, dtype, seed=8)
        b.check(dev)
        b.table[1::6, 3] = -1  # (copies may differ in nothing, so the hole is everywhere)
        b.table[:, 3] = -1
        b.check(dev)


@pytest.mark.parametrize("dtype,eight", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_what_rows_do_not_see(dev, dtype, eight):
    """NaN at a position of the prefix that a shorter sequence does not hold stays away
    from its rows, and reaches the others'."""
    print(f"[gpu] prefix, not seen {dtype} fp8 {eight}", flush=True)
    for seqs, heads in ((4, (8, 2)), (80, (32, 8))):
        own = [-200 if i % 2 else 5 for i in range(seqs)]
        b = Batch([(512, seqs)], own, [1] * seqs, *heads, 64, 16, dtype, fp8_cache=eight, seed=9, cu=False)
        clean, lse0 = b.attend(dev)
        page, row = int(b.table[0, 400 // 16]), 400 % 16
        b.v.view(torch.uint8 if eight else dtype)[page, row, 0, 3] = 0x7f if eight else math.nan
        o, lse = b.attend(dev)
        group = heads[0] // heads[1]
        assert torch.equal(o[1::2], clean[1::2]) and torch.equal(lse, lse0)
        assert torch.isnan(o[::2, :group, 3]).all()
        keep = [c for c in range(64) if c != 3]
        assert torch.equal(o[::2][..., keep], clean[::2][..., keep])
        if not eight:
            b.v[page, row, 0, 3] = math.inf
            b.k[page, row, 0, 7] = math.nan
            o, lse = b.attend(dev)
            assert torch.equal(o[1::2], clean[1::2]) and torch.isnan(o[::2, :group]).all()


def test_groups_that_cannot_be_stay_inside(dev):
    print("[gpu] prefix, malformed", flush=True)
    b = Batch([(100, 3), (60, 3)], [4, 5, 6, 7, 8, 9], [1, 2, 3, 1, 2, 3], 4, 2, 64, 8, torch.bfloat16, seed=10, garbage=0.0)
    from delta_feedback_experiment_amd import paged_prefix_attention

    args, more = b.args(dev)
    i32 = dict(dtype=torch.int32, device=dev)
    for groups in ([0, 3, 900], [0, 5, 2], [4, 3, 6], [-5, 2 ** 31 - 1, 6]):
        for prefix in ([100, 60], [2 ** 31 - 1, -3]):
            for cu in ([0, 1, 3, 6, 7, 9, 12], [0, 12, 3, 3, 900, -1, 12]):
                args[5], args[6] = torch.tensor(groups, **i32), torch.tensor(prefix, **i32)
                more["cu_seqlens"] = torch.tensor(cu, **i32)
                paged_prefix_attention(*args, **more)
                torch.cuda.synchronize()


def test_no_groups_no_tokens(dev):
    from delta_feedback_experiment_amd import paged_attention, paged_prefix_attention

    b = Batch([], [5, 70, 1], [1, 1, 1], 4, 2, 64, 16, torch.float32, seed=11, cu=False, loose=3)
    o, lse = b.check(dev)
    args, more = b.args(dev)
    plain = paged_attention(*args[:5])
    assert rel_l2(o, plain[0]) < 2 * TOL[torch.float32]
    args[0] = args[0][:0]
    args[3], args[4] = args[3][:0], args[4][:0]
    o, lse = paged_prefix_attention(*args, **more)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_checks_of_groups(dev):
    b = Batch([(100, 2), (60, 1)], [4, 5, 6], [1, 1, 1], 4, 2, 64, 8, torch.bfloat16, seed=12, cu=False)
    b.check(dev, check_pages=True)
    for groups, prefix in (([0, 2, 4], [100, 60]), ([0, 2, 1], [100, 60]), ([1, 2, 3], [100, 60]), ([0, 2, 3], [105, 60]),
                           ([0, 2, 3], [100, -1])):
        b.groups, b.prefix = (torch.tensor(x, dtype=torch.int32) for x in (groups, prefix))
        with pytest.raises(ValueError, match="cu_groups|prefix_lens"):
            b.attend(dev, check_pages=True)


def test_repeats_streams_and_graph(dev):
    """The same bits repeated, on another stream, and replayed with other groups,
    prefixes and work between."""
    from delta_feedback_experiment_amd import paged_prefix_attention

    print("[gpu] prefix, repeats", flush=True)
    for seqs, cu in ((9, False), (80, True)):
        b = Batch([(300, seqs)], [5 + i for i in range(seqs)], [1 + i % 3 if cu else 1 for i in range(seqs)], 16, 4, 64, 16,
                  torch.bfloat16, seed=13, cu=cu)
        args, more = b.args(dev)

        def step():
            return paged_prefix_attention(*args, **more)

        first = [t.clone() for t in step()]
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(first, step()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) for x, y in zip(first, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i, prefix in enumerate((300, 128, 64, 0, 299)):
            args[0].normal_()
            args[6].fill_(prefix)
            args[5][1:].fill_(seqs - i)
            eager = [t.clone() for t in step()]
            out[0].fill_(float(i))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager)), i
            b.q, b.prefix[:] = args[0].cpu(), prefix
            ro, _ = b.reference()
            assert rel_l2(out[0].float(), ro) < TOL[torch.bfloat16]


def test_opcheck_and_compile(dev):
    from delta_feedback_experiment_amd import paged_prefix_attention

    print("[gpu] prefix, opcheck and compile", flush=True)
    b = Batch([(100, 2), (60, 1)], [4, 5, 6], [2, 1, 6], 4, 2, 64, 8, torch.bfloat16, seed=14, garbage=0.5)
    args, more = b.args(dev)
    torch.library.opcheck(torch.ops.pkda_mi355x.paged_prefix_attention.default,
                          (*args[:3], None, None, *args[3:], more["cu_seqlens"], 0.125),
                          test_utils=("test_schema", "test_faketensor"))

    def step(q):
        return paged_prefix_attention(q * 1.0, *args[1:], **more)

    for a, c in zip(step(args[0]), torch.compile(step, fullgraph=True, backend="aot_eager")(args[0])):
        assert torch.equal(a, c)
