"""The paged cache of 8-bit floats on the GPU, and heads' norms in both appends,
against the 64-bit oracle.

Bars, from the arithmetic:

* values are quantised from what they are, exactly: codes and scales are equal;
* a head's norm: 16 squares and their sum in turn, three sums over lanes, the
  mean, a square root, a division and two products, each rounded once: at most
  half of 21 and 5 roundings of 2^-24 relative, under 2^-20; the rotation adds
  two products and a sum: together under 2^-19 of the pair's magnitudes, so 2^-18
  of the head's largest normed number.  What is rounded to the type, to a scale or
  to a code lies between the roundings of the exact number less and plus that;
* attention: the cache's numbers are operands as they are, so the bars are those of
  the same operator over a cache of the activations' type (FP32 1e-5, BF16 2^-8,
  relative L2; lse 1e-5 (1 + |lse|)).
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import rel_l2
from oracle import paged_fp8_oracle as fp8
from oracle import paged_oracle as oracle
from test_gpu_paged import RAGGED, TOL, Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


def codes_of(x):
    """Codes and scales of a pool, what is not a number among it."""
    c, s = fp8.quantised(x)
    return c.to(torch.float32).to(torch.float8_e4m3fn), s.to(torch.float32).to(torch.float8_e8m0fnu)


class Cache8(Cache):
    """A used cache of 8-bit floats."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        k, v = self.k_pages.float(), self.v_pages.float()
        # magnitudes all over, so that every block has a scale of its own
        gen = torch.Generator().manual_seed(99)
        self.pools = []
        for x in (k, v):
            power = torch.randint(-3, 4, (*x.shape[:3], x.shape[3] // 32), generator=gen)
            self.pools.append(codes_of(torch.ldexp(x, power.repeat_interleave(32, -1))))
        self.refresh()

    def refresh(self):
        (kc, ks), (vc, vs) = self.pools
        self.k_values, self.v_values = fp8.values(kc, ks), fp8.values(vc, vs)

    def cache(self, dev):
        (kc, ks), (vc, vs) = self.pools
        return [t.to(dev) for t in (kc, vc, ks, vs)]

    def attend(self, dev, **kw):
        from delta_feedback_experiment_amd import paged_attention_fp8

        table, lens, cu = self.tables(dev)
        out = paged_attention_fp8(self.q.to(dev), *self.cache(dev), table, lens, cu_seqlens=cu, **kw)
        torch.cuda.synchronize()
        return out

    def check(self, dev, long=False, **kw):
        o, lse = self.attend(dev, **kw)
        of = oracle.attention_of_sequences if long else oracle.attention_reference
        cu = torch.arange(len(self.lens) + 1, dtype=torch.int32) if long and self.cu is None else self.cu
        k, v = self.k_values, self.v_values
        if long:  # its sums run over every row of the tile
            k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
        ro, rl = of(self.q, k, v, self.table, self.lens, cu, **kw)
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


def slots(c, at, R):
    """(token, page, row) of the tokens that are stored."""
    for t, where in enumerate(at):
        if where is not None and 0 <= int(c.table[where[0], where[1] // R]) < c.pages:
            yield t, int(c.table[where[0], where[1] // R]), where[1] % R


NORMS = [(8, 2, 128, 16, 128, False, "both"), (8, 2, 128, 16, 128, True, "both"), (5, 5, 64, 24, 32, False, "k"),
         (3, 1, 64, 8, 16, True, "q"), (40, 8, 128, 64, 64, False, "both"), (9, 3, 64, 1, 0, False, "both"),
         (4, 2, 128, 7, 96, False, "none"), (4, 2, 128, 16, 0, False, "none")]


def placed_case(Hq, Hkv, D, page, rotary, norms, dtype, norm_dtype, dev):
    c = Cache([0, 1, 16, 33, 64, 65, 130, 3], [0, 1, 1, 33, 2, 5, 64, 5], Hq, Hkv, D, page, dtype, seed=21, garbage=0.5,
              tail=3)
    c.table[5, 0] = -1 if page > 60 else c.table[5, 0]
    gen = torch.Generator().manual_seed(22)
    weights = [(1 + 0.3 * torch.randn(D, generator=gen)).to(norm_dtype) if norms in ("both", n) else None for n in "qk"]
    angle = torch.rand(c.table.shape[1] * page, max(rotary, 16) // 2, generator=gen) * 6.28
    cos, sin = (angle.cos(), angle.sin()) if rotary else (None, None)
    c.k[3, 0] *= 1e-4   # a head whose eps counts
    c.q[2, -1] = 0
    packed = torch.cat((c.q, c.k, c.v), 1).flatten(1).to(dev)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in packed.split((Hq * D, Hkv * D, Hkv * D), -1))
    on = [None if t is None else t.to(dev) for t in (*weights, cos, sin)]
    more = dict(q_norm=on[0], k_norm=on[1], cos=on[2], sin=on[3], eps=1e-5)
    ref = [fp8.placed(x, c.lens, c.cu, w, 1e-5, cos, sin) for x, w in ((c.q, weights[0]), (c.k, weights[1]))]
    return c, (q, k, v), weights, cos, sin, more, ref


def near(x, weight, eps=1e-5):
    """What the bars allow a head's numbers to be off."""
    return 2.0 ** -18 * fp8.normed(x, weight, eps).abs().amax(-1, keepdim=True)


@pytest.mark.parametrize("dtype,norm_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                              (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("Hq,Hkv,D,page,rotary,interleaved,norms", NORMS)
def test_append_fp8_against_the_oracle(dev, dtype, norm_dtype, Hq, Hkv, D, page, rotary, interleaved, norms):
    from delta_feedback_experiment_amd import PagedKVFP8, paged_append_fp8_

    print(f"[gpu] append fp8 {dtype} {Hq}/{Hkv} x {D} rotary {rotary} norms {norms}", flush=True)
    c, (q, k, v), weights, cos, sin, more, _ = placed_case(Hq, Hkv, D, page, rotary, norms, dtype, norm_dtype, dev)
    kv = PagedKVFP8.zeros(c.pages, page, Hkv, D)
    table, lens, cu = c.tables(dev)
    out = paged_append_fp8_(k, v, kv.k, kv.v, kv.k_scale, kv.v_scale, table, lens, cu_seqlens=cu, q=q,
                            interleaved=interleaved, **more)
    torch.cuda.synchronize()
    rq, at = fp8.placed(c.q, c.lens, c.cu, weights[0], 1e-5, cos, sin, interleaved)
    rk, _ = fp8.placed(c.k, c.lens, c.cu, weights[1], 1e-5, cos, sin, interleaved)
    e = near(c.q, weights[0])
    assert out.dtype == dtype
    assert ((out.cpu() >= (rq - e).to(dtype)) & (out.cpu() <= (rq + e).to(dtype))).all()
    kc, ks, vc, vs = (t.cpu().float().double() for t in (kv.k, kv.k_scale, kv.v, kv.v_scale))
    e = near(c.k, weights[1])
    stored = torch.zeros(c.pages, page, dtype=torch.bool)
    for t, p, r in slots(c, at, page):
        stored[p, r] = True
        codes, scales = fp8.quantised(c.v[t])
        assert torch.equal(vc[p, r], codes) and torch.equal(vs[p, r], scales), t
        lo, hi = rk[t].abs() - e[t], rk[t].abs() + e[t]
        assert (ks[p, r] >= fp8.block_scales(lo.clamp(min=0))).all() and (ks[p, r] <= fp8.block_scales(hi)).all(), t
        lo, _ = fp8.quantised(rk[t] - e[t], ks[p, r])
        hi, _ = fp8.quantised(rk[t] + e[t], ks[p, r])
        assert ((kc[p, r] >= lo) & (kc[p, r] <= hi)).all(), t
    assert (kc[~stored] == 0).all() and (vc[~stored] == 0).all()
    assert (ks[~stored] == 1).all() and (vs[~stored] == 1).all()
    # without queries: the same cache
    kv2 = PagedKVFP8.zeros(c.pages, page, Hkv, D)
    more["q_norm"] = None
    assert paged_append_fp8_(k, v, kv2.k, kv2.v, kv2.k_scale, kv2.v_scale, table, lens, cu_seqlens=cu,
                             interleaved=interleaved, **more) is None
    for a, b in ((kv.k, kv2.k), (kv.v, kv2.v), (kv.k_scale, kv2.k_scale), (kv.v_scale, kv2.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype,norm_dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("Hq,Hkv,D,page,rotary,interleaved,norms",
                         NORMS[:6] + [(4, 2, 32, 16, 32, False, "both"), (4, 4, 32, 8, 16, True, "k")])
def test_append_with_norms_against_the_oracle(dev, dtype, norm_dtype, Hq, Hkv, D, page, rotary, interleaved, norms):
    from delta_feedback_experiment_amd import paged_append_

    print(f"[gpu] append with norms {dtype} {Hq}/{Hkv} x {D} rotary {rotary} norms {norms}", flush=True)
    c, (q, k, v), weights, cos, sin, more, _ = placed_case(Hq, Hkv, D, page, rotary, norms, dtype, norm_dtype, dev)
    table, lens, cu = c.tables(dev)
    kp, vp = c.k_pages.to(dev), c.v_pages.to(dev)
    out = paged_append_(k, v, kp, vp, table, lens, cu_seqlens=cu, q=q, interleaved=interleaved, **more)
    torch.cuda.synchronize()
    rq, at = fp8.placed(c.q, c.lens, c.cu, weights[0], 1e-5, cos, sin, interleaved)
    rk, _ = fp8.placed(c.k, c.lens, c.cu, weights[1], 1e-5, cos, sin, interleaved)
    ek, ev, slack = c.k_pages.double(), c.v_pages.double(), torch.zeros(c.pages, page, Hkv, 1, dtype=torch.float64)
    e = near(c.k, weights[1])
    for t, p, r in slots(c, at, page):
        ek[p, r], ev[p, r], slack[p, r] = rk[t], c.v[t].double(), e[t]
    assert torch.equal(vp.cpu().double(), ev)
    for got, ref, off in ((out, rq, near(c.q, weights[0])), (kp, ek, slack)):
        assert ((got.cpu() >= (ref - off).to(dtype)) & (got.cpu() <= (ref + off).to(dtype))).all()


def test_blocks_at_the_edges(dev):
    """Zeros, the smallest and largest numbers, magnitudes at a scale's border, codes'
    ties, NaN and infinities: codes and scales as the definition has them."""
    from delta_feedback_experiment_amd import PagedKVFP8, paged_append_fp8_

    print("[gpu] append fp8, edges", flush=True)
    big = torch.finfo(torch.float32).max
    rows = [torch.zeros(64), torch.full((64,), 1e-45), torch.full((64,), 2.0 ** -126), torch.full((64,), big),
            torch.linspace(-448, 448, 64), torch.linspace(-448.00003, 448.00003, 64), torch.linspace(0, 1, 64) * 2.0 ** -120,
            torch.tensor([448.0, 17, 19, 21, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9 * 2.5, 432, 1, 1.0625, 1.1875] + [0.0] * 53),
            torch.tensor([math.nan, 1, 2, 3] + [0.5] * 60), torch.tensor([math.inf, 1, -math.inf, 3] + [0.5] * 60),
            torch.full((64,), math.nan), torch.full((64,), math.inf), torch.tensor([-0.0, 7.0] * 32),
            torch.tensor([1.75 * 2.0 ** 127, big, -big, 1.8125 * 2.0 ** 127] * 16)]
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.stack(rows).to(dtype)[:, None]  # [N, 1, 64]
        N = x.shape[0]
        kv = PagedKVFP8.zeros(1, N, 1, 64)
        table, lens = (torch.tensor(t, dtype=torch.int32, device=dev) for t in ([[0]], [N]))
        cu = torch.tensor([0, N], dtype=torch.int32, device=dev)
        paged_append_fp8_(x.to(dev), x.flip(2).to(dev), kv.k, kv.v, kv.k_scale, kv.v_scale, table, lens, cu_seqlens=cu)
        torch.cuda.synchronize()
        for got, scale, ref in ((kv.k, kv.k_scale, x), (kv.v, kv.v_scale, x.flip(2))):
            codes, scales = fp8.quantised(ref.float())
            got, scale = got[0].cpu().float().double(), scale[0].cpu().float().double()
            assert torch.equal(scale, scales)
            assert torch.equal(torch.isnan(got), torch.isnan(codes))
            assert torch.equal(got.nan_to_num(9), codes.nan_to_num(9))
            assert torch.isfinite((got * scale.repeat_interleave(32, -1)).float().nan_to_num(0)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 64, 24), (5, 1, 128, 8), (16, 2, 128, 64), (3, 3, 64, 1), (40, 1, 64, 128),
                                           (4, 4, 128, 16)])
def test_attention_of_ragged_chunks(dev, dtype, Hq, Hkv, D, page):
    print(f"[gpu] fp8 attention {dtype} {Hq}/{Hkv} x {D}, pages of {page}", flush=True)
    Cache8(*RAGGED, Hq, Hkv, D, page, dtype, seed=D + page).check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 128, 16), (12, 2, 64, 24), (64, 1, 128, 64), (3, 1, 64, 5)])
def test_attention_of_single_tokens(dev, dtype, Hq, Hkv, D, page):
    """The decode form: no cu_seqlens; empty, short and longer sequences."""
    print(f"[gpu] fp8 decode {dtype} {Hq}/{Hkv} x {D}, pages of {page}", flush=True)
    lens = [0, 1, 2, 63, 64, 65, 511, 700, 1031]
    Cache8(lens, [1] * len(lens), Hq, Hkv, D, page, dtype, seed=D, cu=False).check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 13])
def test_attention_of_long_and_many(dev, dtype, page):
    """Split sequences; tiles of 128 rows, with pages that a wave's rows lie in and with others."""
    print(f"[gpu] fp8 attention, long {dtype}", flush=True)
    Cache8([4999], [1], 4, 1, 64, page, dtype, seed=1, cu=False).check(dev, long=True)
    Cache8([1999], [37], 4, 2, 128, page, dtype, seed=2).check(dev, long=True)
    Cache8([700, 1500], [1, 300], 2, 1, 128, page, dtype, seed=3).check(dev, long=True)
    # enough 128-row tiles that the card takes them
    Cache8([300 + 7 * i for i in range(40)], [60 + i for i in range(40)], 32, 8, 64, page, dtype, seed=4).check(dev, long=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,Hkv", [(130, 4), (64, 8), (512, 1), (513, 1), (65, 8)])
def test_single_tokens_of_many_sequences(dev, dtype, S, Hkv):
    """As many as the card takes the longest first of, and more; equal lengths and none
    among them."""
    print(f"[gpu] fp8 decode, {S} sequences of {Hkv} heads {dtype}", flush=True)
    gen = torch.Generator().manual_seed(S)
    lens = torch.randint(0, 90, (S,), generator=gen)
    lens[::5], lens[3::7], lens[-1] = 40, 0, 300
    Cache8(lens.tolist(), [1] * S, 2 * Hkv, Hkv, 64, 16, dtype, seed=S, cu=False).check(dev, long=True)
    Cache8([33] * S, [1] * S, 2 * Hkv, Hkv, 64, 16, dtype, seed=S, cu=False).check(dev, long=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_tokens_without_keys(dev, dtype):
    """Padding past cu_seqlens[-1], more new tokens than positions, missing pages."""
    print(f"[gpu] fp8 attention without keys {dtype}", flush=True)
    c = Cache8([7, 40, 3], [3, 40, 9], 8, 2, 64, 8, dtype, seed=4, tail=6)
    c.check(dev)
    c.table[1, 0], c.table[1, 2] = -1, c.pages
    c.check(dev)
    c.table[0, 0] = 2 ** 31 - 1
    c.check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_later_tokens_do_not_reach_earlier_ones(dev, dtype):
    """A later token's codes of NaN change no earlier token of its chunk; the row's own do."""
    print(f"[gpu] fp8 attention, later tokens {dtype}", flush=True)
    many = ([200 + i for i in range(40)], [64] * 40, 32, 8)
    for lens, new, Hq, Hkv in (([90], [60], 4, 2), ([200], [150], 16, 1), ([70, 33], [5, 33], 4, 4), many):
        c = Cache8(lens, new, Hq, Hkv, 64, 16, dtype, seed=5)
        clean, _ = c.attend(dev)
        at = lens[0] - 3
        page, row = int(c.table[0, at // 16]), at % 16
        for pool in c.pools:
            pool[0].view(torch.uint8)[page, row, 0, 5] = 0x7f
        o, _ = c.attend(dev)
        first = new[0] - 3
        assert torch.equal(o[:first], clean[:first])
        assert torch.equal(o[new[0]:], clean[new[0]:])
        assert torch.isnan(o[first:new[0], :Hq // Hkv]).all()
        assert torch.equal(o[first:new[0], Hq // Hkv:], clean[first:new[0], Hq // Hkv:])
        # the value alone: only its channel, and not the lse
        for pool, code in zip(c.pools, (0, 0xff)):
            pool[0].view(torch.uint8)[page, row, 0, 5] = code
        k_clean, lse0 = c.attend(dev)
        keep = [i for i in range(64) if i != 5]
        assert torch.isnan(k_clean[first:new[0], :Hq // Hkv, 5]).all()
        assert torch.isfinite(k_clean[first:new[0], :Hq // Hkv][..., keep]).all() and torch.isfinite(lse0).all()
        assert torch.equal(k_clean[:first], clean[:first])


def test_strides_offsets_and_what_is_not_held(dev):
    """Pages of codes and scales apart from each other, more than 2^32 bytes into the
    pool; garbage scales and codes where no sequence has a position."""
    from delta_feedback_experiment_amd import paged_append_fp8_, paged_attention_fp8

    print("[gpu] fp8 cache past 2^32 bytes", flush=True)
    H, D, page, N = 2, 64, 16, 21
    stride = 2 ** 32 + 2 ** 20  # bytes: page 1 begins past 2^32
    raw = [torch.empty(stride + page * H * D, dtype=torch.uint8, device=dev) for _ in range(2)]
    codes = [t.as_strided((2, page, H, D), (stride, H * D, D, 1)) for t in raw]
    both = torch.full((2, 2, page, H, D // 32), 255, dtype=torch.uint8, device=dev)
    scales = [both[:, i] for i in range(2)]
    for t in codes:
        t[0].fill_(0x7f), t[1].fill_(0x7f)
    pools = [t.view(torch.float8_e4m3fn) for t in codes] + [t.view(torch.float8_e8m0fnu) for t in scales]
    gen = torch.Generator().manual_seed(9)
    k, v = (torch.randn(N, H, D, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn(N, 4, D, generator=gen).bfloat16()
    table = torch.tensor([[1, 0, 7]], dtype=torch.int32)
    lens, cu = torch.tensor([N], dtype=torch.int32), torch.tensor([0, N], dtype=torch.int32)
    paged_append_fp8_(k.to(dev), v.to(dev), *pools, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev))
    assert (codes[0][0, 5:] == 0x7f).all() and (both[0, :, 5:] == 255).all()
    o, lse = paged_attention_fp8(q.to(dev), *pools, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev))
    kv, vv = (fp8.values(c.view(torch.float8_e4m3fn).cpu(), s.view(torch.float8_e8m0fnu).cpu())
              for c, s in zip(codes, scales))
    ro, rl = oracle.attention_reference(q, kv, vv, table, lens, cu)
    assert rel_l2(o.float(), ro) < TOL[torch.bfloat16] and float((lse.cpu() - rl).abs().max()) < 1e-5
    # scales of a page in part of a row's bytes: refused
    odd = torch.zeros(2 * page * H * 2 + 1, dtype=torch.uint8, device=dev)[1:].view(2, page, H, 2).view(torch.float8_e8m0fnu)
    with pytest.raises(ValueError, match="scales"):
        paged_attention_fp8(q.to(dev), pools[0], pools[1], odd, odd, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev))


def test_malformed_bounds_stay_inside(dev):
    from delta_feedback_experiment_amd import paged_append_fp8_, paged_attention_fp8

    print("[gpu] fp8 cache, malformed bounds", flush=True)
    c = Cache8([20, 30, 9], [4, 5, 6], 4, 2, 64, 8, torch.bfloat16, seed=10, garbage=0.0)
    table, pools = c.table.to(dev), c.cache(dev)
    weight = torch.ones(64, device=dev)
    for cu in ([0, 4, 9, 900], [0, 12, 3, 15], [3, 4, 9, 15], [-5, -4, 2 ** 31 - 1, 15]):
        for lens in ([20, 30, 9], [2 ** 31 - 1, -3, 9]):
            cu_t, lens_t = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (cu, lens))
            q = paged_append_fp8_(c.k.to(dev), c.v.to(dev), *pools, table, lens_t, cu_seqlens=cu_t, q=c.q.to(dev),
                                  q_norm=weight, k_norm=weight)
            paged_attention_fp8(q, *pools, table, lens_t, cu_seqlens=cu_t)
            torch.cuda.synchronize()


def test_repeats_streams_and_graph(dev):
    """The same bits repeated, on another stream, and replayed with other work between."""
    from delta_feedback_experiment_amd import paged_append_fp8_, paged_attention_fp8

    print("[gpu] fp8 cache, repeats", flush=True)
    for lens, new, cu in ((RAGGED[0], RAGGED[1], True), ([5, 900, 2000], [1, 1, 1], False)):
        c = Cache8(lens, new, 8, 2, 128, 16, torch.bfloat16, seed=11)
        table, lens_t, cu_t = c.tables(dev)
        cu_t = cu_t if cu else None
        q, k, v = (t.to(dev) for t in (c.q, c.k, c.v))
        pools = c.cache(dev)
        weight = torch.rand(128, device=dev) + 0.5

        def step():
            qr = paged_append_fp8_(k, v, *pools, table, lens_t, cu_seqlens=cu_t, q=q, q_norm=weight, k_norm=weight)
            return paged_attention_fp8(qr, *pools, table, lens_t, cu_seqlens=cu_t)

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


def test_no_sequences_and_no_pages(dev):
    from delta_feedback_experiment_amd import PagedKVFP8, paged_append_fp8_, paged_attention_fp8

    i32 = dict(dtype=torch.int32, device=dev)
    kv = PagedKVFP8.zeros(0, 16, 2, 64)
    pools = (kv.k, kv.v, kv.k_scale, kv.v_scale)
    empty = torch.zeros(0, 4, 64, device=dev)
    o, lse = paged_attention_fp8(empty, *pools, torch.zeros(0, 0, **i32), torch.zeros(0, **i32))
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    q, x = torch.randn(3, 4, 64, device=dev), torch.randn(3, 2, 64, device=dev)
    table, lens = torch.zeros(3, 0, **i32), torch.tensor([0, 5, 1], **i32)
    o, lse = paged_attention_fp8(q, *pools, table, lens)
    assert (o == 0).all() and torch.isneginf(lse).all()
    out = paged_append_fp8_(x, x, *pools, table, lens, q=q)
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_opcheck_and_compile(dev):
    """The schemas' marks match what the kernels write, the fake forms agree, and a
    compiled step gives the eager bits."""
    from delta_feedback_experiment_amd import paged_append_, paged_append_fp8_, paged_attention_fp8

    print("[gpu] fp8 cache, opcheck and compile", flush=True)
    c = Cache8([3, 9, 20], [2, 1, 20], 4, 2, 64, 8, torch.bfloat16, seed=18, garbage=0.5)
    table, lens, cu = c.tables(dev)
    q, k, v = (t.to(dev) for t in (c.q, c.k, c.v))
    angle = torch.rand(table.shape[1] * 8, 32, device=dev)
    weight = torch.rand(64, device=dev) + 0.5
    kp, vp = c.k_pages.to(dev), c.v_pages.to(dev)
    ops = torch.ops.pkda_mi355x
    torch.library.opcheck(ops.paged_store_.default, (k, v, kp, vp, None, None, table, lens, cu, q, angle.cos(), angle.sin(),
                                                     False, weight, None, 1e-6), test_utils=("test_schema", "test_faketensor"))
    # (the schema's check multiplies what it is given, which 8-bit floats cannot)
    torch.library.opcheck(ops.paged_attention_fp8.default, (q, *c.cache(dev), table, lens, cu, 0.125),
                          test_utils="test_faketensor")

    def step(q, k, v, kp, vp, *pools):
        paged_append_(k, v, kp, vp, table, lens, cu_seqlens=cu, k_norm=weight)
        q = paged_append_fp8_(k, v, *pools, table, lens, cu_seqlens=cu, q=q, cos=angle.cos(), sin=angle.sin(),
                              q_norm=weight, k_norm=weight)
        return paged_attention_fp8(q * 1.0, *pools, table, lens, cu_seqlens=cu)

    pools = [(kp.clone(), vp.clone(), *c.cache(dev)) for _ in range(2)]
    eager = step(q, k, v, *pools[0])
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, *pools[1])
    for a, b in zip((*eager, *pools[0]), (*compiled, *pools[1])):
        if a.element_size() == 1:
            a, b = a.view(torch.uint8), b.view(torch.uint8)
        assert torch.equal(a, b)


def test_version_counters_rise(dev):
    from delta_feedback_experiment_amd import PagedKVFP8, paged_append_, paged_append_fp8_

    i32 = dict(dtype=torch.int32, device=dev)
    kv = PagedKVFP8.zeros(2, 8, 2, 64)
    pools = (kv.k, kv.v, kv.k_scale, kv.v_scale)
    x, plain = torch.randn(2, 2, 64, device=dev), torch.zeros(2, 8, 2, 64, device=dev)
    table, lens = torch.tensor([[0], [1]], **i32), torch.tensor([1, 5], **i32)
    before = [t._version for t in (*pools, plain)]
    paged_append_fp8_(x, x, *pools, table, lens)
    paged_append_(x, x, plain, plain.clone(), table, lens, k_norm=torch.ones(64, device=dev))
    assert [t._version for t in (*pools, plain)] == [b + 1 for b in before]
