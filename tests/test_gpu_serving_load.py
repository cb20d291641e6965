"""The operators of a loaded server together, as one would run them: sequences
behind a shared prompt, an 8-bit cache written with norms and rotation, several
drafted tokens a step, verified, the cache's lengths set back to what stood.

The model is one attention layer over tables: a token's q, k and v are rows of
random tables, so that what is stored does not depend on how many tokens a step
appends, and its logits a product of the attention's output.  Greedy drafts and
sampling must then give, token for token, what decoding one token at a time gives:
outputs of the two differ by the bars of attention (1e-5 each), and the test asserts
that the two largest logits are further apart than both.
"""

from __future__ import annotations

import pytest
import torch

from oracle import paged_fp8_oracle as fp8
from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


class Model:
    S, K, V, HQ, HKV, D, PAGE = 6, 3, 61, 8, 2, 64, 8

    def __init__(self, dev, eight: bool, prefix: int, steps: int):
        from delta_feedback_experiment_amd import PagedKV, PagedKVFP8

        gen = torch.Generator().manual_seed(31)
        S, V, D = self.S, self.V, self.D
        rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.dev, self.eight = dev, eight
        self.tq, self.tk, self.tv = (rand(V, h, D).to(dev) for h in (self.HQ, self.HKV, self.HKV))
        self.w = rand(self.HQ * D, V).to(dev)
        self.norms = [(1 + 0.2 * rand(D)).to(dev) for _ in range(2)]
        most = prefix + (self.K + 1) * (steps + 2)
        pages_each = -(-most // self.PAGE)
        angle = torch.outer(torch.arange(pages_each * self.PAGE), 100.0 ** (-torch.arange(0, D, 2) / D))
        self.cos, self.sin = angle.cos().to(dev), angle.sin().to(dev)
        shared = prefix // self.PAGE
        pages = shared + S * (pages_each - shared)
        order = torch.randperm(pages, generator=gen).int()
        self.table = torch.empty(S, pages_each, dtype=torch.int32)
        self.table[:, :shared] = order[:shared]
        self.table[:, shared:] = order[shared:].view(S, -1)
        self.table = self.table.to(dev)
        make = PagedKVFP8.zeros if eight else (lambda *a: PagedKV.zeros(*a, dtype=torch.float32))
        self.kv = make(pages, self.PAGE, self.HKV, D)
        self.prompt = torch.randint(0, V, (prefix,), generator=gen).to(dev)
        self.lens = torch.zeros(S, dtype=torch.int32, device=dev)
        self.groups = torch.tensor([0, S], dtype=torch.int32, device=dev)
        self.prefix = torch.zeros(1, dtype=torch.int32, device=dev)
        # the shared prompt: whole pages once, the rest into every sequence's own page
        self._append(self.prompt, self.table[:1], torch.tensor([prefix], dtype=torch.int32, device=dev),
                     torch.tensor([0, prefix], dtype=torch.int32, device=dev))
        rest = prefix - shared * self.PAGE
        if rest:
            full = torch.full((S,), prefix, dtype=torch.int32, device=dev)
            self._append(self.prompt[-rest:].repeat(S), self.table, full,
                         torch.arange(0, S * rest + 1, rest, dtype=torch.int32, device=dev))
        self.lens.fill_(prefix)
        self.prefix.fill_(prefix)

    def _append(self, tokens, table, lens, cu):
        from delta_feedback_experiment_amd import paged_append_, paged_append_fp8_

        more = dict(cu_seqlens=cu, q=self.tq[tokens], cos=self.cos, sin=self.sin, q_norm=self.norms[0], k_norm=self.norms[1])
        if self.eight:
            c = self.kv
            return paged_append_fp8_(self.tk[tokens], self.tv[tokens], c.k, c.v, c.k_scale, c.v_scale, table, lens, **more)
        return paged_append_(self.tk[tokens], self.tv[tokens], self.kv.k, self.kv.v, table, lens, **more)

    def logits(self, tokens, cu):
        """Of new tokens, which ``self.lens`` counts already."""
        from delta_feedback_experiment_amd import paged_prefix_attention

        q = self._append(tokens, self.table, self.lens, cu)
        c = self.kv
        scales = dict(k_scales=c.k_scale, v_scales=c.v_scale) if self.eight else {}
        o, _ = paged_prefix_attention(q, c.k, c.v, self.table, self.lens, self.groups, self.prefix, cu_seqlens=cu, **scales)
        return o.flatten(1) @ self.w


def first_tokens(m):
    return (torch.arange(m.S, device=m.dev) * 7 % m.V).int()


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("prefix", [100, 203])
def test_drafts_give_what_single_tokens_give(dev, eight, prefix):
    from delta_feedback_experiment_amd import sample_tokens, verify_tokens

    print(f"[gpu] serving load, fp8 {eight}, prefix {prefix}", flush=True)
    steps = 12
    # one token at a time
    m = Model(dev, eight, prefix, (steps + 1) * (Model.K + 1))
    last, text, gap = first_tokens(m), [], float("inf")
    zero = torch.zeros(m.S, m.V, device=dev)
    for _ in range((steps + 1) * (m.K + 1)):
        m.lens += 1
        logits = m.logits(last.long(), None)
        top = logits.topk(2, -1).values
        gap = min(gap, float(((top[:, 0] - top[:, 1]) / logits.abs().amax(-1)).min()))
        last, _ = sample_tokens(logits, zero, temperature=0.0)
        text.append(last.clone())
    text = torch.stack(text, 1).cpu()  # [S, tokens]
    # drafts: some right, some not, from the text itself; the step is a graph
    m = Model(dev, eight, prefix, (steps + 1) * (Model.K + 1))
    S, K = m.S, m.K
    cu = torch.arange(0, S * (K + 1) + 1, K + 1, dtype=torch.int32, device=dev)
    last = first_tokens(m)
    drafts = torch.zeros(S, K, dtype=torch.int32, device=dev)
    uniform = torch.rand(S * (K + 1), device=dev)
    ends = cu[:-1].long()
    tokens, accepted = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (S * (K + 1), S))

    def step():
        m.lens.add_(K + 1)
        new = torch.cat((last[:, None], drafts), 1).flatten()
        logits = m.logits(new.long(), cu)
        by_row = torch.cat((drafts, torch.full_like(drafts[:, :1], -1)), 1).flatten()
        t, a = verify_tokens(logits, by_row, uniform, zero, cu, temperature=0.0)
        tokens.copy_(t), accepted.copy_(a)
        m.lens.add_(a - K)  # what did not stand is written over by the next step
        last.copy_(t[ends + a.long()])

    kept = [t.clone() for t in (m.lens, last)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, old in zip((m.lens, last), kept):
        t.copy_(old)
    gen = torch.Generator().manual_seed(5)
    got = [[] for _ in range(S)]
    stood = 0
    for _ in range(steps):
        guess = torch.randint(0, m.V, (S, K), generator=gen).int()
        for s in range(S):
            right = int(torch.randint(0, K + 1, (1,), generator=gen))
            at = len(got[s])
            guess[s, :right] = text[s, at:at + right]
        drafts.copy_(guess)
        graph.replay()
        torch.cuda.synchronize()
        rows, count = tokens.cpu().view(S, K + 1), accepted.cpu()
        for s in range(S):
            a = int(count[s])
            assert (rows[s, a + 1:] == -1).all()
            got[s] += rows[s, :a + 1].tolist()
            stood += a
    assert gap > 2e-5
    print(f"  {stood} drafts stood; the nearest two logits were {gap:.1e} of the largest apart", flush=True)
    for s in range(S):
        assert got[s] == text[s, :len(got[s])].tolist(), s
        assert int(m.lens[s]) == prefix + len(got[s])


def test_the_cache_is_what_was_said(dev):
    """After drafts that did not stand, the cache's rows are those of the text alone,
    and attention over them is the oracle's."""
    from delta_feedback_experiment_amd import paged_prefix_attention

    m = Model(dev, True, 45, 8)
    S = m.S
    text = torch.randint(0, m.V, (S, 9), generator=torch.Generator().manual_seed(1)).to(dev)
    cu = lambda n: torch.arange(0, S * n + 1, n, dtype=torch.int32, device=dev)  # noqa: E731
    m.lens += 5
    m.logits(torch.cat((text[:, :2], text[:, 6:9] * 0), 1).flatten(), cu(5))  # two stand
    m.lens -= 3
    m.lens += 7
    q = m._append(text[:, 2:].flatten(), m.table, m.lens, cu(7))
    c = m.kv
    o, lse = paged_prefix_attention(q, c.k, c.v, m.table, m.lens, m.groups, m.prefix, k_scales=c.k_scale,
                                    v_scales=c.v_scale, cu_seqlens=cu(7))
    whole = torch.cat((m.prompt.repeat(S, 1), text), 1).cpu()
    n = whole.shape[1]
    lens, bounds = torch.full((S,), n, dtype=torch.int32), torch.arange(0, S * n + 1, n, dtype=torch.int32)
    k, v = (t.cpu()[whole.flatten()] for t in (m.tk, m.tv))
    place = dict(cos=m.cos.cpu(), sin=m.sin.cpu())
    rk, at = fp8.placed(k, lens, bounds, m.norms[1].cpu(), 1e-6, **place)
    kv, vv = (fp8.values(a.cpu(), b.cpu()) for a, b in ((c.k, c.k_scale), (c.v, c.v_scale)))
    table = m.table.cpu()
    for t, (s, p) in enumerate(at):
        page, row = int(table[s, p // m.PAGE]), p % m.PAGE
        # a code is within half a step of the number: 2^-4 of it, or 2^-10 of the block's scale
        for got, ref in ((kv[page, row], rk[t]), (vv[page, row], v[t].double())):
            off = torch.maximum(ref.abs() * 2.0 ** -4, fp8.block_scales(ref).repeat_interleave(32, -1) * 2.0 ** -9)
            assert ((got - ref).abs() <= off * (1 + 1e-4) + 1e-5).all(), (s, p)
    ro, rl = oracle.attention_of_sequences(q.cpu(), kv, vv, table, m.lens.cpu(), cu(7).cpu())
    assert float((o.cpu() - ro).norm() / ro.norm()) < 1e-5 and float((lse.cpu() - rl).abs().max()) < 1e-4
