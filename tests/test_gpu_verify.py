"""Verification of drafted tokens on the GPU against the 64-bit definition.

Tokens and counts are whole numbers and have to be the definition's, but where two
sides of a comparison are nearer than what FP32 decides: a probability e^z / sum is
off by the rounding of z log2 e (|z| 2^-24 1.5, |z| up to some 60 here) and of a
sum, together under 2^-16 of its size, and a score log(p - q) by that times (p + q) /
(p - q).  How many rows were decided so is printed; it is next to none.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import verify_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


class Drafts:
    def __init__(self, rows, vocab, dtype, *, seed=0, tail=0, draft=True, near=0.7):
        gen = torch.Generator().manual_seed(seed)
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + r)
        N, S = cu[-1] + tail, len(rows)
        self.cu = torch.tensor(cu, dtype=torch.int32)
        self.logits = 3 * torch.randn(N, vocab, generator=gen)
        self.draft_logits = (self.logits + near * torch.randn(N, vocab, generator=gen)).to(dtype) if draft else None
        self.logits = self.logits.to(dtype)
        gumbel = -torch.empty(N, vocab).exponential_(generator=gen).log()
        base = self.draft_logits if draft else self.logits
        self.drafts = (base.float() + gumbel).argmax(-1).int()
        self.uniform = torch.rand(N, generator=gen)
        self.noise = -torch.empty(S, vocab).exponential_(generator=gen).log()
        self.temperature = 1.0

    def inputs(self):
        return (self.logits, self.drafts, self.uniform, self.noise, self.cu), dict(
            draft_logits=self.draft_logits, temperature=self.temperature)

    def run(self, dev):
        from delta_feedback_experiment_amd import verify_tokens

        args, more = self.inputs()
        out = verify_tokens(*(t.to(dev) for t in args),
                            **{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in more.items()})
        torch.cuda.synchronize()
        return out

    def check(self, dev):
        tokens, accepted = self.run(dev)
        assert tokens.dtype == accepted.dtype == torch.int32
        args, more = self.inputs()
        near = oracle.check(tokens.cpu(), accepted.cpu(), *args, **more)
        print(f"  accepted {accepted.float().mean() if accepted.numel() else 0:.2f} a sequence, {near} near", flush=True)
        return tokens, accepted


RAGGED = [1, 6, 0, 2, 9, 5, 3, 40, 1, 4]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 7, 513, 4096, 50304, 100001])
def test_against_the_definition(dev, dtype, draft, vocab):
    print(f"[gpu] verify {dtype} draft {draft} vocab {vocab}", flush=True)
    d = Drafts(RAGGED, vocab, dtype, seed=vocab, draft=draft, tail=3)
    d.check(dev)
    gen = torch.Generator().manual_seed(1)
    d.temperature = torch.rand(len(RAGGED), generator=gen) + 0.4
    d.temperature[::3] = 0
    d.temperature[4] = -1
    tokens, _ = d.check(dev)
    assert (tokens[-3:] == -1).all()


@pytest.mark.parametrize("seqs", [1, 200])
def test_few_and_many_sequences(dev, seqs):
    print(f"[gpu] verify {seqs} sequences", flush=True)
    Drafts([5] * seqs, 3001, torch.bfloat16, seed=seqs, near=0.3).check(dev)
    Drafts([2] * seqs, 3001, torch.float32, seed=seqs, near=0.1, draft=False).check(dev)


def test_all_accepted_and_none(dev):
    """Drafts of the target itself stand whatever the numbers; hopeless ones never."""
    d = Drafts([8] * 6, 1000, torch.bfloat16, seed=2)
    d.draft_logits = d.logits.clone()
    d.uniform[:] = 1 - 2.0 ** -24
    _, accepted = d.check(dev)
    assert (accepted == 7).all()
    d.uniform[:] = 0  # 0 < p: any draft that can be taken
    d.draft_logits = d.logits.roll(1, 1).clone()
    _, accepted = d.check(dev)
    assert (accepted == 7).all()
    d.logits.scatter_(1, d.drafts[:, None].long(), -torch.inf)
    _, accepted = d.check(dev)
    assert (accepted == 0).all()


def test_infinities_and_nan(dev):
    """Cut logits, rows with nothing, NaN, +inf, in target and draft."""
    for dtype in (torch.float32, torch.bfloat16):
        print(f"[gpu] verify, not finite {dtype}", flush=True)
        for draft in (True, False):
            d = Drafts([4] * 12, 2000, dtype, seed=3, draft=draft)
            d.logits[:, 100:1900] = -torch.inf            # a cut
            d.logits[5], d.logits[8] = -torch.inf, math.nan   # nothing
            d.logits[13, 7] = math.nan
            d.logits[16:24, 30] = math.inf                 # one for all
            d.logits[20:24, 60] = math.inf
            d.drafts[17], d.drafts[21] = 30, 60
            d.drafts[24], d.drafts[28], d.drafts[32] = -1, 2000, 2 ** 31 - 1
            if draft:
                d.draft_logits[1] = -torch.inf
                d.draft_logits[36] = math.nan
                d.draft_logits[41, 3] = math.inf
            d.check(dev)
            d.temperature = 0.0
            d.check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draft", [True, False])
def test_a_draft_at_an_infinite_logit(dev, dtype, draft):
    """Several +inf share a row's probability evenly, the draft's among them."""
    for temperature in (1.0, 0.3):
        d = Drafts([2] * 40, 777, dtype, seed=31, draft=draft)
        d.temperature = temperature
        d.logits[:, 30] = d.logits[:, 60] = math.inf  # p = 1/2
        d.drafts[:] = 30
        d.uniform[::2] = torch.linspace(0.02, 0.98, 40)
        if draft:
            d.draft_logits[:, 30] = math.inf  # q = 1, or 1/4: accepted whatever the number
            d.draft_logits[40:, [1, 2, 700]] = math.inf
        print(f"[gpu] verify, drafts at +inf, T {temperature}", flush=True)
        _, accepted = d.check(dev)
        stands = (d.uniform[::2] < 0.5).int()
        if draft:
            stands[20:] = 1
        assert torch.equal(accepted.cpu(), stands)


@pytest.mark.parametrize("temperature", [math.inf, 1e-6, 1e-38, 1e-45, 30.0])
def test_temperatures(dev, temperature):
    print(f"[gpu] verify, temperature {temperature}", flush=True)
    for draft in (True, False):
        d = Drafts([3] * 8, 700, torch.float32, seed=4, draft=draft)
        d.logits[2, 5:] = -torch.inf
        d.temperature = temperature
        if temperature >= 1:
            d.check(dev)
            continue
        # cold: the largest logit alone
        tokens, accepted = d.run(dev)
        for n in range(8):
            a = int(accepted[n])
            assert int(tokens[3 * n + a]) == int(d.logits[3 * n + a].argmax())
            for j in range(2):
                best = int(d.drafts[3 * n + j]) == int(d.logits[3 * n + j].argmax())
                assert (j < a) <= best


def test_ties_take_the_lowest_index(dev):
    for dtype in (torch.float32, torch.bfloat16):
        d = Drafts([2] * 4, 9001, dtype, seed=5, draft=False)
        d.logits[:] = 1.0
        d.noise[:] = 0.25
        d.uniform[:] = 0.5        # p of a draft is 1/9001: none stands
        d.drafts[0] = 0           # its place is left out
        d.drafts[2], d.drafts[4], d.drafts[6] = 17, 9000, 1
        tokens, accepted = d.run(dev)
        assert accepted.tolist() == [0] * 4 and tokens[::2].tolist() == [1, 0, 0, 0]
        d.temperature = 0.0
        tokens, accepted = d.run(dev)
        assert accepted.tolist() == [1, 0, 0, 0] and tokens.tolist() == [0, 0, 0, -1, 0, -1, 0, -1]
        d.noise[:] = math.inf
        d.temperature = 1.0
        assert d.run(dev)[0][::2].tolist() == [1, 0, 0, 0]
        d.noise[:] = -math.inf
        assert d.run(dev)[0][::2].tolist() == [1, 0, 0, 0]


def test_nothing_left_is_the_target(dev):
    """p <= q everywhere and still not accepted, by a uniform number of 1: p itself."""
    d = Drafts([2] * 3, 5000, torch.float32, seed=6)
    d.draft_logits = d.logits.clone()
    d.uniform[:] = 1.0
    tokens, accepted = d.run(dev)
    assert (accepted == 0).all()
    for n in range(3):
        assert int(tokens[2 * n]) == int((d.logits[2 * n] + d.noise[n]).argmax())
    # the same without draft logits: the draft has all of p
    d.draft_logits = None
    d.logits[:] = -torch.inf
    d.logits[:, 77] = 1.0
    d.drafts[:] = 77
    tokens, accepted = d.run(dev)
    assert (accepted == 0).all() and tokens[::2].tolist() == [77] * 3


def test_strides_and_offsets(dev):
    """Rows any distance apart that begin anywhere; other orders are copied."""
    from delta_feedback_experiment_amd import verify_tokens

    for dtype in (torch.float32, torch.bfloat16):
        d = Drafts(RAGGED, 777, dtype, seed=7)
        plain = d.run(dev)
        args, more = d.inputs()
        N = d.logits.shape[0]
        wide = [torch.zeros(N * 1001 + 3, dtype=t.dtype, device=dev)[3:].view(N, 1001)[:, 5:782] for t in
                (d.logits, d.draft_logits)]
        for w, t in zip(wide, (d.logits, d.draft_logits)):
            w.copy_(t)
        noise = torch.zeros(len(RAGGED), 780, device=dev)[:, 1:778]
        noise.copy_(d.noise)
        uniform = torch.zeros(N, 2, device=dev)[:, 0]
        uniform.copy_(d.uniform)
        got = verify_tokens(wide[0], d.drafts.to(dev), uniform, noise, d.cu.to(dev), draft_logits=wide[1])
        assert all(torch.equal(a, b) for a, b in zip(got, plain))
        turned = d.logits.to(dev).t().contiguous().t()
        got = verify_tokens(turned, d.drafts.to(dev), uniform, noise.t().contiguous().t(), d.cu.to(dev),
                            draft_logits=wide[1])
        assert all(torch.equal(a, b) for a, b in zip(got, plain))


def test_offsets_past_32_bits(dev):
    """A row more than 2^32 bytes into the logits."""
    from delta_feedback_experiment_amd import verify_tokens

    print("[gpu] verify past 2^32 bytes", flush=True)
    d = Drafts([2], 600, torch.bfloat16, seed=8)
    plain = d.run(dev)
    stride = 2 ** 31 + 64
    big = torch.empty(stride + 600, dtype=torch.bfloat16, device=dev).as_strided((2, 600), (stride, 1))
    big.copy_(d.logits)
    got = verify_tokens(big, d.drafts.to(dev), d.uniform.to(dev), d.noise.to(dev), d.cu.to(dev),
                        draft_logits=d.draft_logits.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(got, plain))


def test_malformed_bounds_stay_inside(dev):
    from delta_feedback_experiment_amd import verify_tokens

    d = Drafts([3, 4, 5], 1000, torch.bfloat16, seed=9)
    args, more = d.inputs()
    on = [t.to(dev) for t in args]
    for cu in ([0, 3, 900, 12], [0, 8, 2, 12], [5, 3, 7, 12], [-4, -1, 2 ** 31 - 1, 12]):
        on[4] = torch.tensor(cu, dtype=torch.int32, device=dev)
        verify_tokens(*on, draft_logits=more["draft_logits"].to(dev))
        torch.cuda.synchronize()


def test_no_rows_and_no_sequences(dev):
    from delta_feedback_experiment_amd import verify_tokens

    i32 = dict(dtype=torch.int32, device=dev)
    z = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    tokens, accepted = verify_tokens(z(0, 5), torch.zeros(0, **i32), z(0), z(3, 5), torch.zeros(4, **i32))
    assert tokens.shape == (0,) and accepted.tolist() == [0, 0, 0]
    tokens, accepted = verify_tokens(z(2, 5), torch.zeros(2, **i32), z(2), z(0, 5), torch.zeros(1, **i32))
    assert tokens.tolist() == [-1, -1] and accepted.shape == (0,)
    tokens, accepted = verify_tokens(z(0, 5), torch.zeros(0, **i32), z(0), z(0, 5), torch.zeros(1, **i32))
    assert tokens.shape == accepted.shape == (0,)


def test_draws_are_the_target_s(dev):
    """Drafts and next token together are distributed as the target: 40,000 sequences of
    one draft, a chi-square over 12 tokens (11 degrees of freedom: over 40 has
    probability under 4e-5)."""
    from delta_feedback_experiment_amd import verify_tokens

    gen = torch.Generator(device=dev).manual_seed(10)
    S, V = 40000, 12
    l, ld = (1.5 * torch.randn(V, generator=gen, device=dev) for _ in range(2))
    gumbel = lambda *s: -torch.empty(*s, device=dev).exponential_(generator=gen).log()  # noqa: E731
    drafts = (ld + gumbel(S, V)).argmax(-1).int().repeat_interleave(2)
    logits, draft_logits = (t.expand(2 * S, V).contiguous() for t in (l, ld))
    cu = torch.arange(0, 2 * S + 1, 2, dtype=torch.int32, device=dev)
    uniform = torch.rand(2 * S, generator=gen, device=dev)
    tokens, accepted = verify_tokens(logits, drafts, uniform, gumbel(S, V), cu, draft_logits=draft_logits)
    seen = torch.bincount(tokens[::2].long(), minlength=V).double()
    want = torch.softmax(l.double(), 0) * S
    chi = float(((seen - want) ** 2 / want).sum())
    print(f"[gpu] verify draws: chi-square {chi:.1f}, accepted {accepted.float().mean():.3f}", flush=True)
    assert chi < 40
    # the token after an accepted draft is a draw too
    after = tokens[1::2][accepted == 1].long()
    want = torch.softmax(l.double(), 0) * after.numel()
    chi = float(((torch.bincount(after, minlength=V) - want) ** 2 / want).sum())
    assert chi < 40


def test_repeats_streams_and_graph(dev):
    from delta_feedback_experiment_amd import verify_tokens

    print("[gpu] verify, repeats", flush=True)
    d = Drafts(RAGGED, 30011, torch.bfloat16, seed=11)
    args, more = d.inputs()
    on = [t.to(dev) for t in args]
    heat = torch.full((len(RAGGED),), 0.8, device=dev)
    draft = more["draft_logits"].to(dev)

    def step():
        return verify_tokens(*on, draft_logits=draft, temperature=heat)

    first = [t.clone() for t in step()]
    for _ in range(5):
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
    for i in range(5):
        on[2].uniform_()
        on[3].exponential_().log_().neg_()
        heat.fill_([0.8, 0.0, 1.0, 1.3, 0.5][i])
        eager = [t.clone() for t in step()]
        out[0].fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_opcheck_and_compile(dev):
    from delta_feedback_experiment_amd import verify_tokens

    d = Drafts([3, 1, 4], 301, torch.bfloat16, seed=12)
    args, more = d.inputs()
    on = [t.to(dev) for t in args]
    draft, heat = more["draft_logits"].to(dev), torch.ones(3, device=dev)
    for other, t in ((draft, heat), (None, None)):
        torch.library.opcheck(torch.ops.pkda_mi355x.verify_tokens.default, (*on, other, t, 0.7),
                              test_utils=("test_schema", "test_faketensor"))

    def step(logits):
        return verify_tokens(logits * 1.0, *on[1:], draft_logits=draft, temperature=0.9)

    for a, b in zip(step(on[0]), torch.compile(step, fullgraph=True, backend="aot_eager")(on[0])):
        assert torch.equal(a, b)
