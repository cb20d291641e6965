"""Groups in which some sequences hold less than the prefix, on the GPU: the others
see all of it, whichever of the group's rows names its pages.

Bars: those of ``test_gpu_paged_prefix.py``.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import rel_l2
from test_gpu_paged import TOL
from test_gpu_paged_prefix import KINDS, Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


def batch(groups, own, new, *args, what="none", **kw):
    """Sequences of ``own[n]`` positions behind their group's prefix, or (below 0) so
    many short of it, whose rows of the table name only what they hold."""
    b = Batch(groups, [max(o, 1) for o in own], new, *args, **kw)
    for n, o in enumerate(own):
        b.lens[n] += o - max(o, 1)
    assert (b.lens >= 0).all()
    cut_rows(b, what)
    return b


def cut_rows(b, what):
    """Past its own length a sequence's row of the table names what is not its own."""
    for n, length in enumerate(b.lens.tolist()):
        held = -(-length // b.page)
        rest = b.table.shape[1] - held
        if what == "none":
            b.table[n, held:] = -1
        elif what == "outside":
            b.table[n, held:] = b.pages + 5 * torch.arange(rest, dtype=torch.int32)
        else:  # pages of others, in another order
            b.table[n, held:] = (torch.arange(rest) * 7 + n).int() % b.pages


# own positions behind a prefix of 300 (64-key tiles: 256 of them shared), first ones
# first: nothing, one position, part of the prefix, all of it, more
ORDERS = {"empty first": [-300, 5, 9, -300, 40, 1], "short first": [-299, -40, 3, 70, -300, 2],
          "the last alone": [-300, -300, -250, -20, -299, 6], "none holds it": [-60, -100, -299, -7, -300, -200],
          "just the shared part": [-300, -44, -45, -300, -299, -60]}


@pytest.mark.parametrize("what", ["none", "outside", "others"])
@pytest.mark.parametrize("order", list(ORDERS))
@pytest.mark.parametrize("dtype,eight", KINDS)
def test_sequences_shorter_than_the_prefix(dev, dtype, eight, order, what):
    print(f"[gpu] prefix, {order}, rows past them {what}, {dtype} fp8 {eight}", flush=True)
    own = ORDERS[order]
    for seqs, heads, page, cu in ((6, (8, 2), 16, False), (6, (8, 2), 24, True), (6, (48, 2), 16, True),
                                  (96, (32, 8), 16, True)):
        # (the many in the same order, each kind several times)
        extra = [own[i * 6 // seqs] for i in range(seqs)]
        new = [(1, 3, 2)[i % 3] if cu else 1 for i in range(seqs)]
        batch([(40, 2), (300, seqs)], [4, 9] + extra, [1, 1] + new, *heads, 64, page, dtype, fp8_cache=eight, seed=50, cu=cu,
              garbage=0.5, what=what).check(dev)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("holder", [0, 63, 64, 65, 128, 199])
def test_the_one_that_holds_it_is_found_anywhere(dev, eight, holder):
    """Of 200 sequences one holds the prefix and sees it; the others are finished."""
    print(f"[gpu] prefix, held by sequence {holder} fp8 {eight}", flush=True)
    for cu in (True, False):
        own = [3 if i == holder else -500 + i % 3 for i in range(200)]
        batch([(500, 200)], own, [1] * 200, 4, 1, 64, 16, torch.bfloat16, fp8_cache=eight, seed=51, cu=cu, garbage=0.5,
              what="others").check(dev)


def test_lengths_below_zero_count_as_none(dev):
    print("[gpu] prefix, lengths below zero", flush=True)
    b = batch([(300, 4)], [-300, 5, -300, 9], [1] * 4, 8, 2, 64, 16, torch.bfloat16, seed=52, cu=False)
    plain = b.check(dev)
    b.lens[0], b.lens[2] = -2 ** 31, -1
    got = b.attend(dev)
    assert all(torch.equal(x, y) for x, y in zip(plain, got))


@pytest.mark.parametrize("dtype,eight", KINDS)
def test_what_lies_past_the_holder_is_not_seen(dev, dtype, eight):
    """No sequence holds the whole prefix: NaN behind the longest reaches no row."""
    print(f"[gpu] prefix, past the longest {dtype} fp8 {eight}", flush=True)
    for seqs, heads in ((6, (8, 2)), (80, (32, 8))):
        own = [(-300, -130, -250, -77, -299, -130)[i % 6] for i in range(seqs)]
        batch([(300, seqs)], own, [1] * seqs, *heads, 64, 16, dtype, fp8_cache=eight, seed=53, cu=False, garbage=math.nan,
              what="others").check(dev)


@pytest.mark.parametrize("cu", [False, True])
def test_sequences_that_finish_between_replays(dev, cu):
    """A captured step follows lengths and tables: slots of a group finish, the first
    ones first, and are cleared."""
    from delta_feedback_experiment_amd import paged_prefix_attention

    print("[gpu] prefix, slots that finish", flush=True)
    b = Batch([(200, 5), (330, 70)], [2 + i % 40 for i in range(75)], [1] * 75, 8, 2, 64, 16, torch.bfloat16, seed=54, cu=cu)
    args, more = b.args(dev)
    graph = torch.cuda.CUDAGraph()
    paged_prefix_attention(*args, **more)
    with torch.cuda.graph(graph):
        out = paged_prefix_attention(*args, **more)
    for i, done in enumerate(([], [0], [0, 1, 5, 6, 7], list(range(3)) + list(range(5, 70)), list(range(75)))):
        b.lens[done] = 0
        b.table[done] = -1
        args[3].copy_(b.table)
        args[4].copy_(b.lens)
        args[0].normal_()
        eager = [t.clone() for t in paged_prefix_attention(*args, **more)]
        out[0].fill_(float(i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager)), i
        b.q = args[0].cpu()
        ro, rl = b.reference()
        assert torch.equal(torch.isinf(out[1].cpu()), torch.isinf(rl))
        assert (out[0].cpu()[torch.isinf(rl)] == 0).all()
        if len(done) < 75:
            assert rel_l2(out[0].float(), ro) < TOL[torch.bfloat16]


@pytest.mark.parametrize("dtype,eight", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_a_long_chunk_among_single_tokens(dev, dtype, eight):
    """One sequence prefills while the others of its group decode."""
    print(f"[gpu] prefix, a chunk among single tokens {dtype} fp8 {eight}", flush=True)
    new = [1] * 30
    new[11] = 1100
    own = [n + 3 * (i % 5) for i, n in enumerate(new)]
    Batch([(450, 20), (130, 10)], own, new, 32, 8, 64, 16, dtype, fp8_cache=eight, seed=55).check(dev)
