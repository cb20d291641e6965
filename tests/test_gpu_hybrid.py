"""The serving operators together: the example's trunk of PKDA and attention
layers generates with states and pages, eagerly and by graph.

Bars: in FP32 each of the four layers meets the framework's FP32 bar of 1e-5
(relative L2) in both forms, prompt and decode, and adds its error once to a
residual of comparable size; the logits of the two forms differ by less than
2 x 4 x 1e-5, and the bar is 1e-4.  A graph's replay gives the eager bits.
"""

from __future__ import annotations

import sys

import pytest
import torch

from conftest import ROOT, rel_l2

sys.path.insert(0, str(ROOT / "examples"))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    return torch.device("cuda:0")


def _server(dtype, seqs=5, seed=3, **settings):
    import hybrid_decode as ex

    sizes = ex.Sizes(heads=4, kv_heads=2, head_dim=64, vocab=517, slots=8, pages=64, page_size=8, max_pages=12,
                     dtype=dtype)
    server = ex.Server(ex.Trunk(sizes), seqs, seed=seed, **settings)
    gen = torch.Generator().manual_seed(seed)
    prompts = [torch.randint(0, 517, (n,), generator=gen).cuda() for n in (1, 8, 17, 33, 65)[:seqs]]
    return server, prompts


def test_generation_equals_the_whole_text(dev):
    """Prompts and then single tokens give the logits of the finished text as
    one prompt, and the tokens drawn along the way are in it."""
    print("[gpu] hybrid trunk, generation", flush=True)
    settings = dict(temperature=0.8, top_k=40, top_p=0.9)
    server, prompts = _server(torch.float32, **settings)
    logits = [[server.prefill(n, p)] for n, p in enumerate(prompts)]
    text = [[*p.tolist()] for p in prompts]
    for _ in range(20):
        for n, t in enumerate(server.tokens.tolist()):
            assert 0 <= t < 517
            text[n].append(t)
        got = server.step()
        for n in range(len(prompts)):
            logits[n].append(got[n:n + 1].clone())
    whole, _ = _server(torch.float32, **settings)
    for n, t in enumerate(text):
        ref = whole.prefill(n, torch.tensor(t).cuda())
        err = rel_l2(torch.cat(logits[n]), ref)
        print(f"  sequence {n}: {len(t)} tokens, {err:.2e}", flush=True)
        assert err < 1e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_graph_generates_what_eager_steps_do(dev, dtype):
    print(f"[gpu] hybrid trunk, graph {dtype}", flush=True)
    temperature = torch.tensor([0.0, 0.5, 1.0, 1.5, 1.0], device=dev)
    top_k = torch.tensor([0, 5, 0, 100, 1], dtype=torch.int32, device=dev)
    runs = []
    for graph in (False, True):
        server, prompts = _server(dtype, temperature=temperature, top_k=top_k, top_p=0.95, min_p=0.01)
        for n, p in enumerate(prompts):
            server.prefill(n, p)
        if graph:
            server.capture()
        out = []
        for _ in range(12):
            out.append((server.step().clone(), server.tokens.clone()))
            torch.cuda.synchronize()
        runs.append(out)
    for i, (eager, replay) in enumerate(zip(*runs)):
        assert torch.equal(eager[0], replay[0]) and torch.equal(eager[1], replay[1]), i


def test_pages_and_slots_run_out_with_an_error(dev):
    import hybrid_decode as ex

    server, prompts = _server(torch.bfloat16)
    with pytest.raises(RuntimeError, match="no pages"):
        server.prefill(0, torch.zeros(97, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError, match="slots"):
        ex.Server(server.trunk, 9)
