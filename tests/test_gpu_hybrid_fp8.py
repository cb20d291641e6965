"""The example's trunk with head norms and a cache of 8-bit floats: a graph's replay
gives the eager bits, and generation stays by what a cache of the activations' type
gives as far as 8 bits go."""

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


def _server(dtype, **settings):
    import hybrid_decode as ex

    sizes = ex.Sizes(heads=4, kv_heads=2, head_dim=64, vocab=517, slots=8, pages=64, page_size=8, max_pages=12,
                     dtype=dtype, fp8=True)
    server = ex.Server(ex.Trunk(sizes), 5, seed=3, **settings)
    gen = torch.Generator().manual_seed(3)
    return server, [torch.randint(0, 517, (n,), generator=gen).cuda() for n in (1, 8, 17, 33, 65)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_graph_generates_what_eager_steps_do(dev, dtype):
    print(f"[gpu] hybrid trunk, 8-bit cache, graph {dtype}", flush=True)
    runs = []
    for graph in (False, True):
        server, prompts = _server(dtype, temperature=0.9, top_k=50, top_p=0.95)
        for n, p in enumerate(prompts):
            server.prefill(n, p)
        if graph:
            server.capture()
        out = []
        for _ in range(10):
            out.append((server.step().clone(), server.tokens.clone()))
            torch.cuda.synchronize()
        runs.append(out)
    for i, (eager, replay) in enumerate(zip(*runs)):
        assert torch.equal(eager[0], replay[0]) and torch.equal(eager[1], replay[1]), i
        assert torch.isfinite(eager[0]).all() and ((eager[1] >= 0) & (eager[1] < 517)).all()


def test_eight_bits_are_near_the_whole(dev):
    """One prompt over both kinds of cache, the same norms.  A code is off by at most
    2^-4 of its number, in the mean of squares 2^-4 / sqrt(3) of it over an evenly
    filled octave and less over one: keys and values so put at most 0.036 / ln 2 of
    relative error on a layer's output, two layers into a residual of comparable
    size; the bar is 0.1."""
    import hybrid_decode as ex
    from delta_feedback_experiment_amd import PagedKV, paged_append_, paged_attention

    server, prompts = _server(torch.float32)
    got = server.prefill(4, prompts[4])
    trunk = server.trunk
    s = trunk.s
    for w in trunk.layers:
        if "cache" in w:
            w["cache"] = PagedKV.zeros(s.pages, s.page_size, s.kv_heads, s.head_dim, dtype=s.dtype)

    def attention(w, h, table, lens, cu):
        q, k, v = (h @ w["qkv"]).unflatten(-1, (-1, s.head_dim)).split((s.heads, s.kv_heads, s.kv_heads), 1)
        c = w["cache"]
        q = paged_append_(k, v, c.k, c.v, table, lens, cu_seqlens=cu, q=q, cos=trunk.cos, sin=trunk.sin,
                          q_norm=w["norms"][0], k_norm=w["norms"][1])
        return paged_attention(q, c.k, c.v, table, lens, cu_seqlens=cu)[0].flatten(1)

    trunk._attention = attention
    ref = ex.Server(trunk, 5).prefill(4, prompts[4])
    err = rel_l2(got, ref)
    print(f"[gpu] hybrid trunk, 8-bit cache against whole: {err:.3f}", flush=True)
    assert 1e-4 < err < 0.1
