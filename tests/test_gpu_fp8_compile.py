"""The 8-bit cache's operators under the compiler's default backend, on the GPU:
outputs and the caches that are written in place are those of the eager call, bit
for bit."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged_fp8 import Cache8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_and_attention_compiled(dev, dtype):
    from delta_feedback_experiment_amd import paged_append_fp8_, paged_attention_fp8, paged_prefix_attention

    print(f"[gpu] fp8 cache, compiled {dtype}", flush=True)
    c = Cache8([20, 33, 9], [4, 5, 6], 8, 2, 128, 16, dtype, seed=61, garbage=0.5)
    table, lens, cu = c.tables(dev)
    q, k, v = (t.to(dev) for t in (c.q, c.k, c.v))
    weight = torch.rand(128, generator=torch.Generator().manual_seed(1)).to(dev) + 0.5
    groups, prefix = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 3], [0]))

    def step(q, k, v, *pools):
        for _ in range(2):  # (the second writes what the first wrote)
            qr = paged_append_fp8_(k, v, *pools, table, lens, cu_seqlens=cu, q=q * 1.0, q_norm=weight, k_norm=weight)
        o, lse = paged_attention_fp8(qr * 1.0, *pools, table, lens, cu_seqlens=cu)
        po, plse = paged_prefix_attention(qr, *pools[:2], table, lens, groups, prefix, k_scales=pools[2],
                                          v_scales=pools[3], cu_seqlens=cu)
        return qr, o, lse, po, plse

    torch._dynamo.reset()
    kept = [c.cache(dev) for _ in range(2)]
    eager = step(q, k, v, *kept[0])
    compiled = torch.compile(step, fullgraph=True)(q, k, v, *kept[1])
    before = c.cache(dev)
    for a, b, old in zip(*kept, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert not torch.equal(a.view(torch.uint8), old.view(torch.uint8))
    for a, b in zip(eager, compiled):
        assert torch.equal(a, b)
