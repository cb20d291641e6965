"""PKDA recurrence benchmark on one MI355X.

    python bench.py [--gpus 1] [--steps K] [--warmup W] [--workload c2|c3|c5]
                    [--decode-steps 1000] [--no-decode] [--no-cpu] [--no-serve]

Mirrors the structure of the reference's ``scripts/pkda_bench.py`` (seeded
synthetic inputs, warm-up, event-timed repeats): one *step* is one forward +
backward of the chunked PKDA recurrence over one batch of the workload
(default ``c2``: B=8, T=4096, H=16, d=128, chunk 64, BF16 q/k/v, FP32 state,
per-head log-decay, returning dq, dk, dv, dbeta, dg).  Inputs are resident in
HBM before the timed region starts.

Printed as ONE JSON line:
  value           tokens/s of the whole fwd+bwd step: K steps between two
                  synchronised events, as K replays of the step captured in a
                  HIP graph or as K eager steps after W warm-up steps on the
                  warm GPU, whichever is faster (``timing`` names it; on this
                  ROCm a graph replay costs ~10 us per kernel over the same
                  launches issued eagerly, and the eager step's host work
                  stays behind the GPU's);
  roofline        the dominant kernel of the step, timed with HIP events on
                  the stream it runs on.  Both of its rates are measured --
                  algorithmic flops per launch (per token-head figures below)
                  against dense BF16 MFMA peak, and the HBM bytes the committed
                  PMC summary records per launch against 8 TB/s -- and
                  ``bound`` is the roof it runs closer to; ``achieved`` and
                  ``frac`` are against that roof (algorithmic bytes per launch
                  for an HBM-bound kernel), the other roof's figures, the
                  counter pass's MFMA busy share and the ratio of measured to
                  algorithmic bytes stay beside them;
  step_traffic    the PMC bytes of every kernel of one c2 step summed, against
                  the step's algorithmic 2,828 B per token-head;
  median_ms/min_ms  the median and fastest of the K replays (each between
                  its own events; value uses the K replays back to back);
  checks          before timing: every output and gradient finite, and two
                  backwards accumulated in FP32 and halved equal to one;
  agreement       before timing: the GPU step on a slice of the workload's
                  own inputs against the CPU oracle, relative L2 <= 2e-2 for
                  o and every gradient (a failed check exits non-zero);
  cpu_baseline    the CPU oracle (a restatement of the reference's portable
                  recurrence) timed on this host over a bounded sample, with
                  BASELINE configs 1 (whole forward) and 4 (decode steps);
  c3, c5          the packed-document and long-context workloads, timed as
                  the headline step;
  production      the reference model's own operator (pkda_recurrence: raw
                  per-channel gate, preconditioner, ten gradients) at the c2
                  geometry, checked (finite, FP32 accumulation; oracle
                  agreement on a slice in the CPU leg) and timed as HIP graph
                  replays;
  decode          the batched slot-pool decode step (B=256 live sequences in
                  a 512-slot [512, 32, 128, 128] FP32 pool, 1000 steps with
                  1000 distinct slot subsets), achieved HBM GB/s against 8 TB/s;
  qkv_conv        the recurrence's producer (fused Q/K/V short convolution +
                  SiLU + L2 norm), forward and backward at the screen
                  geometry, achieved HBM GB/s against 8 TB/s;
  norm_gate       its consumer (RMSNorm sigmoid output gate) on the c2
                  output shape, achieved HBM GB/s against 8 TB/s;
  controls        the control path at the c2 geometry: control activations
                  and their packed gradient, and the gate with the decay
                  expansion fused against the materialised form;
  serve           the slot-pool serving path: a cached prefill of the c2
                  shape into pool slots (tokens/s, MFMA fraction) and one
                  decode token of the convolution with slot histories
                  (achieved GB/s).

Algorithmic work per token-head (C = 64, dk = dv = d; the triangular solve,
gate scans and elementwise work are not counted).  The step's MFMA fraction
uses the fixed convention 18d^2 + 30Cd = 540,672 flop at d = 128 (the
forward as Akk, Aqk, w, u, Aqk U plus the three d^2 products, the backward
twice that); each kernel's figure below is the work it performs:
  fwd intra   4Cd           (Akk, Aqk)
  fwd state   6d^2 + 4Cd    (K S, Q S, Kg^T U; U = T Y, Aqk U)
  bwd state   6d^2 + 4Cd    (Kg dS, Qg^T dO, K^T (beta e^G dBv); dBv = T^T dU,
                             Aqk^T dO)
  bwd chunk   6d^2 + 16Cd   (dO S^T, dBv S^T, U dS^T; dO U^T, dBv U^T, dW-side
                             T^T terms; pairwise dq, dk, dkw products)
BF16 with a per-head gate never forms W = T diag(beta e^G) K or u: the state
passes contract with T instead (18d^2 + 28Cd performed in all), and the
reverse pass hands dBv = T^T dU to the per-chunk kernel.
"""

from __future__ import annotations

import argparse
import json
import math
import os
import sys
import time
from pathlib import Path

ROOT = Path(__file__).resolve().parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

import torch  # noqa: E402
import torch.nn.functional as F  # noqa: E402

MFMA_BF16_PEAK = 2.5e15  # dense bf16 MFMA, flop/s (MI355X published figure)
HBM_PEAK = 8.0e12        # bytes/s
CHUNK = 64

WORKLOADS = {
    "c2": dict(B=8, T=4096, H=16, D=128, strong=False, s0=False, varlen=False),
    "c3": dict(B=1, T=32768, H=16, D=128, strong=False, s0=False, varlen=True),
    "c5": dict(B=2, T=16384, H=32, D=128, strong=True, s0=True, varlen=False),
}


def stage_flops(D: int, C: int = CHUNK) -> dict[str, int]:
    """Algorithmic flops per token-head that each kernel of the step performs."""
    return {
        "fwd_intra": 4 * C * D,
        "fwd_state": 6 * D * D + 4 * C * D,
        "bwd_state": 6 * D * D + 4 * C * D,
        "bwd_chunk": 6 * D * D + 16 * C * D,
    }


def step_flops_convention(D: int, C: int = CHUNK) -> int:
    """The fixed algorithmic work of one fwd+bwd per token-head the MFMA
    fraction is quoted on: F_fwd = 6 dk dv + 2C (3 dk + 2 dv), total 3 F_fwd."""
    return 3 * (6 * D * D + 2 * C * (3 * D + 2 * D))


# The kernel each timed stage launches for the default BF16, d = 128 workloads,
# as rocprofv3 names it (template arguments with bf16 for unsigned short).
STAGE_KERNEL = {
    "fwd_intra": "chunk_intra_fwd_kernel<bf16, 128, true, false>",
    "fwd_state": "chunk_state_fwd_rr_kernel<128, 64, true, true>",
    "bwd_state": "chunk_state_bwd_rr_kernel<128, 64, true, true>",
    "bwd_chunk": "chunk_fused_bwd_w4_kernel<128>",
    "decode": "decode_kernel<bf16, 128, 512>",
}
# The production operator's chunk kernels (per-channel gate, BF16 keys with
# the preconditioner's write key, d = 128), by the same stage split.
PRODUCTION_STAGE_KERNEL = {
    "fwd_intra": "chunk_intra_fwd_pc2_kernel<false>",
    "fwd_state": "chunk_state_fwd_rr_pc_kernel<128, 64>",
    "bwd_state": "chunk_state_bwd_rr_pc_kernel<128, 64>",
    "bwd_chunk": "chunk_fused_bwd_pc_kernel<bf16, 128, bf16, bf16>",
}
TRAFFIC_PROFILE = ROOT / "profiles" / "pkda_chunk_c2_decode_c4_hbm_traffic.md"
COUNTER_PROFILE = ROOT / "profiles" / "pkda_chunk_c2_mfma_counters.md"
# Every kernel one c2 step launches (the traffic of the whole step is their sum).
STEP_KERNELS = ("gate_fwd_kernel", STAGE_KERNEL["fwd_intra"], STAGE_KERNEL["fwd_state"], STAGE_KERNEL["bwd_state"],
                STAGE_KERNEL["bwd_chunk"], "gate_bwd_kernel")
# Algorithmic HBM bytes of one c2 fwd+bwd per token-head (per-head gate, BF16
# activations): forward q, k, v, g, beta in and o out (1,028 B), backward q,
# k, v, dO, g, beta in and dq, dk, dv, dg, dbeta out (1,800 B).
STEP_ALG_BYTES = 2828


def stage_alg_bytes(D: int, per_channel: bool = False) -> dict[str, int]:
    """The bytes per token-head each stage kernel has to move at minimum: the
    step's own inputs and outputs it touches (BF16 activations, FP32 per-head
    gate and beta; per channel, a BF16 gate in and its gradient out), nothing
    of the intermediates the kernels hand each other."""
    a = 2 * D                      # one BF16 activation row
    gate = 2 * D if per_channel else 4
    return {
        "fwd_intra": 2 * a + gate + 4,                 # q, k; g, beta
        "fwd_state": 3 * a + gate + 4 + a,             # q, k, v; g, beta; o
        "bwd_state": 3 * a + gate + 4,                 # q, k, dO; g, beta
        "bwd_chunk": 4 * a + gate + 4 + 3 * a + gate + 4,  # q, k, v, dO; g, beta; dq, dk, dv; dg, dbeta
    }


def kernel_source_hash(serving: bool = False) -> str:
    """SHA-256 over the library's kernel sources and C ABI header (sorted by
    name): what a committed counter summary was measured on.  The serving
    operators' sources, which the PKDA kernels do not read, have one of their
    own, with the header they share."""
    import hashlib

    h = hashlib.sha256()
    csrc, include = ROOT / "delta_feedback_experiment_amd" / "csrc", ROOT / "include"
    if serving:
        files = sorted((csrc / "serve").glob("*.hip")) + sorted((csrc / "serve").glob("*.h"))
        files += sorted((include / "serve").glob("*.h")) + [csrc / "pkda_common.h"]
    else:
        files = sorted(csrc.glob("*.hip"))
        files += sorted(csrc.glob("*.h"))
        files += sorted(include.glob("*.h"))
    for f in files:
        h.update(f.name.encode())
        h.update(f.read_bytes())
    return h.hexdigest()[:16]


def profiled_traffic(kernel: str) -> dict | None:
    """HBM bytes per launch of ``kernel`` from the committed rocprofv3 PMC summary
    (FETCH_SIZE and WRITE_SIZE passes, scaled by the counters of a 1 GiB copy).
    None when the summary has no row for this kernel; a summary measured on
    other kernel sources than these (its ``source hash`` line) is refused and
    reported as stale instead of as bytes."""
    if not TRAFFIC_PROFILE.exists():
        return None
    text = TRAFFIC_PROFILE.read_text()
    recorded = None
    for line in text.splitlines():
        if line.lower().startswith("source hash:"):
            recorded = line.split(":", 1)[1].strip().strip("`")
    current = kernel_source_hash()
    for line in text.splitlines():
        cells = [c.strip() for c in line.strip().strip("|").split("|")]
        if len(cells) == 4 and cells[0].strip("`").startswith(kernel + "("):
            if recorded != current:
                return {"stale": True, "profile_source_hash": recorded, "source_hash": current,
                        "source": TRAFFIC_PROFILE.name}
            read_mib, write_mib = float(cells[2]), float(cells[3])
            return {"bytes": (read_mib + write_mib) * 2**20, "read_MiB": read_mib, "written_MiB": write_mib,
                    "source": TRAFFIC_PROFILE.name, "source_hash": recorded}
    return None


def traffic_bytes(t: dict | None) -> float | None:
    return None if t is None or t.get("stale") else t["bytes"]


def profiled_mfma_busy(kernel: str) -> float | None:
    """The committed SQ counter pass's MFMA busy fraction of ``kernel`` (share
    of the SIMDs' cycles the matrix units were issued work), or None when the
    summary has no row for it or was taken on other kernel sources."""
    if not COUNTER_PROFILE.exists():
        return None
    text = COUNTER_PROFILE.read_text()
    recorded = None
    for line in text.splitlines():
        if line.lower().startswith("source hash:"):
            recorded = line.split(":", 1)[1].strip().strip("`")
    if recorded != kernel_source_hash():
        return None
    for line in text.splitlines():
        cells = [c.strip() for c in line.strip().strip("|").split("|")]
        if len(cells) == 8 and cells[0].strip("`").startswith(kernel + "("):
            try:
                return float(cells[4]) / 100.0
            except ValueError:
                return None
    return None


def roofline_for(stage: str, kernel: str, ms: float, flops: float, alg_bytes: float) -> dict:
    """The roofline object of one kernel launch from its measured duration.

    Both rates are measured: the algorithmic flops per launch over the launch
    time (fraction of dense BF16 MFMA peak) and the HBM bytes the PMC counters
    saw per launch over the same time (fraction of 8 TB/s).  ``bound`` is the
    roof the kernel runs closer to; ``achieved`` / ``frac`` are quoted against
    it -- algorithmic bytes per launch for an HBM-bound kernel, algorithmic
    flops for an MFMA-bound one -- and the other roof's figures stay beside
    them, with the counter pass's MFMA busy share and the ratio of measured to
    algorithmic bytes (above 1: bytes the kernel moves beyond its minimum)."""
    sec = ms / 1e3
    traffic = profiled_traffic(kernel)
    tbytes = traffic_bytes(traffic)
    mfma_frac = flops / sec / MFMA_BF16_PEAK
    hbm_meas = None if tbytes is None else tbytes / sec / HBM_PEAK
    hbm_alg = alg_bytes / sec / HBM_PEAK
    bound = "hbm" if (hbm_meas if hbm_meas is not None else hbm_alg) > mfma_frac else "mfma"
    out = {"bound": bound, "kernel": stage, "kernel_name": kernel, "ms": ms}
    if bound == "hbm":
        out.update(achieved=alg_bytes / sec / 1e9, peak=HBM_PEAK / 1e9, unit="GB/s", frac=hbm_alg)
    else:
        out.update(achieved=flops / sec / 1e12, peak=MFMA_BF16_PEAK / 1e12, unit="TFLOP/s", frac=mfma_frac)
    out.update(traffic=tbytes, traffic_detail=traffic, alg_bytes=alg_bytes,
               traffic_ratio=None if tbytes is None else tbytes / alg_bytes,
               hbm_GBps=None if tbytes is None else tbytes / sec / 1e9, hbm_frac_measured=hbm_meas,
               mfma_TFLOPs=flops / sec / 1e12, mfma_frac=mfma_frac, mfma_busy_counter=profiled_mfma_busy(kernel))
    return out


def step_traffic(token_heads: int) -> dict:
    """HBM bytes of one c2 step from the committed PMC summary (the sum over
    the kernels the step launches) against the step's algorithmic bytes."""
    rows = {k: profiled_traffic(k) for k in STEP_KERNELS}
    alg = STEP_ALG_BYTES * token_heads
    if any(traffic_bytes(r) is None for r in rows.values()):
        return {"bytes": None, "alg_bytes": alg, "ratio": None,
                "missing_or_stale": [k for k, r in rows.items() if traffic_bytes(r) is None]}
    total = sum(traffic_bytes(r) for r in rows.values())
    return {"bytes": total, "GiB": total / 2**30, "alg_bytes": alg, "alg_GiB": alg / 2**30, "ratio": total / alg,
            "per_kernel_MiB": {k: traffic_bytes(r) / 2**20 for k, r in rows.items()}}


def l2norm(t: torch.Tensor) -> torch.Tensor:
    f = t.float()
    return f * torch.rsqrt(f.square().sum(-1, keepdim=True) + 1e-6)


def geometric_cu_seqlens(total: int, gen: torch.Generator) -> torch.Tensor:
    """Document lengths 16 + Geometric(p = 1/1009) (mean 1024), truncated to ``total``."""
    p = 1.0 / 1009.0
    lens = []
    acc = 0
    while acc < total:
        u = torch.rand((), generator=gen, dtype=torch.float64).item()
        n = 16 + int(math.floor(math.log1p(-u) / math.log1p(-p)))
        n = min(n, total - acc)
        lens.append(n)
        acc += n
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def make_chunk_inputs(w: dict, dev: torch.device, seed: int = 42):
    B, T, H, D = w["B"], w["T"], w["H"], w["D"]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen, device=dev)

    q = l2norm(randn(B, T, H, D)).to(torch.bfloat16)
    k = l2norm(randn(B, T, H, D)).to(torch.bfloat16)
    v = randn(B, T, H, D).to(torch.bfloat16)
    beta = torch.sigmoid(randn(B, T, H))
    g = -F.softplus(randn(B, T, H))
    if w["strong"]:
        mask = torch.rand(B, T, generator=gen, device=dev) < 0.1
        g = torch.where(mask[:, :, None], torch.full_like(g, -8.0), g)
    do = randn(B, T, H, D).to(torch.bfloat16)
    cu = None
    N = B
    if w["varlen"]:
        cu = geometric_cu_seqlens(T, torch.Generator().manual_seed(seed)).to(dev)
        N = cu.numel() - 1
    s0 = 0.02 * randn(N, H, D, D) if w["s0"] else None
    return dict(q=q, k=k, v=v, g=g, beta=beta, do=do, cu=cu, s0=s0)


def fwd_bwd(inp: dict, leaves: list[torch.Tensor]):
    from delta_feedback_experiment_amd import chunk_pkda

    q, k, v, g, beta = leaves[:5]
    s0 = leaves[5] if len(leaves) > 5 else None
    o, S, _ = chunk_pkda(q, k, v, g, beta, initial_state=s0, output_final_state=s0 is not None,
                         cu_seqlens=inp["cu"])
    outs = [o] if S is None else [o, S]
    grads = [inp["do"]] if S is None else [inp["do"], torch.zeros_like(S)]
    return torch.autograd.grad(outs, leaves, grads)


def time_step(inp: dict, steps: int, warmup: int) -> float:
    """Eager: K fwd+bwd steps between two events on the stream; ms per step."""
    names = ["q", "k", "v", "g", "beta"] + (["s0"] if inp["s0"] is not None else [])
    leaves = [inp[n].detach().requires_grad_() for n in names]
    for _ in range(warmup):
        fwd_bwd(inp, leaves)
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(steps):
        fwd_bwd(inp, leaves)
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / steps


def time_step_graph(inp: dict, steps: int, warmup: int) -> dict:
    """Captured: one fwd+bwd step of the workload (:func:`capture_replays`)."""
    names = ["q", "k", "v", "g", "beta"] + (["s0"] if inp["s0"] is not None else [])
    leaves = [inp[n].detach().requires_grad_() for n in names]
    return capture_replays(lambda: fwd_bwd(inp, leaves), steps, warmup)


def capture_replays(step, steps: int, warmup: int) -> dict:
    """One call of ``step`` (a fwd+bwd returning its gradients) recorded into a
    HIP graph after warm-up on a side stream, replayed K times back to back,
    each replay between its own pair of events (the reference's
    ``captured_run``, scripts/pkda_bench.py:239-285).  Every replay's
    gradients are checked bitwise against an eager call.  Returns ms per step
    over the K replays (first event to last), the median and minimum replay,
    the samples, and whether the replays agree."""
    import statistics

    eager = [gr.clone() for gr in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(max(warmup, 3)):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static_grads = step()
    agree = True
    for _ in range(3):  # replays interleaved with eager work and synchronisation
        graph.replay()
        torch.cuda.synchronize()
        agree &= all(torch.equal(a, b) for a, b in zip(static_grads, eager))
        step()
        torch.cuda.synchronize()
    events = [(torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)) for _ in range(steps)]
    torch.cuda.synchronize()
    for e0, e1 in events:
        e0.record()
        graph.replay()
        e1.record()
    torch.cuda.synchronize()
    samples = [a.elapsed_time(b) for a, b in events]
    agree &= all(torch.equal(a, b) for a, b in zip(static_grads, eager))
    return {"ms_per_step": events[0][0].elapsed_time(events[-1][1]) / steps,
            "median_ms": statistics.median(samples), "min_ms": min(samples), "samples_ms": samples,
            "agree": agree}


def step_checks(inp: dict) -> dict:
    """Before timing: every output and gradient of one eager step is finite,
    and two independent backwards accumulated in FP32 buffers and halved give
    the single step's gradients (the reference's ``accumulation_check``,
    scripts/pkda_bench.py:224-236; these kernels are deterministic, so the
    deviation is FP32 rounding of the sum)."""
    from delta_feedback_experiment_amd import chunk_pkda

    names = ["q", "k", "v", "g", "beta"] + (["s0"] if inp["s0"] is not None else [])
    leaves = [inp[n].detach().requires_grad_() for n in names]
    s0 = leaves[5] if len(leaves) > 5 else None
    o, S, _ = chunk_pkda(*leaves[:5], initial_state=s0, output_final_state=s0 is not None, cu_seqlens=inp["cu"])
    outs = [o] if S is None else [o, S]
    first = torch.autograd.grad(outs, leaves, [inp["do"]] + ([torch.zeros_like(S)] if S is not None else []))
    finite = all(bool(torch.isfinite(t).all()) for t in (*outs, *first))
    sinks = [g.detach().float().clone() for g in first]
    for sink, g in zip(sinks, fwd_bwd(inp, leaves)):
        sink.add_(g.float())
    dev = 0.0
    for name, sink, g in zip(names, sinks, first):
        ref = g.float()
        dev = max(dev, float((sink * 0.5 - ref).norm() / ref.norm().clamp_min(1e-30)))
    return {"finite": finite, "accumulation_max_rel": dev, "accumulation_ok": dev <= 1e-6}


def time_stages(inp: dict, w: dict, steps: int) -> dict[str, float]:
    """Average duration (ms) of each kernel of the step, launched one stage at a
    time on the current stream with events around each launch."""
    from delta_feedback_experiment_amd import _lib
    from delta_feedback_experiment_amd.chunk import ChunkPlan, gate_forward
    from delta_feedback_experiment_amd.pkda import _ptr, _stream

    dev = inp["q"].device
    plan = ChunkPlan.make(inp["q"], inp["cu"])
    ntok, H, D = plan.num_tokens, plan.heads, plan.head_dim
    flat = lambda t: t.reshape(ntok, H, D)  # noqa: E731
    q, k, v, do = (flat(inp[n].contiguous()) for n in ("q", "k", "v", "do"))
    beta = inp["beta"].float().reshape(ntok, H).contiguous()
    gcum = gate_forward(plan, inp["g"].reshape(ntok, H).contiguous(), _lib.GATE_LOG_HEAD, None, None)
    bf = dict(device=dev, dtype=torch.bfloat16)
    f32 = dict(device=dev, dtype=torch.float32)
    o, wbuf, ubuf = torch.empty(ntok, H, D, **bf), torch.empty(ntok, H, D, **bf), torch.empty(ntok, H, D, **bf)
    # Aqk and T packed (their ten lower blocks per chunk), as the step stores them
    aqk, akk = torch.empty(plan.num_chunks, H, 10, 256, **bf), torch.empty(plan.num_chunks, H, 10, 256, **bf)
    h = torch.empty(plan.num_chunks, H, D, D, **bf)
    dh = torch.empty(plan.num_chunks, H, D, D, **bf)
    du = torch.empty(ntok, H, D, **bf)
    dq, dk, dv = (torch.empty(ntok, H, D, **bf) for _ in range(3))  # the step's own gradient dtype
    dbeta, dgcum = torch.empty(ntok, H, **f32), torch.empty(ntok, H, **f32)
    s0 = inp["s0"]
    scale = D ** -0.5
    fa = _lib.ChunkFwdArgs(
        dtype=_lib.PKDA_BF16, **plan.common(), q=_ptr(q), k=_ptr(k), kw=_ptr(k), v=_ptr(v), gcum=_ptr(gcum),
        gate_per_channel=0, beta=_ptr(beta), scale=scale, initial_state=_ptr(s0), final_state=None, o=_ptr(o),
        w=_ptr(wbuf), u=_ptr(ubuf), aqk=_ptr(aqk), akk=_ptr(akk), h=_ptr(h), tri_packed=1,
    )
    ba = _lib.ChunkBwdArgs(
        dtype=_lib.PKDA_BF16, **plan.common(), q=_ptr(q), k=_ptr(k), kw=_ptr(k), v=_ptr(v), gcum=_ptr(gcum),
        gate_per_channel=0, beta=_ptr(beta), scale=scale, initial_state=_ptr(s0),
        w=_ptr(wbuf), u=_ptr(ubuf), aqk=_ptr(aqk), akk=_ptr(akk), h=_ptr(h), do=_ptr(do), dht=None, dh=_ptr(dh),
        du=_ptr(du), dq=_ptr(dq), dk=_ptr(dk), dkw=None, dv=_ptr(dv),
        dbeta=_ptr(dbeta), dgcum=_ptr(dgcum), dh0=None, grad_dtype=_lib.PKDA_BF16, key_grad_dtype=_lib.PKDA_BF16,
        tri_packed=1,
    )
    return _event_stages(fa, ba, _stream(dev), steps)


def _event_stages(fa, ba, stream, steps: int) -> dict[str, float]:
    """Average duration (ms) of each kernel of one chunked fwd+bwd, launched
    stage by stage on ``stream`` (torch's current stream) with events around
    each launch."""
    from delta_feedback_experiment_amd import _lib

    stages = [
        ("fwd_intra", "pkda_chunk_fwd", fa, _lib.STAGE_FWD_INTRA),
        ("fwd_state", "pkda_chunk_fwd", fa, _lib.STAGE_FWD_STATE),
        ("bwd_state", "pkda_chunk_bwd", ba, _lib.STAGE_BWD_STATE),
        ("bwd_chunk", "pkda_chunk_bwd", ba, _lib.STAGE_BWD_CHUNK),
    ]
    events = {name: [] for name, *_ in stages}

    def run(record: bool):
        for name, fn, args, mask in stages:
            args.stages = mask
            if record:
                e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                e0.record()
            _lib.call(fn, args, stream)
            if record:
                e1.record()
                events[name].append((e0, e1))

    run(False)
    torch.cuda.synchronize()
    for _ in range(steps):
        run(True)
    torch.cuda.synchronize()
    return {name: sum(a.elapsed_time(b) for a, b in ev) / len(ev) for name, ev in events.items()}


def bench_decode(dev: torch.device, steps: int, warmup: int = 10, seed: int = 7) -> dict:
    """B=256 live sequences in a 512-slot FP32 pool [512, 32, 128, 128]."""
    from delta_feedback_experiment_amd import pkda_decode_step_

    P, N, H, D = 512, 256, 32, 128
    gen = torch.Generator(device=dev).manual_seed(seed)
    pool = 0.02 * torch.randn(P, H, D, D, generator=gen, device=dev)
    cpu_gen = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(P, generator=cpu_gen)[:N] for _ in range(steps)]).to(torch.int32).to(dev)
    sets = []
    for _ in range(4):
        q = l2norm(torch.randn(N, H, D, generator=gen, device=dev)).to(torch.bfloat16)
        k = l2norm(torch.randn(N, H, D, generator=gen, device=dev)).to(torch.bfloat16)
        v = torch.randn(N, H, D, generator=gen, device=dev).to(torch.bfloat16)
        beta = torch.sigmoid(torch.randn(N, H, generator=gen, device=dev))
        g = -F.softplus(torch.randn(N, H, generator=gen, device=dev))
        sets.append((q, k, v, g, beta))
    out = torch.empty(N, H, D, device=dev, dtype=torch.bfloat16)
    for i in range(warmup):
        pkda_decode_step_(*sets[i % 4], pool, idx[i % steps], out=out)
    torch.cuda.synchronize()
    # eager: one event pair around all steps
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for i in range(steps):
        pkda_decode_step_(*sets[i % 4], pool, idx[i], out=out)
    t1.record()
    torch.cuda.synchronize()
    wall_ms = t0.elapsed_time(t1)
    # captured: all `steps` steps, each with its own slot permutation, in one
    # HIP graph (one launch per step), replayed `reps` times
    import statistics

    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pkda_decode_step_(*sets[0], pool, idx[0], out=out)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        for i in range(steps):
            pkda_decode_step_(*sets[i % 4], pool, idx[i], out=out)
    graph.replay()
    torch.cuda.synchronize()
    reps = 5
    samples = []
    for _ in range(reps):
        t0.record()
        graph.replay()
        t1.record()
        torch.cuda.synchronize()
        samples.append(t0.elapsed_time(t1) / steps)
    kern_ms = statistics.median(samples)
    finite = bool(torch.isfinite(out).all()) and bool(torch.isfinite(pool).all())
    nbytes = 2 * N * H * D * D * 4 + N * H * (2 * (2 * D + D) + 2 * 2) + N * H * D * 2 + 4 * N
    traffic = profiled_traffic(STAGE_KERNEL["decode"])
    return {
        "workload": "c4 decode: 256 live of 512 slots, H32 d128, fp32 state, bf16 q/k/v",
        "steps": steps,
        "ms_per_step": kern_ms,
        "ms_per_step_eager": wall_ms / steps,
        "tokens_per_s": N / (kern_ms / 1e3),
        "kernel_us": kern_ms * 1e3,
        "min_us": min(samples) * 1e3,
        "distinct_slot_permutations": steps,
        "finite": finite,
        "timing": f"HIP graph of {steps} steps (each its own random slot subset), replayed {reps} times; "
                  "kernel_us = median replay time / steps (launch gaps included)",
        "bytes_per_step": nbytes,
        "roofline": {
            "bound": "hbm",
            "kernel": STAGE_KERNEL["decode"],
            "achieved": nbytes / (kern_ms / 1e3) / 1e9,
            "peak": HBM_PEAK / 1e9,
            "unit": "GB/s",
            "frac": nbytes / (kern_ms / 1e3) / HBM_PEAK,
            "traffic": traffic_bytes(traffic),
            "traffic_detail": traffic,
        },
    }


def bench_qkv_conv(dev: torch.device, reps: int = 20) -> dict:
    """The recurrence's producer, the fused Q/K/V short convolution + SiLU +
    per-head L2 norm (delta_feedback_experiment/fla_ops.py:134-249), forward
    and backward at the reference's screen geometry: 8 rows x 4,096 tokens,
    projection width 1,024 (8 heads of 128), conv_size 4, BF16 activations,
    FP32 weights.  Algorithmic bytes: forward reads x and writes q, k, v;
    backward reads x, dq, dk, dv and writes dx (dw and its per-tile partials
    are not counted)."""
    from delta_feedback_experiment_amd import pkda_qkv_conv
    from delta_feedback_experiment_amd.conv import pkda_qkv_conv_backward

    B, T, H, D, W = 8, 4096, 8, 128, 4
    P = H * D
    gen = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(B, T, 3 * P, generator=gen, device=dev).to(torch.bfloat16)
    w = 0.5 * torch.randn(3 * P, W, generator=gen, device=dev)
    do = [torch.randn(B, T, P, generator=gen, device=dev).to(torch.bfloat16) for _ in range(3)]

    def timed(fn) -> float:
        fn()
        torch.cuda.synchronize()
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(reps):
            fn()
        t1.record()
        torch.cuda.synchronize()
        return t0.elapsed_time(t1) / reps

    fwd_ms = timed(lambda: pkda_qkv_conv(x, w, D, 2 * P, 1e-6))
    bwd_ms = timed(lambda: pkda_qkv_conv_backward(x, w, *do, D, 2 * P, 1e-6))
    elem = B * T * 3 * P * 2
    fwd_bytes, bwd_bytes = 2 * elem, 3 * elem
    return {
        "workload": "screen geometry: B8 T4096, 3 x 1024 channels (8 heads of 128), conv_size 4, bf16",
        "fwd_ms": fwd_ms, "bwd_ms": bwd_ms,
        "fwd_bytes": fwd_bytes, "bwd_bytes": bwd_bytes,
        "fwd_GBps": fwd_bytes / (fwd_ms / 1e3) / 1e9, "bwd_GBps": bwd_bytes / (bwd_ms / 1e3) / 1e9,
        "fwd_frac_hbm": fwd_bytes / (fwd_ms / 1e3) / HBM_PEAK, "bwd_frac_hbm": bwd_bytes / (bwd_ms / 1e3) / HBM_PEAK,
        "reference_h100_pcie_ms": {"fwd": 0.215, "bwd": 0.504,
                                   "source": "delta_feedback_experiment/fla_ops.py:39-43, rows not stated"},
    }


def bench_norm_gate(dev: torch.device, reps: int = 20) -> dict:
    """The recurrence's consumer, the RMSNorm sigmoid output gate
    (delta_feedback_experiment/fla_ops.py:572-657), on the c2 recurrence
    output [8, 4096, 16, 128] BF16 with an FP32 weight.  Algorithmic bytes:
    forward reads x, gate and writes y, rstd; backward reads x, gate, dy, rstd
    and writes dx, dgate (dweight and its partials are not counted)."""
    from delta_feedback_experiment_amd import pkda_norm_gate
    from delta_feedback_experiment_amd.norm_gate import pkda_norm_gate_backward

    shape = (8, 4096, 16, 128)
    gen = torch.Generator(device=dev).manual_seed(6)
    x, g, dy = (torch.randn(*shape, generator=gen, device=dev).to(torch.bfloat16) for _ in range(3))
    w = torch.ones(shape[-1], device=dev)
    _, rstd = pkda_norm_gate(x, g, w, 1e-6)

    def timed(fn) -> float:
        fn()
        torch.cuda.synchronize()
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(reps):
            fn()
        t1.record()
        torch.cuda.synchronize()
        return t0.elapsed_time(t1) / reps

    fwd_ms = timed(lambda: pkda_norm_gate(x, g, w, 1e-6))
    bwd_ms = timed(lambda: pkda_norm_gate_backward(x, g, w, rstd, dy, 1e-6))
    rows = x.numel() // shape[-1]
    elem = x.numel() * 2
    fwd_bytes, bwd_bytes = 3 * elem + 4 * rows, 5 * elem + 4 * rows
    return {
        "workload": "c2 recurrence output [8, 4096, 16, 128] bf16, fp32 weight",
        "fwd_ms": fwd_ms, "bwd_ms": bwd_ms, "fwd_bytes": fwd_bytes, "bwd_bytes": bwd_bytes,
        "fwd_GBps": fwd_bytes / (fwd_ms / 1e3) / 1e9, "bwd_GBps": bwd_bytes / (bwd_ms / 1e3) / 1e9,
        "fwd_frac_hbm": fwd_bytes / (fwd_ms / 1e3) / HBM_PEAK, "bwd_frac_hbm": bwd_bytes / (bwd_ms / 1e3) / HBM_PEAK,
    }


def bench_serve(dev: torch.device, reps: int = 10) -> dict:
    """The slot-pool serving path (``delta_feedback_experiment_amd.serve``).

    prefill: a cached prefill of the c2 shape (8 prompts x 4,096 tokens, H16
    d128, BF16, per-head log-decay) whose final states land in 8 slots of a
    64-slot FP32 pool -- the chunked forward only; algorithmic flops
    6 d^2 + 8 C d + 2 C d per token-head (intra + state).
    conv_token: one decode token of the fused Q/K/V convolution for the c4
    batch (256 live sequences of a 512-slot history pool, 3 x 32 x 128
    channels, conv_size 4, BF16): reads x and the 3-row histories, writes
    q, k, v and the new histories (algorithmic bytes)."""
    from delta_feedback_experiment_amd import pkda_prefill_, pkda_qkv_conv_cached_

    def timed(fn) -> float:
        fn()
        torch.cuda.synchronize()
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(reps):
            fn()
        t1.record()
        torch.cuda.synchronize()
        return t0.elapsed_time(t1) / reps

    w = WORKLOADS["c2"]
    inp = make_chunk_inputs(w, dev, seed=11)
    B, T, H, D = w["B"], w["T"], w["H"], w["D"]
    pool = torch.zeros(64, H, D, D, device=dev)
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(1))[:B].to(torch.int32).to(dev)
    prefill_ms = timed(lambda: pkda_prefill_(inp["q"], inp["k"], inp["v"], inp["g"], inp["beta"], pool, slots))
    flops = B * T * H * step_flops_convention(D) // 3  # the forward of the convention
    del inp, pool
    N, P, Hd, Wc = 256, 512, 32, 4
    C = 3 * Hd * D
    gen = torch.Generator(device=dev).manual_seed(12)
    x = torch.randn(N, 1, C, generator=gen, device=dev).to(torch.bfloat16)
    wt = 0.5 * torch.randn(C, Wc, generator=gen, device=dev)
    hist = torch.randn(P, Wc - 1, C, generator=gen, device=dev).to(torch.bfloat16)
    cslots = torch.randperm(P, generator=torch.Generator().manual_seed(2))[:N].to(torch.int32).to(dev)
    conv_ms = timed(lambda: pkda_qkv_conv_cached_(x, wt, D, 2 * Hd * D, 1e-6, hist, cslots))
    conv_bytes = N * C * 2 * (1 + 2 * (Wc - 1) + 1)
    return {
        "prefill": {
            "workload": "c2 shape prefill into 8 of 64 FP32 slots: B8 T4096 H16 d128 bf16, forward only",
            "ms": prefill_ms, "tokens_per_s": B * T / (prefill_ms / 1e3),
            "mfma_frac": flops / (prefill_ms / 1e3) / MFMA_BF16_PEAK,
        },
        "conv_token": {
            "workload": "c4 decode token: 256 of 512 history slots, 3 x 32 x 128 channels, conv_size 4, bf16",
            "us": conv_ms * 1e3, "bytes": conv_bytes, "GBps": conv_bytes / (conv_ms / 1e3) / 1e9,
            "frac_hbm": conv_bytes / (conv_ms / 1e3) / HBM_PEAK,
        },
    }


def bench_controls(dev: torch.device, reps: int = 20) -> dict:
    """The control path at the c2 geometry (8 x 4,096 tokens, H16 d128, BF16):
    the control activations with their packed gradient, and the gate with the
    decay expansion fused (hidden rows in, chunk-local cumsum out) against the
    materialised form (F.linear's raw decay, then the raw-gate kernel).
    Algorithmic bytes: controls forward reads the 3H logits and writes beta,
    precond_decay (FP32), precond_beta; backward reads the logits and five
    gradients and writes the packed gradient; the gate reads the hidden rows
    and writes the FP32 cumsum [N, H, d]."""
    from delta_feedback_experiment_amd import _lib, pkda_controls
    from delta_feedback_experiment_amd.chunk import ChunkPlan, gate_forward, low_rank_rows
    from delta_feedback_experiment_amd.controls import pkda_controls_act, pkda_controls_backward

    def timed(fn) -> float:
        fn()
        torch.cuda.synchronize()
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(reps):
            fn()
        t1.record()
        torch.cuda.synchronize()
        return t0.elapsed_time(t1) / reps

    B, T, H, D = 8, 4096, 16, 128
    N = B * T
    width = 2 * D + 3 * H
    gen = torch.Generator(device=dev).manual_seed(21)
    packed = (torch.randn(B, T, width, generator=gen, device=dev) / 3 ** 0.5).to(torch.bfloat16)
    A_p = torch.rand(H, generator=gen, device=dev) + 1
    dt_p = 0.1 * torch.randn(H, generator=gen, device=dev)
    grads = (torch.randn(B, T, D, generator=gen, device=dev).to(torch.bfloat16),
             torch.randn(B, T, H, generator=gen, device=dev).to(torch.bfloat16),
             torch.randn(B, T, H, generator=gen, device=dev),
             torch.randn(B, T, H, generator=gen, device=dev).to(torch.bfloat16),
             torch.randn(B, T, D, generator=gen, device=dev).to(torch.bfloat16))
    fwd_ms = timed(lambda: pkda_controls_act(packed, A_p, dt_p, D, H))
    bwd_ms = timed(lambda: pkda_controls_backward(packed, A_p, dt_p, *grads, D, H))
    fwd_bytes = N * 3 * H * 2 + N * H * (2 + 4 + 2)
    bwd_bytes = N * 3 * H * 2 + N * (2 * D * 2 + H * (2 + 4 + 2)) + N * width * 2
    hidden = pkda_controls(packed, A_p, dt_p, D, H)[0]
    up = ((torch.rand(H * D, D, generator=gen, device=dev) * 2 - 1) / D ** 0.5).to(torch.bfloat16)
    A_log = torch.rand(H, generator=gen, device=dev) + 1
    dt = 0.1 * torch.randn(H * D, generator=gen, device=dev)
    plan = ChunkPlan.make(torch.empty(B, T, H, D, device=dev, dtype=torch.bfloat16), None)
    rows = low_rank_rows(hidden, N)
    fused_ms = timed(lambda: gate_forward(plan, rows, _lib.GATE_LOW_RANK, A_log, dt, up))

    def materialised():
        raw = torch.nn.functional.linear(hidden, up).reshape(N, H, D)
        return gate_forward(plan, raw, _lib.GATE_RAW_CHANNEL, A_log, dt)

    mat_ms = timed(materialised)
    gate_bytes = N * D * 2 + N * H * D * 4
    return {
        "workload": "c2 geometry: 8 x 4096 tokens, H16 d128, bf16 packed controls [.., 2d + 3H]",
        "controls_fwd_us": fwd_ms * 1e3, "controls_bwd_us": bwd_ms * 1e3,
        "controls_fwd_GBps": fwd_bytes / (fwd_ms / 1e3) / 1e9, "controls_bwd_GBps": bwd_bytes / (bwd_ms / 1e3) / 1e9,
        "gate_fused_ms": fused_ms, "gate_materialised_ms": mat_ms,
        "gate_fused_GBps": gate_bytes / (fused_ms / 1e3) / 1e9,
    }


def production_inputs(dev: torch.device, B: int = 8, T: int = 4096, H: int = 16, D: int = 128, seed: int = 31):
    """The production operator's inputs as the reference's bench draws them
    (scripts/pkda_bench.py:162-187): normalised q, k; raw per-channel decay
    projection 0.2 N(0, 1); A_log = log U(1, 16); preconditioner decay and
    strength; dO ~ N(0, 1).  BF16 activations, FP32 controls."""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen, device=dev)

    q, k = l2norm(rn(B, T, H, D)).to(torch.bfloat16), l2norm(rn(B, T, H, D)).to(torch.bfloat16)
    v = rn(B, T, H, D).to(torch.bfloat16)
    g_raw = (0.2 * rn(B, T, H, D)).to(torch.bfloat16)
    beta = torch.sigmoid(0.2 * rn(B, T, H))
    A_log = torch.empty(H, device=dev).uniform_(1, 16, generator=gen).log()
    dt_bias = 0.1 * rn(H * D)
    g_atk = -F.softplus(0.2 * rn(B, T, H) + 0.3)
    beta_atk = torch.sigmoid(rn(B, T, H))
    center = -0.2 + 0.1 * rn(H)
    do = rn(B, T, H, D).to(torch.bfloat16)
    return (q, k, v, g_raw, g_atk, beta_atk, beta, A_log, dt_bias, center), do


PRODUCTION_NAMES = ("q", "k", "v", "g", "g_atk", "beta_atk", "beta", "A_log", "dt_bias", "log_atk_scale")


def production_slice(inputs, do, row: int, heads: slice, T_s: int):
    """Row ``row``, tokens 0..T_s-1, heads ``heads`` of the production inputs,
    with the per-head parameters of those heads."""
    q, k, v, g, g_atk, beta_atk, beta, A_log, dt_bias, center = inputs
    H, D = q.shape[2], q.shape[3]
    tok = lambda t: t[row:row + 1, :T_s, heads].contiguous()  # noqa: E731
    h0, h1 = heads.start, heads.stop
    return ((tok(q), tok(k), tok(v), tok(g), tok(g_atk), tok(beta_atk), tok(beta), A_log[h0:h1].contiguous(),
             dt_bias.view(H, D)[h0:h1].reshape(-1).contiguous(), center[h0:h1].contiguous()), tok(do))


def bench_production(dev: torch.device, steps: int = 10, warmup: int = 3) -> dict:
    """The reference model's own training operator (``pkda_recurrence``:
    raw per-channel decay projection with the gate computed on the device,
    write-key preconditioner with x = 1.5, ``fla_ops.py:252-569``) at the c2
    geometry (B8 T4096 H16 d128, BF16), forward and backward of all ten
    inputs, intermediates retained (``lean=False``).

    Before timing, as the reference bench does (scripts/pkda_bench.py:
    205-236): every output and gradient finite, and two backwards
    accumulated in FP32 and halved equal to one (deterministic kernels: FP32
    rounding only).  Agreement with the oracle on a slice runs in the CPU
    leg.  Timing: one step captured in a HIP graph and replayed K times back
    to back, then K eager steps after the warm-up; the faster K-step timing
    is reported (the median and minimum replay beside it).  Flops are
    reported on the same fixed per-token-head convention as the headline
    step."""
    from delta_feedback_experiment_amd import pkda_recurrence

    B, T, H, D = 8, 4096, 16, 128
    inputs, do = production_inputs(dev, B, T, H, D)
    leaves = [x.clone().requires_grad_() for x in inputs]

    def step():
        o, _ = pkda_recurrence(*leaves, D ** -0.5, 1.5, 1e-6, False)
        return torch.autograd.grad(o, leaves, do)

    # -- checks before timing
    o, _ = pkda_recurrence(*leaves, D ** -0.5, 1.5, 1e-6, False)
    first = torch.autograd.grad(o, leaves, do)
    finite = bool(torch.isfinite(o).all()) and all(bool(torch.isfinite(t).all()) for t in first)
    sinks = [t.detach().float().clone() for t in first]
    for sink, t in zip(sinks, step()):
        sink.add_(t.float())
    acc_dev = max(float((sink * 0.5 - t.float()).norm() / t.float().norm().clamp_min(1e-30))
                  for sink, t in zip(sinks, first))
    checks = {"finite": finite, "accumulation_max_rel": acc_dev, "accumulation_ok": acc_dev <= 1e-6}
    del o, first, sinks
    print(f"[bench] production checks {json.dumps(checks)}", file=sys.stderr, flush=True)

    # K graph replays back to back, then K eager steps after the warm-up, as
    # for the headline step: the faster of the two K-step timings
    graph = capture_replays(step, steps, warmup)
    for _ in range(warmup):
        step()
    torch.cuda.synchronize()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(steps):
        step()
    t1.record()
    torch.cuda.synchronize()
    ms_eager = t0.elapsed_time(t1) / steps
    use_graph = graph["agree"] and graph["ms_per_step"] < ms_eager
    ms = graph["ms_per_step"] if use_graph else ms_eager
    stage_ms = time_production_stages([x.detach() for x in leaves], do, D ** -0.5, steps)
    # dominant kernel: the per-channel fused backward, priced on the products
    # it shares with the per-head kernel (its pair terms come on top)
    dom = max(stage_ms, key=stage_ms.get)
    roofline = roofline_for(dom, PRODUCTION_STAGE_KERNEL[dom], stage_ms[dom], B * T * H * stage_flops(D)[dom],
                            B * T * H * stage_alg_bytes(D, per_channel=True)[dom])
    return {
        "workload": "c2 geometry, production operator: B8 T4096 H16 d128 bf16, raw per-channel gate, "
                    "preconditioner x=1.5, fwd+bwd of all ten inputs",
        "ms_per_step": ms, "ms_per_step_eager": ms_eager, "median_ms": graph["median_ms"], "min_ms": graph["min_ms"],
        "graph_ms_per_step": graph["ms_per_step"], "graph_replays_agree": graph["agree"],
        "timing": (f"HIP graph, {steps} replays back to back" if use_graph
                   else f"eager, {steps} steps back to back after {warmup} warm-up steps"),
        "tokens_per_s": B * T / (ms / 1e3),
        "mfma_frac_step": B * T * H * step_flops_convention(D) / (ms / 1e3) / MFMA_BF16_PEAK,
        "checks": checks, "stage_ms": stage_ms, "stage_kernels": PRODUCTION_STAGE_KERNEL, "roofline": roofline,
    }


def time_production_stages(leaves: list[torch.Tensor], do: torch.Tensor, scale: float, steps: int) -> dict:
    """The production operator's four chunk kernels timed one by one (events
    around each launch), on the intermediates its own forward retains."""
    from delta_feedback_experiment_amd import _lib, ops
    from delta_feedback_experiment_amd.pkda import _ptr, _stream

    q, k, v, g, g_atk, beta_atk, beta, A_log, dt_bias, center = leaves
    with torch.no_grad():
        plan, qf, kf, vf, gf, A32, dt32, gcum, _, pstate, beta32, o, fs = ops._forward(
            q, k, v, g, g_atk, beta_atk, beta, A_log, dt_bias, center, scale, 1.5, 1e-6, save_all=True)
    ntok, H, D = plan.num_tokens, plan.heads, plan.head_dim
    dev = q.device
    bf = dict(device=dev, dtype=torch.bfloat16)
    f32 = dict(device=dev, dtype=torch.float32)
    dof = do.contiguous().reshape(ntok, H, D)
    ob = torch.empty(ntok, H, D, **bf)
    dh = torch.empty(plan.num_chunks, H, D, D, **bf)
    du = torch.empty(ntok, H, D, **bf)
    dq, dk, dkw, dv = (torch.empty(ntok, H, D, **bf) for _ in range(4))
    dbeta, dgcum = torch.empty(ntok, H, **f32), torch.empty(ntok, H, D, **f32)
    common = dict(dtype=_lib.PKDA_BF16, **plan.common(), q=_ptr(qf), k=_ptr(kf), kw=_ptr(pstate.kw), v=_ptr(vf),
                  gcum=_ptr(gcum), gate_per_channel=1, beta=_ptr(beta32), scale=scale, initial_state=None,
                  w=_ptr(fs.w), u=_ptr(fs.u), aqk=_ptr(fs.aqk), akk=_ptr(fs.akk), h=_ptr(fs.h),
                  qg=_ptr(fs.qg), kg=_ptr(fs.kg))
    fa = _lib.ChunkFwdArgs(**common, final_state=None, o=_ptr(ob))
    ba = _lib.ChunkBwdArgs(
        **common, do=_ptr(dof), dht=None, dh=_ptr(dh), du=_ptr(du), dq=_ptr(dq), dk=_ptr(dk), dkw=_ptr(dkw),
        dv=_ptr(dv), dbeta=_ptr(dbeta), dgcum=_ptr(dgcum), dh0=None, grad_dtype=_lib.PKDA_BF16,
        key_grad_dtype=_lib.PKDA_BF16, kw32=_ptr(pstate.kw32))
    return _event_stages(fa, ba, _stream(dev), steps)


def copy_bandwidth(dev: torch.device, nbytes: int = 1 << 30, reps: int = 10) -> dict:
    """A plain device copy of ``nbytes`` (read + write), the practical HBM
    ceiling beside the kernels' rates and the scale for the byte counters."""
    src = torch.empty(nbytes // 4, device=dev, dtype=torch.float32).fill_(1.0)
    dst = torch.empty_like(src)
    dst.copy_(src)
    torch.cuda.synchronize()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(reps):
        dst.copy_(src)
    t1.record()
    torch.cuda.synchronize()
    ms = t0.elapsed_time(t1) / reps
    return {"bytes_read": nbytes, "bytes_written": nbytes, "us": ms * 1e3,
            "GBps": 2 * nbytes / (ms / 1e3) / 1e9}


def workload_line(name: str, dev: torch.device, steps: int, warmup: int) -> dict:
    """One more workload's fwd+bwd step (c3 packed documents, c5 long
    context), captured and replayed as the headline step, with the same
    pre-timing checks."""
    w = WORKLOADS[name]
    inp = make_chunk_inputs(w, dev)
    checks = step_checks(inp)
    g = time_step_graph(inp, steps, warmup)
    ntok = w["B"] * w["T"]
    flops = ntok * w["H"] * step_flops_convention(w["D"])
    line = {
        "workload": f"{name}: " + {"c3": "one packed row of 32,768 tokens, geometric documents (mean 1,024), "
                                          "state reset per document",
                                   "c5": "B2 T16384, S0 ~ N(0, 0.02), 10% of tokens g = -8"}[name]
                    + f", H{w['H']} d{w['D']} bf16 fwd+bwd",
        "ms_per_step": g["ms_per_step"], "median_ms": g["median_ms"], "min_ms": g["min_ms"],
        "tokens_per_s": ntok / (g["median_ms"] / 1e3),
        "mfma_frac_step": flops / (g["median_ms"] / 1e3) / MFMA_BF16_PEAK,
        "graph_replays_agree": g["agree"], **checks,
    }
    if w["varlen"]:
        line["documents"] = int(inp["cu"].numel() - 1)
    return line


def _slice_inputs(inp: dict, T_s: int) -> dict:
    """The first row's first ``T_s`` tokens of a workload's inputs (packed
    documents cut at ``T_s``), on the host in FP32 (the BF16 values as they
    are), and the same on the device in the workload's dtypes."""
    out = {}
    for n in ("q", "k", "v", "g", "beta", "do"):
        out[n] = inp[n][:1, :T_s].contiguous()
    out["s0"] = None if inp["s0"] is None else inp["s0"][:1].contiguous()
    out["cu"] = None
    if inp["cu"] is not None:
        cu = [c for c in inp["cu"].tolist() if c < T_s] + [T_s]
        out["cu"] = torch.tensor(cu, dtype=torch.int32, device=inp["q"].device)
        if out["s0"] is not None:
            out["s0"] = inp["s0"][:len(cu) - 1].contiguous()
    return out


def production_agreement(dev: torch.device, oracle, T_s: int, heads: slice = slice(4, 8)) -> dict:
    """The production operator on a slice of its bench inputs (row 2, tokens
    0..T_s-1, four heads) against the oracle in FP32 on the same BF16-rounded
    values, every output and all ten gradients (rows and heads of the
    recurrence are independent, so this is the full run's arithmetic on a
    sub-problem of the same data); bar 2e-2 as the headline check."""
    from delta_feedback_experiment_amd import pkda_recurrence

    inputs, do = production_inputs(dev)
    sl, do_s = production_slice(inputs, do, 2, heads, T_s)
    del inputs, do
    D = sl[0].shape[-1]
    leaves = [x.clone().requires_grad_() for x in sl]
    o, _ = pkda_recurrence(*leaves, D ** -0.5, 1.5, 1e-6, False)
    got = torch.autograd.grad(o, leaves, do_s)
    cl = [x.detach().float().cpu().clone().requires_grad_() for x in sl]
    o_r = oracle.pkda_reference(cl[0], cl[1], cl[2], cl[3], cl[6], A_log=cl[7], dt_bias=cl[8],
                                use_gate_in_kernel=True, g_atk=cl[4], beta_atk=cl[5], log_atk_scale=cl[9],
                                x=1.5, eps=1e-6, out_dtype=torch.float32)[0]
    ref = torch.autograd.grad(o_r, cl, do_s.float().cpu())

    def rel(a, b):
        a, b = a.detach().double().cpu(), b.detach().double()
        return float((a - b).norm() / b.norm().clamp_min(1e-30))

    errs = {"o": rel(o.float(), o_r)}
    errs.update({"d" + n: rel(a.float(), b) for n, a, b in zip(PRODUCTION_NAMES, got, ref)})
    finite = bool(torch.isfinite(o).all()) and all(bool(torch.isfinite(t).all()) for t in got)
    print(f"[bench] production agreement vs oracle: {json.dumps({k: f'{v:.2e}' for k, v in errs.items()})}",
          file=sys.stderr, flush=True)
    return {"slice": f"row 2, tokens 0..{T_s - 1}, heads {heads.start}..{heads.stop - 1} of the production inputs",
            "bar": 2e-2, "rel_l2": errs, "finite": finite, "ok": finite and max(errs.values()) <= 2e-2}


def cpu_baseline(inp: dict, D: int = 128, H: int = 16, T: int = 512, seed: int = 3, budget_s: float = 12.0,
                 max_rows: int = 32, agree_tokens: int = 512, c4_seconds: float = 10.0) -> tuple[dict, dict]:
    """The CPU leg: the oracle (a CPU restatement of the reference's portable
    recurrence, pkda.py:355-410) as the checker and the host baseline.

    agreement -- before any timing, the GPU step on a slice of the workload's
      own inputs (first row, first ``agree_tokens`` tokens) against the
      oracle in FP32 on the same BF16-rounded inputs: relative L2 of o and
      every gradient <= 2e-2 (the reference checks agreement before it keeps
      a timing, scripts/pkda_bench.py:343-353);
    value -- the oracle's fwd+bwd over B=1 row slices of the workload (all
      host cores) until ``budget_s`` seconds or ``max_rows`` rows;
    c1_forward -- BASELINE config 1 (B1 T256 H4 d64 FP32) forward, whole;
    c4_decode -- BASELINE config 4 decode steps on the host (256 live of a
      512-slot [512, 32, 128, 128] FP32 pool) until ``c4_seconds``."""
    from delta_feedback_experiment_amd import chunk_pkda
    from oracle import pkda_oracle as oracle

    threads = len(os.sched_getaffinity(0))
    torch.set_num_threads(threads)

    # -- agreement on a slice of the workload, before timing
    sl = _slice_inputs(inp, agree_tokens)
    names = ["q", "k", "v", "g", "beta"] + (["s0"] if sl["s0"] is not None else [])
    dl = [sl[n].detach().clone().requires_grad_() for n in names]
    s0 = dl[5] if len(dl) > 5 else None
    o, S, _ = chunk_pkda(*dl[:5], initial_state=s0, output_final_state=s0 is not None, cu_seqlens=sl["cu"])
    dS = torch.zeros_like(S) if S is not None else None
    got = torch.autograd.grad([o] + ([S] if S is not None else []), dl, [sl["do"]] + ([dS] if dS is not None else []))
    cl = [sl[n].detach().float().cpu().clone().requires_grad_() for n in names]
    o_r, S_r, _ = oracle.pkda_reference(*cl[:5], initial_state=cl[5] if len(cl) > 5 else None,
                                        output_final_state=S is not None,
                                        cu_seqlens=None if sl["cu"] is None else sl["cu"].cpu(),
                                        out_dtype=torch.float32)
    ref = torch.autograd.grad([o_r] + ([S_r] if S_r is not None else []), cl,
                              [sl["do"].float().cpu()] + ([torch.zeros_like(S_r)] if S_r is not None else []))

    def rel(a, b):
        a, b = a.detach().double().cpu(), b.detach().double()
        return float((a - b).norm() / b.norm().clamp_min(1e-30))

    errs = {"o": rel(o.float(), o_r)}
    errs.update({"d" + n: rel(a.float(), b) for n, a, b in zip(names, got, ref)})
    finite = all(bool(torch.isfinite(t).all()) for t in (o, *got))
    agreement = {"slice": f"row 0, tokens 0..{agree_tokens - 1}" + (" (documents cut there)" if sl["cu"] is not None
                                                                     else ""),
                 "bar": 2e-2, "rel_l2": errs, "finite": finite, "ok": finite and max(errs.values()) <= 2e-2}
    print(f"[bench] agreement vs oracle: {json.dumps({k: f'{v:.2e}' for k, v in errs.items()})}", file=sys.stderr,
          flush=True)
    agreement["production"] = production_agreement(inp["q"].device, oracle, agree_tokens)

    # -- the oracle's fwd+bwd rate over row slices
    gen = torch.Generator().manual_seed(seed)
    total = 0.0
    rows = 0
    while rows < max_rows and total < budget_s:
        q = l2norm(torch.randn(1, T, H, D, generator=gen)).to(torch.bfloat16).float()
        k = l2norm(torch.randn(1, T, H, D, generator=gen)).to(torch.bfloat16).float()
        v = torch.randn(1, T, H, D, generator=gen).to(torch.bfloat16).float()
        beta = torch.sigmoid(torch.randn(1, T, H, generator=gen))
        g = -F.softplus(torch.randn(1, T, H, generator=gen))
        do = torch.randn(1, T, H, D, generator=gen)
        leaves = [t.clone().requires_grad_() for t in (q, k, v, g, beta)]
        t0 = time.perf_counter()
        o, _, _ = oracle.pkda_reference(*leaves)
        torch.autograd.grad(o, leaves, do)
        total += time.perf_counter() - t0
        rows += 1

    # -- the whole forward
    with torch.no_grad():
        q1 = l2norm(torch.randn(1, 256, 4, 64, generator=gen))
        k1 = l2norm(torch.randn(1, 256, 4, 64, generator=gen))
        v1 = torch.randn(1, 256, 4, 64, generator=gen)
        b1 = torch.sigmoid(torch.randn(1, 256, 4, generator=gen))
        g1 = -F.softplus(torch.randn(1, 256, 4, generator=gen))
        oracle.pkda_reference(q1, k1, v1, g1, b1)  # warm
        t0 = time.perf_counter()
        reps1 = 0
        while reps1 < 3 or time.perf_counter() - t0 < 2.0:
            oracle.pkda_reference(q1, k1, v1, g1, b1, output_final_state=True)
            reps1 += 1
        c1_ms = (time.perf_counter() - t0) / reps1 * 1e3

    # -- decode steps on the host
    with torch.no_grad():
        P, N4, H4, D4 = 512, 256, 32, 128
        pool = 0.02 * torch.randn(P, H4, D4, D4, generator=gen)
        steps4, t4 = 0, 0.0
        while steps4 < 20 and t4 < c4_seconds:
            idx = torch.randperm(P, generator=gen)[:N4].to(torch.int32)
            q4 = l2norm(torch.randn(N4, H4, D4, generator=gen)).to(torch.bfloat16)
            k4 = l2norm(torch.randn(N4, H4, D4, generator=gen)).to(torch.bfloat16)
            v4 = torch.randn(N4, H4, D4, generator=gen).to(torch.bfloat16)
            b4 = torch.sigmoid(torch.randn(N4, H4, generator=gen))
            g4 = -F.softplus(torch.randn(N4, H4, generator=gen))
            t0 = time.perf_counter()
            oracle.decode_step_reference(q4, k4, v4, g4, b4, pool, idx)
            t4 += time.perf_counter() - t0
            steps4 += 1
        del pool
    base = {
        "value": rows * T / total,
        "unit": "tokens/s",
        "cores": threads,
        "kind": "port",
        "sample": f"oracle fwd+bwd (token-recurrent FP32 torch CPU) over {rows} row(s) of B=1 T={T} H={H} "
                  f"d={D} ({total:.1f} s); same per-token work as one row of the GPU workload",
        "seconds": total,
        "token_heads_per_s": rows * T * H / total,
        "c1_forward": {"workload": "BASELINE config 1: B1 T256 H4 d64 FP32 forward (with final state)",
                       "ms": c1_ms, "tokens_per_s": 256 / (c1_ms / 1e3), "repeats": reps1},
        "c4_decode": {"workload": "BASELINE config 4 on the host: 256 live of 512 FP32 slots [512,32,128,128]",
                      "steps": steps4, "ms_per_step": t4 / steps4 * 1e3, "tokens_per_s": N4 * steps4 / t4},
    }
    return base, agreement


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=10)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--workload", choices=sorted(WORKLOADS), default="c2")
    ap.add_argument("--decode-steps", type=int, default=1000)
    ap.add_argument("--no-decode", action="store_true")
    ap.add_argument("--no-cpu", action="store_true")
    ap.add_argument("--no-conv", action="store_true", help="skip the Q/K/V convolution and norm-gate lines")
    ap.add_argument("--no-graph", action="store_true", help="time the eager step only")
    ap.add_argument("--no-serve", action="store_true", help="skip the slot-pool prefill and conv-token lines")
    ap.add_argument("--no-production", action="store_true",
                    help="skip the production-operator line (per-channel gate + preconditioner)")
    ap.add_argument("--no-extra", action="store_true", help="skip the c3 and c5 lines")
    ap.add_argument("--cpu-tokens", type=int, default=512)
    ap.add_argument("--cpu-seconds", type=float, default=12.0)
    args = ap.parse_args()
    if args.gpus != 1:
        print(f"bench.py measures one GPU; --gpus {args.gpus} is not supported in this build "
              "(the recurrence never communicates; every (sequence, head) shards with no exchange).",
              file=sys.stderr)
        sys.exit(2)
    if not torch.cuda.is_available():
        print("bench.py needs a HIP device", file=sys.stderr)
        sys.exit(2)
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    w = WORKLOADS[args.workload]
    print(f"[bench] workload {args.workload} {w}", file=sys.stderr, flush=True)
    inp = make_chunk_inputs(w, dev)
    ntok = w["B"] * w["T"]
    # before any timing: the CPU leg (oracle agreement on a slice, host
    # baselines) and the step's own checks (finite, FP32 accumulation)
    base = agreement = None
    if not args.no_cpu:
        base, agreement = cpu_baseline(inp, D=w["D"], H=w["H"], T=args.cpu_tokens, budget_s=args.cpu_seconds)
    checks = step_checks(inp)
    print(f"[bench] checks {json.dumps(checks)}", file=sys.stderr, flush=True)
    # Two timings of K whole steps: K replays of the step captured as a HIP
    # graph, then W eager warm-up steps and K eager steps back to back (after
    # the graph, so neither runs on a GPU still at its idle clocks).  A graph
    # replay costs ~10 us per kernel on this ROCm beyond the same launches
    # issued eagerly, and the eager step's host work (0.33 ms) stays behind
    # the GPU's; `value` is the faster of the two and `timing` says which.
    graph_ok, graph = None, None
    if not args.no_graph:
        try:
            graph = time_step_graph(inp, args.steps, args.warmup)
            graph_ok = graph["agree"]
            print(f"[bench] fwd+bwd graph {graph['ms_per_step']:.3f} ms/step, median {graph['median_ms']:.3f}, "
                  f"min {graph['min_ms']:.3f} (replays agree: {graph_ok})", file=sys.stderr, flush=True)
        except RuntimeError as exc:  # capture unsupported here: report eager
            print(f"[bench] graph capture failed ({exc}); reporting eager timing", file=sys.stderr, flush=True)
    ms_eager = time_step(inp, args.steps, args.warmup)
    print(f"[bench] fwd+bwd eager {ms_eager:.3f} ms/step", file=sys.stderr, flush=True)
    ms, timing = ms_eager, f"eager, {args.steps} steps back to back after {args.warmup} warm-up steps"
    if graph_ok and graph["ms_per_step"] < ms_eager:
        ms, timing = graph["ms_per_step"], f"HIP graph, {args.steps} replays back to back"
    per_th = stage_flops(w["D"])
    token_heads = ntok * w["H"]
    step_flops = token_heads * step_flops_convention(w["D"])
    stage_ms = time_stages(inp, w, args.steps)
    print(f"[bench] stages (ms): {json.dumps({k: round(v, 4) for k, v in stage_ms.items()})}",
          file=sys.stderr, flush=True)
    dom = max(stage_ms, key=stage_ms.get)
    roofline = roofline_for(dom, STAGE_KERNEL[dom], stage_ms[dom], token_heads * per_th[dom],
                            token_heads * stage_alg_bytes(w["D"])[dom])
    if args.workload != "c2":  # the committed counter summaries are of the c2 workload
        for key in ("traffic", "traffic_detail", "traffic_ratio", "hbm_GBps", "hbm_frac_measured",
                    "mfma_busy_counter"):
            roofline[key] = None
    result = {
        "metric": "PKDA fwd+bwd tokens/s & %MFMA peak; decode state-update GB/s & %HBM peak",
        "value": ntok / (ms / 1e3),
        "unit": "tokens/s",
        "n_gpus": 1,
        "steps": args.steps,
        "warmup": args.warmup,
        "ms_per_step": ms,
        "ms_per_step_eager": ms_eager,
        "timing": timing,
        "median_ms": None if graph is None else graph["median_ms"],
        "min_ms": None if graph is None else graph["min_ms"],
        "graph_replays_agree": graph_ok,
        "checks": checks,
        "agreement": agreement,
        "higher_is_better": True,
        "scaling": "weak",
        "vs_baseline": None,
        "dtype": "bf16",
        "data": "synthetic",
        "config": {
            "workload": f"{args.workload} chunked PKDA fwd+bwd",
            "batch": w["B"], "seq_len": w["T"], "heads": w["H"], "head_dim": w["D"], "chunk": CHUNK,
            "state": "fp32", "gate": "per-head log-decay", "varlen": w["varlen"],
        },
        "mfma_frac_step": step_flops / (ms / 1e3) / MFMA_BF16_PEAK,
        "roofline": roofline,
        "step_traffic": step_traffic(token_heads) if args.workload == "c2" else None,
        "stage_ms": stage_ms,
    }
    print(f"[bench] roofline {json.dumps({k: v for k, v in roofline.items() if k != 'traffic_detail'})}",
          file=sys.stderr, flush=True)
    if result["step_traffic"] is not None:
        print(f"[bench] step traffic {json.dumps(result['step_traffic'])}", file=sys.stderr, flush=True)
    result["copy"] = copy_bandwidth(dev)
    print(f"[bench] copy {result['copy']['GBps']:.0f} GB/s", file=sys.stderr, flush=True)
    if not args.no_conv:
        result["qkv_conv"] = bench_qkv_conv(dev)
        c = result["qkv_conv"]
        print(f"[bench] qkv conv fwd {c['fwd_ms']:.3f} ms ({c['fwd_GBps']:.0f} GB/s), "
              f"bwd {c['bwd_ms']:.3f} ms ({c['bwd_GBps']:.0f} GB/s)", file=sys.stderr, flush=True)
        result["norm_gate"] = bench_norm_gate(dev)
        c = result["norm_gate"]
        print(f"[bench] norm gate fwd {c['fwd_ms']:.3f} ms ({c['fwd_GBps']:.0f} GB/s), "
              f"bwd {c['bwd_ms']:.3f} ms ({c['bwd_GBps']:.0f} GB/s)", file=sys.stderr, flush=True)
    if not args.no_conv:
        result["controls"] = bench_controls(dev)
        c = result["controls"]
        print(f"[bench] controls fwd {c['controls_fwd_us']:.1f} us, bwd {c['controls_bwd_us']:.1f} us; "
              f"gate with decay expansion {c['gate_fused_ms']:.3f} ms (materialised {c['gate_materialised_ms']:.3f} ms)",
              file=sys.stderr, flush=True)
    if not args.no_serve:
        del inp
        torch.cuda.empty_cache()
        result["serve"] = bench_serve(dev)
        c = result["serve"]
        print(f"[bench] serve prefill {c['prefill']['ms']:.3f} ms ({c['prefill']['tokens_per_s'] / 1e6:.1f} M tok/s), "
              f"conv token {c['conv_token']['us']:.1f} us ({c['conv_token']['GBps']:.0f} GB/s)", file=sys.stderr,
              flush=True)
        inp = None
    if not args.no_production:
        del inp
        torch.cuda.empty_cache()
        result["production"] = bench_production(dev, args.steps, args.warmup)
        c = result["production"]
        print(f"[bench] production operator {c['ms_per_step']:.3f} ms/step ({c['timing']}; eager "
              f"{c['ms_per_step_eager']:.3f}, graph {c['graph_ms_per_step']:.3f}, replay median {c['median_ms']:.3f}, "
              f"min {c['min_ms']:.3f}, replays agree {c['graph_replays_agree']}) "
              f"({c['tokens_per_s'] / 1e6:.2f} M tok/s); stages (ms): "
              f"{json.dumps({n: round(t, 4) for n, t in c['stage_ms'].items()})}", file=sys.stderr, flush=True)
        inp = None
    if not args.no_extra and args.workload == "c2":
        del inp
        torch.cuda.empty_cache()
        for extra in ("c3", "c5"):
            result[extra] = workload_line(extra, dev, args.steps, args.warmup)
            c = result[extra]
            print(f"[bench] {extra} {c['median_ms']:.3f} ms/step median ({c['tokens_per_s'] / 1e6:.1f} M tok/s, "
                  f"{100 * c['mfma_frac_step']:.1f}% MFMA)", file=sys.stderr, flush=True)
            torch.cuda.empty_cache()
        inp = None
    if not args.no_decode:
        del inp
        torch.cuda.empty_cache()
        result["decode"] = bench_decode(dev, args.decode_steps)
        print(f"[bench] decode {result['decode']['kernel_us']:.1f} us/step", file=sys.stderr, flush=True)
    if base is not None:
        result["cpu_baseline"] = base
    ok = checks["finite"] and checks["accumulation_ok"] and graph_ok is not False
    ok &= agreement is None or agreement["ok"]
    for extra in ("c3", "c5"):
        if extra in result:
            ok &= result[extra]["finite"] and result[extra]["graph_replays_agree"]
    if "decode" in result:
        ok &= result["decode"]["finite"]
    print(json.dumps(result), flush=True)
    if not ok:
        print("[bench] a correctness check failed (see checks / agreement); the timing above is not valid",
              file=sys.stderr, flush=True)
        sys.exit(1)


if __name__ == "__main__":
    main()
