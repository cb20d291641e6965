"""What device data says wrong stays inside the buffers of the loaded server's
operators: outputs, caches and workspaces are cut from larger ones whose bytes
around them have to stay what they were, and bounds that are right once they are
clamped give what the clamped ones give.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from test_gpu_paged_fp8 import Cache8
from test_gpu_paged_prefix import Batch
from test_gpu_verify import Drafts

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    from delta_feedback_experiment_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


class Guards:
    """Tensors inside larger buffers of one byte value."""

    BYTE, EDGE = 0xA5, 1 << 16

    def __init__(self, dev):
        self.dev, self.held = dev, []

    def empty(self, shape, dtype):
        size = torch.empty(0, dtype=dtype).element_size()
        for n in shape:
            size *= n
        buf = torch.full((2 * self.EDGE + size,), self.BYTE, dtype=torch.uint8, device=self.dev)
        self.held.append((buf, size))
        return buf[self.EDGE:self.EDGE + size].view(dtype).view(shape)

    def of(self, t):
        out = self.empty(t.shape, t.dtype)
        out.copy_(t)
        return out

    def check(self):
        torch.cuda.synchronize()
        for buf, size in self.held:
            assert (buf[:self.EDGE] == self.BYTE).all() and (buf[self.EDGE + size:] == self.BYTE).all()


def clamped(bounds, most):
    """The bounds as they are taken, or None where those fall."""
    out = [0] + [min(max(x, 0), most) for x in bounds[1:]]
    return out if all(a <= b for a, b in zip(out, out[1:])) else None


def shared_args(q, table, lens, cu, kp, kv_heads, D):
    return dict(num_seqs=lens.shape[0], num_tokens=q.shape[0], q_heads=q.shape[1], kv_heads=kv_heads, head_dim=D,
                page_size=kp.shape[1], max_pages=table.shape[1], num_pages=kp.shape[0], table_stride=table.stride(0),
                cu_seqlens=None if cu is None else cu.data_ptr(), seq_lens=lens.data_ptr(), page_table=table.data_ptr())


def scale_args(ks, vs):
    return dict(k_scales=ks.data_ptr(), v_scales=vs.data_ptr(), k_scale_stride=ks.stride(0), v_scale_stride=vs.stride(0))


def attend(struct, entry, sizes, g, q, kp, vp, table, lens, cu, **more):
    """An attention entry point with outputs and workspace in guarded buffers."""
    from delta_feedback_experiment_amd import _lib

    N, Hq, D = q.shape
    o, lse = g.empty((N, Hq, D), q.dtype), g.empty((N, Hq), torch.float32)
    args = struct(dtype=1 if q.dtype == torch.bfloat16 else 0, **shared_args(q, table, lens, cu, kp, kp.shape[2], D),
                  q=q.data_ptr(), q_stride=q.stride(0), k_pages=kp.data_ptr(), v_pages=vp.data_ptr(),
                  k_page_stride=kp.stride(0), v_page_stride=vp.stride(0), scale=D ** -0.5, o=o.data_ptr(),
                  lse=lse.data_ptr(), **more)
    args.struct_size = ctypes.sizeof(args)
    floats = getattr(_lib.lib(), sizes)(ctypes.byref(args))
    assert floats >= 0
    workspace = g.empty((floats,), torch.float32)
    args.workspace = workspace.data_ptr() if floats else None
    _lib.call(entry, args, torch.cuda.current_stream().cuda_stream)
    return o, lse


CU = ([0, 4, 9, 900], [0, 12, 3, 15], [3, 4, 9, 15], [-5, -4, TOP, 15], [0, TOP, TOP, TOP], [0, 0, 0, 0], [TOP, 15, 4, 0])
LENS = ([20, 30, 9], [TOP, -3, 9], [-2 ** 31, 0, TOP])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_writes_no_other_rows(dev, dtype):
    """Pages that no row of the table names, and what lies around the pools and the
    queries, stay; rows are stored as by bounds that are clamped beforehand."""
    from delta_feedback_experiment_amd import _lib

    i32 = dict(dtype=torch.int32, device=dev)
    c = Cache8([20, 30, 9], [4, 5, 6], 4, 2, 64, 8, dtype, seed=10, garbage=0.0)
    named = c.table[(c.table >= 0) & (c.table < c.pages)].long()
    extra = 3
    weight = torch.ones(64, device=dev)
    q, k, v = (t.to(dev).contiguous() for t in (c.q, c.k, c.v))
    table = c.table.to(dev)

    def run(cu, lens, eight):
        print(f"[gpu] guards, append {dtype} fp8 {eight} cu {cu} lens {lens}", flush=True)
        g = Guards(dev)
        if eight:
            pools = [torch.full((c.pages + extra, 8, 2, n), 0x31, dtype=torch.uint8, device=dev) for n in (64, 64, 2, 2)]
        else:
            pools = [torch.full((c.pages + extra, 8, 2, 64), 7.0, dtype=dtype, device=dev) for _ in range(2)]
        pools = [g.of(t) for t in pools]
        out = g.empty(q.shape, dtype)
        cu_t, lens_t = torch.tensor(cu, **i32), torch.tensor(lens, **i32)
        args = _lib.PagedStoreArgs(
            dtype=1 if dtype == torch.bfloat16 else 0, **shared_args(q, table, lens_t, cu_t, pools[0], 2, 64),
            q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0),
            q_out=out.data_ptr(), k_pages=pools[0].data_ptr(), v_pages=pools[1].data_ptr(),
            k_page_stride=pools[0].stride(0), v_page_stride=pools[1].stride(0),
            cache_dtype=2 if eight else (1 if dtype == torch.bfloat16 else 0), norm_dtype=0, q_norm=weight.data_ptr(),
            k_norm=weight.data_ptr(), eps=1e-6, **(scale_args(*pools[2:]) if eight else {}))
        _lib.call("pkda_paged_store", args, torch.cuda.current_stream().cuda_stream)
        g.check()
        free = torch.ones(c.pages + extra, dtype=torch.bool)
        free[named] = False
        for t in pools:
            t = t.cpu()
            assert (t[free] == t[-1, 0, 0, 0]).all() and t[-1, 0, 0, 0] == (0x31 if eight else 7.0)
        return [t.cpu() for t in (*pools, out)]

    for eight in (True, False):
        for cu in CU:
            for lens in LENS:
                got, right = run(cu, lens, eight), clamped(cu, 15)
                if right and right != cu:
                    assert all(torch.equal(a, b) for a, b in zip(got, run(right, lens, eight)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_writes_its_outputs_alone(dev, dtype):
    from delta_feedback_experiment_amd import _lib

    i32 = dict(dtype=torch.int32, device=dev)
    c = Cache8([20, 30, 9], [4, 5, 6], 4, 2, 64, 8, dtype, seed=10, garbage=0.0)
    kp, vp, ks, vs = c.cache(dev)
    plain = [t.to(dev) for t in (c.k_pages, c.v_pages)]
    q, table = c.q.to(dev).contiguous(), c.table.to(dev)

    def run(cu, lens, eight):
        print(f"[gpu] guards, attention {dtype} fp8 {eight} cu {cu} lens {lens}", flush=True)
        g = Guards(dev)
        cu_t, lens_t = torch.tensor(cu, **i32), torch.tensor(lens, **i32)
        if eight:
            out = attend(_lib.PagedAttentionFP8Args, "pkda_paged_attention_fp8", "pkda_paged_attention_fp8_workspace", g,
                         q, kp, vp, table, lens_t, cu_t, **scale_args(ks, vs))
        else:
            out = attend(_lib.PagedAttentionArgs, "pkda_paged_attention", "pkda_paged_attention_workspace", g, q, *plain,
                         table, lens_t, cu_t)
        g.check()
        return out

    for eight in (True, False):
        for cu in CU:
            for lens in LENS:
                got, right = run(cu, lens, eight), clamped(cu, 15)
                if right:
                    assert torch.isfinite(got[0]).all()
                    if right != cu:
                        assert all(torch.equal(a, b) for a, b in zip(got, run(right, lens, eight)))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seqs", [6, 90])
def test_groups_write_their_outputs_alone(dev, eight, seqs):
    from delta_feedback_experiment_amd import _lib

    i32 = dict(dtype=torch.int32, device=dev)
    half = seqs // 2
    new = [1 + i % 3 for i in range(seqs)]
    b = Batch([(100, half), (130, half)], [4 + i % 9 for i in range(seqs)], new, 8, 2, 64, 8, torch.bfloat16, seed=10,
              garbage=0.0, fp8_cache=eight)
    (q, kp, vp, table, lens, _, _), more = b.args(dev)
    N, right = q.shape[0], b.cu.tolist()
    scales = scale_args(more["k_scales"], more["v_scales"]) if eight else {}

    def run(groups, prefix, cu):
        print(f"[gpu] guards, prefix fp8 {eight} groups {groups} prefix {prefix} cu {cu[:4]}", flush=True)
        g = Guards(dev)
        groups_t, prefix_t, cu_t = (torch.tensor(x, **i32) for x in (groups, prefix, cu))
        out = attend(_lib.PagedPrefixArgs, "pkda_paged_prefix_attention", "pkda_paged_prefix_workspace", g, q, kp, vp,
                     table, lens, cu_t, **scales, cu_groups=groups_t.data_ptr(), prefix_lens=prefix_t.data_ptr(),
                     num_groups=2)
        g.check()
        return out

    for groups in ([0, half, seqs], [0, half, 900], [0, half + 1, 2], [4, half, TOP], [-5, TOP, 6]):
        for prefix in ([100, 130], [TOP, -3]):
            for cu in (right, right[:-1] + [TOP], [5] + right[1:], right[:2] + [TOP, -1] + right[4:]):
                got = run(groups, prefix, cu)
                if (bounds := clamped(groups, seqs)) and (starts := clamped(cu, N)):
                    assert torch.isfinite(got[0]).all()
                    if bounds != groups or starts != cu:
                        assert all(torch.equal(x, y) for x, y in zip(got, run(bounds, prefix, starts)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("draft", [True, False])
def test_verification_writes_its_outputs_alone(dev, dtype, draft):
    from delta_feedback_experiment_amd import _lib

    i32 = dict(dtype=torch.int32, device=dev)
    for vocab in (1000, 40007):
        d = Drafts([3, 4, 5], vocab, dtype, seed=9, draft=draft)
        args, more = d.inputs()
        logits, drafts, uniform, noise, _ = (t.to(dev) for t in args)
        drafts[1], drafts[7] = TOP, -2 ** 31
        of_drafts = more["draft_logits"].to(dev) if draft else None

        def run(cu):
            print(f"[gpu] guards, verify {dtype} draft logits {draft} cu {cu}", flush=True)
            g = Guards(dev)
            tokens, accepted = g.empty((12,), torch.int32), g.empty((3,), torch.int32)
            cu_t = torch.tensor(cu, **i32)
            a = _lib.VerifyArgs(
                dtype=1 if dtype == torch.bfloat16 else 0, rows=12, vocab=vocab, num_seqs=3, logits=logits.data_ptr(),
                logits_stride=vocab, draft_logits=of_drafts.data_ptr() if draft else None, draft_stride=vocab if draft else 0,
                drafts=drafts.data_ptr(), uniform=uniform.data_ptr(), noise=noise.data_ptr(), noise_stride=vocab,
                cu_seqlens=cu_t.data_ptr(), temperature_all=1.0, tokens=tokens.data_ptr(), accepted=accepted.data_ptr())
            a.struct_size = ctypes.sizeof(a)
            workspace = g.empty((_lib.lib().pkda_verify_workspace(ctypes.byref(a)),), torch.float32)
            a.workspace = workspace.data_ptr()
            _lib.call("pkda_verify", a, torch.cuda.current_stream().cuda_stream)
            g.check()
            return tokens.cpu(), accepted.cpu()

        for cu in ([0, 3, 900, 12], [0, 8, 2, 12], [5, 3, 7, 12], [-4, -1, TOP, 12], [0, 0, 0, 0], [0, TOP, TOP, TOP], [0, 3, 3, 5],
                   [TOP, 12, 4, 0]):
            got, right = run(cu), clamped(cu, 12)
            if right:
                tokens, accepted = got
                assert ((tokens >= -1) & (tokens < vocab)).all() and (tokens[right[-1]:] == -1).all()
                assert ((accepted >= 0) & (accepted <= 11)).all()
                if right != cu:
                    assert all(torch.equal(a, b) for a, b in zip(got, run(right)))
