"""Text generation by a small trunk of alternating PKDA and attention layers.

What a server does with the serving operators: a prompt is prefilled into a
slot of every PKDA layer's pool and into pages of every attention layer's
cache; then all live sequences decode together, one HIP graph replay a token,
and the next token of each is drawn with its own settings.

    python examples/hybrid_decode.py --seqs 64 --tokens 128 [--fp8]

With ``--fp8`` the attention layers norm their heads and keep 8-bit floats.

The weights are random: the tokens mean nothing, the calls are the real ones.
"""

from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path

import torch
from torch import Tensor
from torch.nn import functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from delta_feedback_experiment_amd import (DecodePool, PagedKV, PagedKVFP8, paged_append_, paged_append_fp8_,
                                           paged_attention, paged_attention_fp8, pkda_decode_step_, pkda_prefill_,
                                           pkda_qkv_conv_cached_, sample_tokens)


@dataclass
class Sizes:
    layers: int = 4          # alternating: PKDA, attention, ...
    heads: int = 8           # of both kinds
    kv_heads: int = 2        # of the attention layers
    head_dim: int = 64
    vocab: int = 4096
    slots: int = 64          # sequences at a time
    page_size: int = 16
    pages: int = 1024        # of each attention layer's cache
    max_pages: int = 32      # of one sequence
    dtype: torch.dtype = torch.bfloat16
    fp8: bool = False        # attention layers with head norms and a cache of 8-bit floats


class Trunk:
    """The weights, and every layer's state between calls."""

    def __init__(self, s: Sizes, seed: int = 0, device: str = "cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.s, self.width = s, s.heads * s.head_dim

        def weight(*shape, gain=1.0, dtype=s.dtype):
            return (torch.randn(*shape, generator=gen, device=device) * gain * shape[0] ** -0.5).to(dtype)

        self.embed = weight(s.vocab, self.width, gain=s.vocab ** 0.5)
        self.head = weight(self.width, s.vocab, gain=2.0)
        self.layers = []
        for i in range(s.layers):
            out = weight(self.width, self.width)
            if i % 2 == 0:  # q, k, v for the short convolution; a decay and a write strength a head
                self.layers.append(dict(
                    qkv=weight(self.width, 3 * self.width), out=out, ctl=weight(self.width, 2 * s.heads),
                    conv=torch.randn(3 * self.width, 4, generator=gen, device=device) * 0.5,
                    pool=DecodePool.zeros(s.slots, s.heads, s.head_dim, dtype=s.dtype, precond=False, device=device)))
            else:
                size = (s.pages, s.page_size, s.kv_heads, s.head_dim)
                self.layers.append(dict(
                    qkv=weight(self.width, (s.heads + 2 * s.kv_heads) * s.head_dim), out=out,
                    cache=PagedKVFP8.zeros(*size, device=device) if s.fp8 else
                    PagedKV.zeros(*size, dtype=s.dtype, device=device)))
                if s.fp8:
                    self.layers[-1]["norms"] = [1 + 0.1 * torch.randn(s.head_dim, generator=gen, device=device)
                                                for _ in range(2)]
        angle = torch.outer(torch.arange(s.max_pages * s.page_size, device=device),
                            10000.0 ** (-torch.arange(0, s.head_dim, 2, device=device) / s.head_dim))
        self.cos, self.sin = angle.cos(), angle.sin()

    def _pkda(self, w: dict, h: Tensor, slots: Tensor, prompt: bool) -> Tensor:
        s, N = self.s, h.shape[0]
        rows = (1, N) if prompt else (N, 1)  # one prompt, or one token a sequence
        q, k, v = pkda_qkv_conv_cached_((h @ w["qkv"]).view(*rows, -1), w["conv"], s.head_dim, 2 * self.width, 1e-6,
                                        w["pool"].conv, slots, continue_state=not prompt)
        heads = (*rows, s.heads) if prompt else (N, s.heads)
        q, k, v = (t.view(*heads, s.head_dim) for t in (q, k, v))
        decay, write = (h @ w["ctl"]).float().chunk(2, -1)
        decay, write = -F.softplus(decay).view(heads), torch.sigmoid(write).view(heads)
        step = pkda_prefill_ if prompt else pkda_decode_step_
        return step(q, k, v, decay, write, w["pool"].state, slots).view(N, self.width)

    def _attention(self, w: dict, h: Tensor, table: Tensor, lens: Tensor, cu: Tensor | None) -> Tensor:
        s = self.s
        q, k, v = (h @ w["qkv"]).unflatten(-1, (-1, s.head_dim)).split((s.heads, s.kv_heads, s.kv_heads), 1)
        c = w["cache"]
        place = dict(cu_seqlens=cu, q=q, cos=self.cos, sin=self.sin)
        if s.fp8:
            q = paged_append_fp8_(k, v, c.k, c.v, c.k_scale, c.v_scale, table, lens, q_norm=w["norms"][0],
                                  k_norm=w["norms"][1], **place)
            o, _ = paged_attention_fp8(q, c.k, c.v, c.k_scale, c.v_scale, table, lens, cu_seqlens=cu)
        else:
            q = paged_append_(k, v, c.k, c.v, table, lens, **place)
            o, _ = paged_attention(q, c.k, c.v, table, lens, cu_seqlens=cu)
        return o.flatten(1)

    def __call__(self, tokens: Tensor, slots: Tensor, table: Tensor, lens: Tensor, cu: Tensor | None = None) -> Tensor:
        """Logits ``[tokens, vocab]`` FP32 of one prompt (``cu`` given) or of one token a sequence."""
        x = self.embed[tokens].float()
        for w in self.layers:
            h = F.rms_norm(x, (self.width,)).to(self.s.dtype)
            o = self._pkda(w, h, slots, cu is not None) if "pool" in w else self._attention(w, h, table, lens, cu)
            x = x + (o @ w["out"]).float()
        return (F.rms_norm(x, (self.width,)).to(self.s.dtype) @ self.head).float()


class Server:
    """Live sequences on the slots of a trunk; sequence ``n`` has slot ``n``."""

    def __init__(self, trunk: Trunk, seqs: int, seed: int = 0, **settings):
        s, dev = trunk.s, trunk.embed.device
        if seqs > s.slots:
            raise ValueError(f"{seqs} sequences on {s.slots} slots")
        i32 = dict(dtype=torch.int32, device=dev)
        self.trunk, self.seqs, self.settings = trunk, seqs, settings
        self.free = list(range(s.pages))[::-1]
        self.held = [0] * seqs                       # pages of each sequence
        self.length = [0] * seqs                     # its positions, as the host knows them
        self.table = torch.zeros(seqs, s.max_pages, **i32)
        self.lens = torch.zeros(seqs, **i32)
        self.slots = torch.arange(seqs, **i32)
        self.tokens = torch.zeros(seqs, **i32)       # each sequence's last token, not yet in the states
        self.noise = torch.empty(seqs, s.vocab, device=dev)
        self.gen = torch.Generator(device=dev).manual_seed(seed)
        self.logits = self.graph = None

    def _grow(self, n: int, length: int) -> None:
        """Pages for ``length`` positions of sequence ``n``."""
        s = self.trunk.s
        need = -(-length // s.page_size)
        if need > s.max_pages or need - self.held[n] > len(self.free):
            raise RuntimeError(f"no pages for {length} positions of sequence {n}")
        if need > self.held[n]:
            new = [self.free.pop() for _ in range(need - self.held[n])]
            self.table[n, self.held[n]:need] = torch.tensor(new, dtype=torch.int32).to(self.table.device)
            self.held[n] = need
        self.length[n] = length

    def _draw(self, logits: Tensor, noise: Tensor, **settings) -> Tensor:
        return sample_tokens(logits, noise, **settings)[0]

    def prefill(self, n: int, prompt: Tensor) -> Tensor:
        """A new sequence in slot ``n``; draws its first token and returns its prompt's logits."""
        self._grow(n, len(prompt))
        at = slice(n, n + 1)
        self.lens[at] = len(prompt)
        cu = torch.tensor([0, len(prompt)], dtype=torch.int32).to(self.lens.device)
        logits = self.trunk(prompt, self.slots[at], self.table[at], self.lens[at], cu)
        noise = self.noise[at].exponential_(generator=self.gen).log_().neg_()
        self.tokens[at] = self._draw(logits[-1:], noise, **{k: v[at] if isinstance(v, Tensor) else v
                                                            for k, v in self.settings.items()})
        return logits

    def _step(self) -> Tensor:
        self.lens.add_(1)
        logits = self.trunk(self.tokens, self.slots, self.table, self.lens)
        self.tokens.copy_(self._draw(logits, self.noise, **self.settings))
        return logits

    def capture(self) -> None:
        """One decode step as a graph.  The eager steps that warm it up run on
        copies of what a step changes; the page table keeps its address."""
        kept = [self.lens, self.tokens] + [t for w in self.trunk.layers if "pool" in w
                                           for t in (w["pool"].state, w["pool"].conv)]
        before = [t.clone() for t in kept]
        self.noise.zero_()
        for n in range(self.seqs):  # the warm-up's token has a place in the cache; the real one writes over it
            length = self.length[n]
            self._grow(n, length + 1)
            self.length[n] = length
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.logits = self._step()
        for t, old in zip(kept, before):
            t.copy_(old)
        self.graph = graph

    def step(self) -> Tensor:
        """One token for every sequence; returns the logits it was drawn from."""
        for n in range(self.seqs):
            self._grow(n, self.length[n] + 1)
        self.noise.exponential_(generator=self.gen).log_().neg_()
        if self.graph is None:
            return self._step()
        self.graph.replay()
        return self.logits


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--seqs", type=int, default=64)
    ap.add_argument("--tokens", type=int, default=128)
    ap.add_argument("--fp8", action="store_true")
    args = ap.parse_args()
    s = Sizes(slots=args.seqs, pages=args.seqs * 32, fp8=args.fp8)
    trunk = Trunk(s)
    dev = trunk.embed.device
    gen = torch.Generator().manual_seed(1)
    # every sequence its own settings: greedy, then ever wider
    wide = torch.linspace(0, 1, args.seqs, device=dev)
    server = Server(trunk, args.seqs, temperature=wide, top_p=0.7 + 0.3 * wide,
                    top_k=torch.full((args.seqs,), 50, dtype=torch.int32, device=dev))
    lengths = torch.randint(1, 300, (args.seqs,), generator=gen).tolist()
    start = time.perf_counter()
    for n, length in enumerate(lengths):
        server.prefill(n, torch.randint(0, s.vocab, (length,), generator=gen).to(dev))
    torch.cuda.synchronize()
    print(f"prefilled {sum(lengths)} tokens of {args.seqs} prompts in {time.perf_counter() - start:.3f} s")
    server.capture()
    out = [server.tokens.clone()]
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(args.tokens):
        server.step()
        out.append(server.tokens.clone())
    torch.cuda.synchronize()
    took = time.perf_counter() - start
    print(f"decoded {args.tokens} tokens each: {1e3 * took / args.tokens:.3f} ms a step, "
          f"{args.tokens * args.seqs / took:.0f} tokens/s")
    print("sequence 0:", torch.stack(out)[:12, 0].tolist())


if __name__ == "__main__":
    main()
