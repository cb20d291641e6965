"""What a server under load calls beside the plain paged cache, and how it is measured.

Four operators, in the order a step of a server with drafts meets them:

* ``append``     the new tokens' keys and values into the paged cache, with the norm of every query and key head and
                 the position rotation on the way: into a cache of 8-bit floats with a scale for each 32 channels
                 (``paged_append_fp8_``), or of the activations' type (``paged_append_`` with norms);
* ``attention``  the new tokens' queries over the 8-bit cache, causal (``paged_attention_fp8``);
* ``prefix``     the same where groups of sequences share a long prefix, whose attention is computed once for all of a
                 group, over a cache of either kind (``paged_prefix_attention``);
* ``verify``     drafted tokens against the target's probabilities, from given random numbers, and the token after
                 them (``verify_tokens``).

Heads of 64 and 128 channels, 8 to 32 of them, the packed prompts and the 256 live sequences are those of ``bench.py``,
``perf/cases.py`` and ``perf/operators.py``; page sizes, prefixes and vocabularies are generic.
"""

from __future__ import annotations

import math
import random

import torch

own = False  # True: the framework's operators; False: their plain forms

BLOCK = 32               # channels of a scale
MAX_PAIRS = 2 ** 24      # a drawn attention's (new token, position) pairs
MAX_CACHED = 2 ** 18     # its positions in the cache


# -- the cases -----------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # a chat server between requests: four sequences decode, so launch and latency are the cost
        _append("append8_few", seqs=4, new=1, cached=700, Hq=8, Hkv=2, D=128, page=16),
        # a batch of prompts of mixed lengths, packed
        _append("append8_packed", seqs=13, new=923, cached=0, Hq=16, Hkv=4, D=128, page=64),
        # the same into a cache of the activations' type
        _append("append_norm_packed", seqs=13, new=923, cached=0, Hq=16, Hkv=4, D=128, page=64, cache="same"),
        # the chat server's attention: four short rows that cannot fill the card
        _attention("decode8_few", seqs=4, new=1, cached=700, Hq=8, Hkv=2, D=128, page=16),
        # a loaded server: 256 live sequences of mixed lengths, the cache is the traffic
        _attention("decode8_full", seqs=256, new=1, cached=2600, Hq=32, Hkv=8, D=128, page=64),
        # a chunk of a long prompt after the chunks before it
        _attention("chunk8_long", seqs=1, new=2048, cached=14336, Hq=32, Hkv=8, D=128, page=64),
        # one long instruction before every request: 64 sequences, a token each
        _prefix("prefix_decode", seqs=64, groups=1, prefix=16384, new=1, cached=300, Hq=32, Hkv=8, D=128, page=64),
        # six documents, sixteen questions about each, in the 8-bit cache; prefixes that end inside a page
        _prefix("prefix_groups8", seqs=96, groups=6, prefix=2500, new=1, cached=200, Hq=16, Hkv=4, D=128, page=16,
                cache="fp8"),
        # drafts for 32 sequences behind one prefix are checked at once
        _prefix("prefix_drafts", seqs=32, groups=1, prefix=7000, new=5, cached=500, Hq=16, Hkv=4, D=64, page=16),
        # the chat server with four drafts a sequence
        _verify("verify_few", seqs=4, drafts=4, vocab=50304),
        # the loaded server's
        _verify("verify_full", seqs=64, drafts=5, vocab=131072),
        # drafts looked up in the prompt, without probabilities of their own
        _verify("verify_lookup", seqs=32, drafts=8, vocab=50304, draft="none", dtype="float32"),
    ]


def _append(name, *, seqs, new, cached, Hq, Hkv, D, page, cache="fp8", dtype="bfloat16", rotary=None,
            interleaved=False, norm=True):
    return _named(name, op="append", seqs=seqs, new=new, cached=cached, Hq=Hq, Hkv=Hkv, D=D, page=page, cache=cache,
                  dtype=dtype, rotary=D if rotary is None else rotary, interleaved=interleaved, norm=norm, groups=0,
                  prefix=0)


def _attention(name, *, seqs, new, cached, Hq, Hkv, D, page, dtype="bfloat16"):
    return _named(name, op="attention", seqs=seqs, new=new, cached=cached, Hq=Hq, Hkv=Hkv, D=D, page=page,
                  cache="fp8", dtype=dtype, groups=0, prefix=0)


def _prefix(name, *, seqs, groups, prefix, new, cached, Hq, Hkv, D, page, cache="same", dtype="bfloat16"):
    return _named(name, op="prefix", seqs=seqs, groups=groups, prefix=prefix, new=new, cached=cached, Hq=Hq, Hkv=Hkv,
                  D=D, page=page, cache=cache, dtype=dtype)


def _verify(name, *, seqs, drafts, vocab, draft="logits", dtype="bfloat16"):
    return _named(name, op="verify", seqs=seqs, drafts=drafts, vocab=vocab, draft=draft, dtype=dtype)


def _named(name, **case):
    return case if name is None else {"name": name, **case}


def draw(rng) -> dict:
    """One more case of the same ranges, sizes spread over their logarithm."""
    op = rng.choice(("append", "attention", "attention", "prefix", "prefix", "verify"))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    if op == "verify":
        seqs, drafts = _log_int(rng, 1, 64), rng.randint(1, 8)
        vocab = _log_int(rng, 1000, min(160000, 2 ** 25 // (seqs * (drafts + 1))))
        return _verify(None, seqs=seqs, drafts=drafts, vocab=vocab, dtype=dtype,
                       draft=rng.choice(("logits", "logits", "none")))
    D = rng.choice((64, 128, 128))
    Hkv, G = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 4, 5, 8))
    page = rng.choice((8, 16, 16, 24, 64, 64, 128))
    kind = dict(Hq=Hkv * G, Hkv=Hkv, D=D, page=page, dtype=dtype)
    if op == "prefix":
        seqs = _log_int(rng, 2, 128)
        groups = _log_int(rng, 1, max(1, seqs // 4))
        new = rng.choice((1, 1, 1, rng.randint(2, 9), _log_int(rng, 10, 64)))
        room = min(20000, MAX_CACHED // seqs, MAX_PAIRS // (seqs * new))
        prefix = _log_int(rng, 1, room)
        return _prefix(None, seqs=seqs, groups=groups, prefix=prefix, new=new, cached=_log_int(rng, 1, min(600, room)),
                       cache=rng.choice(("same", "fp8")), **kind)
    form = rng.choice(("decode", "decode", "few", "chunk", "prompt"))
    seqs = _log_int(rng, 1, 256 if form == "decode" else 64 if form == "few" else 16)
    new = {"decode": 1, "few": rng.randint(2, 9)}.get(form) or _log_int(rng, 16, 2048)
    if form in ("chunk", "prompt"):
        new = max(1, min(new, 8192 // seqs))
    cached = 0 if form == "prompt" else _log_int(rng, 1, max(1, min(100000, MAX_CACHED // seqs,
                                                                  MAX_PAIRS // (seqs * new))))
    kind.update(seqs=seqs, new=new, cached=cached)
    if op == "append":
        return _append(None, **kind, cache=rng.choice(("fp8", "fp8", "same")), rotary=rng.choice((D, D, D // 2, 0)),
                       interleaved=rng.random() < 0.3, norm=rng.random() < 0.8)
    return _attention(None, **kind)


def _log_int(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(max(low, high)))))))


def _lengths(case: dict) -> dict:
    """New tokens and own positions of each sequence, mixed around the case's means (the means for one sequence and for
    single tokens); each group's prefix and the sequences that begin a group."""
    rng = random.Random(f"{case['seqs']} {case['new']} {case['cached']} {case['groups']}")
    n, g = case["seqs"], case["groups"]

    def mixed(mean):
        return mean if n == 1 else rng.randint(max(0, mean // 8), mean + mean - mean // 8)

    new = [1 if case["new"] == 1 else max(1, mixed(case["new"])) for _ in range(n)]
    cached = [mixed(case["cached"]) for _ in range(n)]
    prefix = [case["prefix"] if g == 1 else max(1, mixed(case["prefix"])) for _ in range(g)]
    starts = [round(i * n / g) for i in range(g + 1)] if g else [0]
    of = [max(i for i in range(g) if starts[i] <= s) for s in range(n)] if g else []
    return {"new": new, "cached": cached, "prefix": prefix, "groups": starts, "of": of,
            "lens": [a + b + (prefix[of[i]] if g else 0) for i, (a, b) in enumerate(zip(new, cached))]}


def _rows(case: dict) -> list[int]:
    """A row for every draft of a sequence and one for the token after them; every fourth sequence has fewer drafts."""
    rng = random.Random(f"{case['seqs']} {case['drafts']}")
    return [case["drafts"] + 1 if i % 4 else rng.randint(1, case["drafts"] + 1) for i in range(case["seqs"])]


# -- inputs --------------------------------------------------------------------

def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    return (_prepare_verify if case["op"] == "verify" else _prepare_cache)(case, seed, dev, gen, dtype)


def _prepare_cache(case, seed, dev, gen, dtype):
    sizes = _lengths(case)
    new, lens, prefix, groups, of = (sizes[k] for k in ("new", "lens", "prefix", "groups", "of"))
    page, Hq, Hkv, D = case["page"], case["Hq"], case["Hkv"], case["D"]
    # whole pages of a prefix are shared; a page that it fills in part is each sequence's own
    shared = [p // page for p in prefix]
    need = [-(-length // page) - (shared[of[i]] if of else 0) for i, length in enumerate(lens)]
    pages = sum(need) + sum(shared) + 8
    # the pool in use for a while: a sequence's pages lie anywhere in it, what is past its length is an earlier one's
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.zeros(len(new), max(-(-length // page) for length in lens), dtype=torch.int32), 0
    for g, n in enumerate(shared):
        table[groups[g]:groups[g + 1], :n] = order[at:at + n]
        at += n
    for i, n in enumerate(need):
        first = shared[of[i]] if of else 0
        table[i, first:first + n] = order[at:at + n]
        at += n
    table = table.to(dev)
    tokens = sum(new)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dtype)

    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {"case": case, "page_table": table, "seq_lens": ints(lens),
             "cu_seqlens": None if tokens == len(new) else ints(starts),
             "seq": torch.repeat_interleave(torch.arange(len(new), device=dev), ints(new), output_size=tokens)}
    # every token's place among its sequence's new ones, and its position: the plain forms' index
    state["nth"] = torch.arange(tokens, device=dev) - ints(starts)[state["seq"]]
    state["pos"] = (ints(lens) - ints(new))[state["seq"]] + state["nth"]
    for name in ("k", "v"):
        state.update(_pool(name, case["cache"], (pages, page, Hkv, D), gen, dev, dtype))
    if of:
        state.update(cu_groups=ints(groups), prefix_lens=ints(prefix), of=torch.tensor(of, device=dev))
        for g, p in enumerate(prefix):
            if p % page:
                rows = table[groups[g]:groups[g + 1], p // page].long()
                for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
                    if state[name] is not None:
                        x = state[name].view(torch.uint8) if case["cache"] == "fp8" else state[name]
                        x[rows, :p % page] = x[rows[0], :p % page].clone()
    if case["op"] != "append":
        state["q"] = 2 * normal(tokens, Hq, D)
        return state
    # one packed projection, as the layer's matrix product leaves it
    qkv = normal(tokens, (Hq + 2 * Hkv) * D)
    state["q"], state["k"], state["v"] = (t.unflatten(-1, (-1, D)) for t in
                                          qkv.split((Hq * D, Hkv * D, Hkv * D), dim=-1))
    state["q_norm"], state["k_norm"] = ((1 + 0.2 * torch.randn(2, D, generator=gen, device=dev)).unbind()
                                        if case["norm"] else (None, None))
    state["cos"] = state["sin"] = None
    if case["rotary"]:
        r = case["rotary"]
        rate = 10000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)
        angle = torch.arange(table.shape[1] * page, device=dev, dtype=torch.float64)[:, None] * rate
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


def _pool(name, cache, shape, gen, dev, dtype):
    if cache == "same":
        return {name + "_pages": torch.randn(*shape, generator=gen, device=dev).to(dtype), name + "_scales": None}
    codes, scales = torch.empty(shape, dtype=torch.uint8, device=dev), []
    step = max(1, 2 ** 27 // math.prod(shape[1:]))
    for at in range(0, shape[0], step):
        part = codes[at:at + step]
        c, s = _quantised(torch.randn(part.shape, generator=gen, device=dev))
        part.copy_(c.view(torch.uint8))
        scales.append(s.view(torch.uint8))
    return {name + "_pages": codes.view(torch.float8_e4m3fn), name + "_scales": torch.cat(scales).view(torch.float8_e8m0fnu)}


def _prepare_verify(case, seed, dev, gen, dtype):
    rng = random.Random(seed)
    n, vocab, rows = case["seqs"], case["vocab"], _rows(case)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    N = starts[-1]
    seq = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(rows, device=dev), output_size=N)
    cu = torch.tensor(starts, dtype=torch.int32, device=dev)

    def gumbel(*shape):
        return torch.empty(*shape, device=dev).exponential_(generator=gen).log_().neg_()

    logits = 3 * torch.randn(N, vocab, generator=gen, device=dev)
    draft = logits + 0.7 * torch.randn(N, vocab, generator=gen, device=dev)  # a smaller model's, near the target's
    temperature = torch.tensor([rng.choice((0.0, 1.0, rng.uniform(0.5, 1.2), rng.uniform(0.5, 1.2))) for _ in range(n)],
                               dtype=torch.float32, device=dev)
    heat = temperature[seq][:, None]
    logits, draft = logits.to(dtype), draft.to(dtype)
    z = torch.where(heat > 0, draft.float() / torch.where(heat > 0, heat, 1.0) + gumbel(N, vocab), draft.float())
    return {"case": case, "cu_seqlens": cu, "seq": seq, "logits": logits,
            "draft_logits": draft if case["draft"] == "logits" else None, "drafts": z.argmax(-1).int(),
            "uniform": torch.rand(N, generator=gen, device=dev), "noise": gumbel(n, vocab), "temperature": temperature}


# -- one pass ------------------------------------------------------------------

def run(state: dict):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "prefix": _own_prefix, "verify": _own_verify}[op](state)
    return {"append": _plain_append, "attention": _plain_attention, "prefix": _plain_prefix,
            "verify": _plain_verify}[op](state)


def _own_append(s):
    from delta_feedback_experiment_amd import paged_append_, paged_append_fp8_
    more = dict(cu_seqlens=s["cu_seqlens"], q=s["q"], cos=s["cos"], sin=s["sin"], q_norm=s["q_norm"],
                k_norm=s["k_norm"], eps=1e-6, interleaved=s["case"]["interleaved"])
    if s["case"]["cache"] == "fp8":
        q = paged_append_fp8_(s["k"], s["v"], s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"],
                              s["page_table"], s["seq_lens"], **more)
    else:
        q = paged_append_(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"], **more)
    return {"q": q, **_cache(s)}


def _own_attention(s):
    from delta_feedback_experiment_amd import paged_attention_fp8
    o, lse = paged_attention_fp8(s["q"], s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["page_table"],
                                 s["seq_lens"], cu_seqlens=s["cu_seqlens"])
    return {"o": o, "lse": lse}


def _own_prefix(s):
    from delta_feedback_experiment_amd import paged_prefix_attention
    o, lse = paged_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"], s["cu_groups"],
                                    s["prefix_lens"], k_scales=s["k_scales"], v_scales=s["v_scales"],
                                    cu_seqlens=s["cu_seqlens"])
    return {"o": o, "lse": lse}


def _own_verify(s):
    from delta_feedback_experiment_amd import verify_tokens
    tokens, accepted = verify_tokens(s["logits"], s["drafts"], s["uniform"], s["noise"], s["cu_seqlens"],
                                     draft_logits=s["draft_logits"], temperature=s["temperature"])
    return {"tokens": tokens, "accepted": accepted}


def _cache(s):
    return {k: s[k] for k in ("k_pages", "v_pages", "k_scales", "v_scales") if s[k] is not None}


# -- the plain forms -----------------------------------------------------------

def _quantised(x):
    """Codes and scales of ``x`` by blocks of 32 channels: the least power of two by which a block fits +-448."""
    x = x.unflatten(-1, (-1, BLOCK))
    mantissa, exponent = torch.frexp((x.abs().amax(-1, keepdim=True) / 448).clamp(2.0 ** -117, 2.0 ** 119))
    scale = torch.ldexp(torch.ones_like(mantissa), exponent - (mantissa == 0.5).int())
    return (x / scale).to(torch.float8_e4m3fn).flatten(-2), scale[..., 0].to(torch.float8_e8m0fnu)


def _values(codes, scales):
    """What a cache's rows stand for, in 32 bits."""
    if scales is None:
        return codes.float()
    return (codes.float().unflatten(-1, (-1, BLOCK)) * scales.float()[..., None]).flatten(-2)


def _rotated(x, cos, sin, interleaved):
    """The first channels of every head turned by their position's angles, in 32 bits."""
    half = cos.shape[-1]
    c, d = cos[:, None], sin[:, None]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    turned = (a * c - b * d, b * c + a * d)
    head = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((head, rest), -1)


def _plain_append(s):
    page = s["case"]["page"]
    where = (s["page_table"].long()[s["seq"], s["pos"] // page], s["pos"] % page)

    def placed(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
        return x if s["cos"] is None else _rotated(x, s["cos"][s["pos"]], s["sin"][s["pos"]], s["case"]["interleaved"])

    q, k, v = placed(s["q"], s["q_norm"]), placed(s["k"], s["k_norm"]), s["v"].float()
    if s["case"]["cache"] == "fp8":
        (k, k_scale), (v, v_scale) = _quantised(k), _quantised(v)
        for pool, x in (("k_pages", k), ("v_pages", v), ("k_scales", k_scale), ("v_scales", v_scale)):
            s[pool].view(torch.uint8)[where] = x.view(torch.uint8)
    else:
        s["k_pages"][where], s["v_pages"][where] = k.to(s["k"].dtype), v.to(s["k"].dtype)
    return {"q": q.to(s["q"].dtype), **_cache(s)}


def _gathered(s, table, begin, length):
    """Keys and values of ``length`` positions of each row of the table from ``begin`` (one number a row), in 32 bits,
    and the positions; those past the table's end are its last one again."""
    page = s["case"]["page"]
    place = begin[:, None] + torch.arange(length, device=begin.device)
    held = place.clamp(max=table.shape[1] * page - 1)
    where = (table.gather(1, held // page).long(), held % page)

    def rows(pool, scales):
        return _values(s[pool][where], None if s[scales] is None else s[scales][where])

    return rows("k_pages", "k_scales"), rows("v_pages", "v_scales"), place


def _padded(s, of, nth, batch):
    """Queries (in 32 bits, scaled) and positions by batch row and place in it; places without a token see nothing."""
    most = int(max(1, s["places"]))
    q = torch.zeros(batch, most, *s["q"].shape[1:], device=of.device)
    pos = torch.full((batch, most), -1, device=of.device)
    q[of, nth], pos[of, nth] = s["q"].float() * s["case"]["D"] ** -0.5, s["pos"]
    return q, pos


def _part(q, k, v, seen):
    """Maximum, sum and weighted values of each query's softmax over some of its keys."""
    (B, n, Hq, D), Hkv = q.shape, k.shape[2]
    G = Hq // Hkv
    rows = q.unflatten(2, (Hkv, G)).permute(0, 2, 1, 3, 4).reshape(B * Hkv, n * G, D)
    scores = torch.bmm(rows, k.permute(0, 2, 3, 1).reshape(B * Hkv, D, -1).contiguous()).view(B, Hkv, n, G, -1)
    scores.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    w = (scores - top.clamp(min=torch.finfo(torch.float32).min)).exp_()
    out = torch.bmm(w.view(B * Hkv, n * G, -1), v.transpose(1, 2).reshape(B * Hkv, -1, D).contiguous())

    def back(x):
        return x.view(B, Hkv, n, G, -1).permute(0, 2, 1, 3, 4).reshape(B, n, Hq, -1)

    return back(top), back(w.sum(-1)), back(out)


def _own_part(s, begin):
    """Every token's softmax over its sequence's positions from ``begin`` (one number a sequence)."""
    sizes = _lengths(s["case"])
    s["places"] = max(sizes["new"])
    q, pos = _padded(s, s["seq"], s["nth"], len(sizes["new"]))
    k, v, place = _gathered(s, s["page_table"], begin, max(a + b for a, b in zip(sizes["new"], sizes["cached"])))
    return [x[s["seq"], s["nth"]] for x in _part(q, k, v, place[:, None] <= pos[..., None])]


def _result(s, top, total, out):
    return {"o": (out / total).to(s["q"].dtype), "lse": (top + total.log())[..., 0]}


def _plain_attention(s):
    return _result(s, *_own_part(s, torch.zeros_like(s["seq_lens"]).long()))


def _plain_prefix(s):
    sizes = _lengths(s["case"])
    of, starts = s["of"][s["seq"]], sizes["groups"]
    counts = [sum(sizes["new"][a:b]) for a, b in zip(starts, starts[1:])]  # each group's tokens
    first = torch.searchsorted(of, torch.arange(len(counts), device=of.device))
    nth = torch.arange(of.numel(), device=of.device) - first[of]
    s["places"] = max(counts)
    q, _ = _padded(s, of, nth, len(counts))
    rows = s["page_table"][s["cu_groups"][:-1].long()]
    k, v, place = _gathered(s, rows, torch.zeros_like(s["prefix_lens"]).long(), max(sizes["prefix"]))
    seen = (place < s["prefix_lens"][:, None])[:, None].expand(-1, q.shape[1], -1)
    one = [x[of, nth] for x in _part(q, k, v, seen)]
    two = _own_part(s, s["prefix_lens"].long()[s["of"]])
    top = torch.maximum(one[0], two[0])
    a, b = (one[0] - top).exp(), (two[0] - top).exp()
    return _result(s, top, one[1] * a + two[1] * b, one[2] * a + two[2] * b)


def _plain_verify(s):
    logits, drafts, cu, seq = s["logits"].float(), s["drafts"].long(), s["cu_seqlens"].long(), s["seq"]
    vocab, dev = logits.shape[1], logits.device
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, 1.0, s["temperature"])[seq]

    def log_probs(x, rows):
        z = (x - x.amax(-1, keepdim=True)) / heat[rows][:, None]
        return z - z.exp().sum(-1, keepdim=True).log()

    every = torch.arange(len(seq), device=dev)
    best = torch.where(logits == logits.amax(-1, keepdim=True), torch.arange(vocab, device=dev), vocab).amin(-1)
    p = log_probs(logits, every).gather(1, drafts[:, None])[:, 0].exp()
    q = torch.ones_like(p)
    if s["draft_logits"] is not None:
        q = log_probs(s["draft_logits"].float(), every).gather(1, drafts[:, None])[:, 0].exp()
    nth = every - cu[:-1][seq]
    last = every == cu[1:][seq] - 1
    taken = torch.where(greedy[seq], drafts == best, s["uniform"] * q < p) & ~last
    # accepted: the drafts before the first that is not
    stop = torch.full_like(cu[1:], len(seq)).scatter_reduce(0, seq, torch.where(taken, len(seq), nth), "amin")
    at = cu[:-1] + stop
    # the next token's distribution, in 64 bits: what is left of p next to q is a difference
    probs = log_probs(logits[at].double(), at).exp()
    if s["draft_logits"] is not None:
        other = log_probs(s["draft_logits"][at].double(), at).exp()
    else:
        other = torch.zeros_like(probs).scatter_(1, drafts[at][:, None], 1.0)
    left = torch.where(last[at][:, None], probs, (probs - other).clamp(min=0))
    left = torch.where((left > 0).any(-1, keepdim=True), left, probs)
    token = torch.where(greedy, best[at], (left.log() + s["noise"]).argmax(-1))
    tokens = torch.where(nth < stop[seq], drafts, torch.where(nth == stop[seq], token[seq], -1))
    return {"tokens": tokens.int(), "accepted": stop.int()}


# -- the definition in 64 bits -------------------------------------------------

def exact(case: dict, seed: int):
    state = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "prefix": _exact_attention,
            "verify": _exact_verify}[case["op"]](state)


def _exact_blocks(x):
    """Codes' values and scales in 64 bits."""
    x = x.unflatten(-1, (-1, BLOCK))
    scale = 2.0 ** torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448)).clamp(-117, 119)
    y = x / scale
    # three bits after the first of a normal number, steps of 2^-9 under 2^-6
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).flatten(-2), scale[..., 0]


def _exact_append(s):
    case = s["case"]
    r, page = case["rotary"], case["page"]
    both = []
    for x, weight in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        x = x.double().contiguous()
        if weight is not None:
            x = x * weight.double() / (x.pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6).sqrt()
        if r:
            turn = torch.complex(s["cos"][s["pos"]].double(), s["sin"][s["pos"]].double())[:, None]
            first = slice(0, r, 2) if case["interleaved"] else slice(0, r // 2)
            second = slice(1, r, 2) if case["interleaved"] else slice(r // 2, r)
            turned = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
            x[..., first], x[..., second] = turned.real, turned.imag
        both.append(x)
    out = {"q": both[0], **{k: x.double() for k, x in _cache(s).items()}}
    k, v = both[1], s["v"].double()
    if case["cache"] == "fp8":
        (k, ks), (v, vs) = _exact_blocks(k), _exact_blocks(v)
    slot = s["page_table"].flatten()[s["seq"] * s["page_table"].shape[1] + s["pos"] // page].long() * page + s["pos"] % page
    for name, x in (("k_pages", k), ("v_pages", v)) + ((("k_scales", ks), ("v_scales", vs)) if case["cache"] == "fp8" else ()):
        out[name].view(-1, *x.shape[1:])[slot] = x
    return out


def _exact_attention(s):
    case, sizes = s["case"], _lengths(s["case"])
    G, D, page, dev = case["Hq"] // case["Hkv"], case["D"], case["page"], s["q"].device
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device=dev)
    at = 0
    for i, (n, length) in enumerate(zip(sizes["new"], sizes["lens"])):
        place = torch.arange(length, device=dev)
        rows = s["page_table"][i].long()[place // page] * page + place % page
        seen = place[None] <= torch.arange(length - n, length, device=dev)[:, None]
        for h in range(case["Hkv"]):
            k, v = (s[x + "_pages"].flatten(0, 1)[rows, h].double() for x in "kv")
            if case["cache"] == "fp8":
                k, v = (t * s[x + "_scales"].flatten(0, 1)[rows, h].double().repeat_interleave(BLOCK, -1)
                        for t, x in ((k, "k"), (v, "v")))
            q = s["q"][at:at + n, h * G:(h + 1) * G].double()  # [n, G, D]
            logit = (q.flatten(0, 1) @ k.t()).view(n, G, length) / math.sqrt(D)
            logit = torch.where(seen[:, None], logit, -math.inf)
            norm = torch.logsumexp(logit, -1)
            prob = (logit - norm[..., None]).exp()
            o[at:at + n, h * G:(h + 1) * G] = (prob.flatten(0, 1) @ v).view(n, G, D)
            lse[at:at + n, h * G:(h + 1) * G] = norm
        at += n
    return {"o": o, "lse": lse}


def _exact_verify(s):
    cu = s["cu_seqlens"].tolist()
    tokens, accepted = torch.full((cu[-1],), -1, dtype=torch.int32), []
    for n, t in enumerate(s["temperature"].double().tolist()):
        for row in range(cu[n], cu[n + 1]):
            x = s["logits"][row].double()
            d = int(s["drafts"][row])
            final = row == cu[n + 1] - 1
            if t <= 0:
                token = int((x == x.max()).nonzero()[0])
                if not final and token == d:
                    tokens[row] = d
                    continue
                break
            p = torch.softmax(x / t, 0)
            if s["draft_logits"] is None:
                q = torch.zeros_like(p)
                q[d] = 1.0
            else:
                q = torch.softmax(s["draft_logits"][row].double() / t, 0)
            if not final and float(s["uniform"][row]) * float(q[d]) < float(p[d]):
                tokens[row] = d
                continue
            rest = p if final else torch.relu(p - q)
            token = int((torch.log(rest) + s["noise"][n].double()).argmax())
            break
        tokens[row] = token
        accepted.append(row - cu[n])
    dev = s["logits"].device
    return {"tokens": tokens.to(dev), "accepted": torch.tensor(accepted, dtype=torch.int32, device=dev)}


# -- the work of one pass ------------------------------------------------------

def work(case: dict) -> dict:
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "verify":
        rows = sum(_rows(case))
        # every row's logits, the drafts' too, and the noise of one row a sequence
        sides = 2 if case["draft"] == "logits" else 1
        n = case["vocab"] * (sides * rows - (case["seqs"] if sides == 2 else 0))
        return {"bytes": size * n + 4 * case["seqs"] * case["vocab"] + 16 * rows, "flops": 4 * n}
    sizes = _lengths(case)
    new, cached, prefix = sizes["new"], sizes["cached"], sizes["prefix"]
    tokens, Hq, Hkv, D = sum(new), case["Hq"], case["Hkv"], case["D"]
    stored = size * D if case["cache"] == "same" else D + D // BLOCK  # a head's row in the cache
    table = 4 * (sum(-(-(a + b) // case["page"]) for a, b in zip(new, cached)) + sum(p // case["page"] for p in prefix))
    if case["op"] == "append":
        return {"bytes": size * tokens * (2 * Hq + 2 * Hkv) * D + 2 * tokens * Hkv * stored
                + 4 * tokens * case["rotary"] + table,
                "flops": tokens * ((Hq + Hkv) * (3 * case["rotary"] + 4 * D) + 2 * Hkv * 3 * D)}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
    if prefix:
        pairs += sum(n * prefix[g] for n, g in zip(new, sizes["of"]))
    return {"bytes": size * 2 * tokens * Hq * D + 2 * Hkv * stored * (tokens + sum(cached) + sum(prefix))
            + 4 * tokens * Hq + table, "flops": 4 * D * Hq * pairs}
