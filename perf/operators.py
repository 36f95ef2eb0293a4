"""Operators of a serving step over a paged KV cache, measured on one MI355X: the QK-norm + RoPE that
writes new keys and values into pages, the attention of new tokens (one or many per sequence) over
those pages, and the logits' penalties, biases and token masks before a token is picked.

``listed`` holds the measured cases, ``draw`` spreads over the same ranges. Head layouts, histories and
vocabularies are those of the benchmark's configurations (Qwen3-0.6B and 4B widths, 8192-position
histories, 4096-row sweeps, 151936 logits) and of the parity tests (head_dim 64 and 256, 40960
positions). All inputs come from the seed through torch's generators; lengths come from the case alone.

With ``own`` false the operators run in their plain form, elementary torch operations in 32 bits (angles
in 64) rounded once at the end; with ``own`` true through the library's entry points.
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
EPS = 1e-6


def _package():
    if "llm_inference_amd" not in sys.modules:
        home = ROOT / "llm-inference_amd"
        spec = importlib.util.spec_from_file_location(
            "llm_inference_amd", home / "__init__.py", submodule_search_locations=[str(home)])
        module = importlib.util.module_from_spec(spec)
        sys.modules["llm_inference_amd"] = module
        spec.loader.exec_module(module)
    return sys.modules["llm_inference_amd"]


# ---- cases ----

def _append(**c):
    return dict(dict(kind="append", theta=1e6, norm=True, rotary=c["dim"], interleaved=False, stretch=1.0,
                     origin=40960, fused=True), **c)


def _attend(**c):
    return dict(dict(kind="attend", window=0), **c)


def listed():
    return [
        # one sequence's next token at 0.6B heads, a short conversation
        _append(name="append_token", heads=16, kv_heads=8, dim=128, seqs=1, chunks=0, new=1, past=260, page=16, mix=1),
        # the next token of 64 conversations at 4B heads
        _append(name="append_batch", heads=32, kv_heads=8, dim=128, seqs=64, chunks=0, new=1, past=2047, page=16, mix=2),
        # the rows of several prompts at 4B heads
        _append(name="append_prompts", heads=32, kv_heads=8, dim=128, seqs=5, chunks=5, new=1500, past=700, page=64, mix=3),
        # part of each head rotated in interleaved pairs, no norms, positions stretched past the trained length
        _append(name="append_partial", heads=12, kv_heads=4, dim=64, rotary=32, interleaved=True, norm=False,
                theta=1e4, stretch=4.0, origin=32768, fused=False, seqs=3, chunks=3, new=701, past=90000, page=32, mix=4),
        # one new token of one conversation at 0.6B heads: the smallest attention call
        _attend(name="attend_token", heads=16, kv_heads=8, dim=128, seqs=1, chunks=0, new=1, past=260, page=16, mix=5),
        # one new token after a very long document at 4B heads
        _attend(name="attend_document", heads=32, kv_heads=8, dim=128, seqs=1, chunks=0, new=1, past=40959, page=64, mix=6),
        # the next token of 64 conversations of unequal length at 4B heads
        _attend(name="attend_batch", heads=32, kv_heads=8, dim=128, seqs=64, chunks=0, new=1, past=8447, page=16, mix=7),
        # a chunk of a long prompt after what is already cached, at 4B heads: the largest product
        _attend(name="attend_chunk", heads=32, kv_heads=8, dim=128, seqs=1, chunks=1, new=2048, past=6144, page=64, mix=8),
        # a mixed step: chunks of two prompts beside the next tokens of 20 conversations, 0.6B heads
        _attend(name="attend_mixed", heads=16, kv_heads=8, dim=128, seqs=22, chunks=2, new=511, past=4095, page=32, mix=9),
        # sliding-window layers with six query heads to a kv head and small heads, two prompts' chunks
        _attend(name="attend_window", heads=24, kv_heads=4, dim=64, seqs=2, chunks=2, new=1501, past=5000, page=16, window=1024, mix=10),
        # a token pick for one conversation: penalties over its history, a few biases, a grammar's mask
        dict(name="penalty_row", kind="penalty", rows=1, vocab=151936, history=700, biases=12, mask=True, mix=11),
        # the same for a batch with long histories
        dict(name="penalty_batch", kind="penalty", rows=64, vocab=151936, history=8192, biases=300, mask=True, mix=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    bound = {c["kind"]: work(c) for c in listed() if c["name"] in ("append_prompts", "penalty_batch")}
    bound["attend"] = dict(bytes=work(listed()[6])["bytes"], flops=work(listed()[7])["flops"])
    while True:
        kind = rng.choice(["append", "attend", "attend", "penalty"])
        mix = rng.randrange(1 << 20)
        if kind == "penalty":
            c = dict(kind=kind, rows=_log(rng, 1, 64), vocab=_log(rng, 1000, 151936), history=_log(rng, 1, 8192),
                     biases=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.7, mix=mix)
        else:
            dim, kv_heads = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
            seqs = _log(rng, 1, 64)
            c = dict(heads=kv_heads * rng.choice([1, 2, 3, 4, 6, 8]), kv_heads=kv_heads, dim=dim, seqs=seqs,
                     chunks=rng.choice([0, 0, rng.randint(0, seqs), min(seqs, 2)]), new=_log(rng, 1, 2048),
                     page=rng.choice([1, 16, 16, 24, 32, 64, 128]), mix=mix)
            if kind == "attend":
                c = _attend(**c, past=_log(rng, 1, 40960), window=rng.choice([0, 0, _log(rng, 1, 4096)]))
            else:
                rotary = rng.choice([dim, dim, dim // 2, 16])
                c = _append(**c, past=_log(rng, 1, 2048), rotary=rotary, interleaved=rng.random() < 0.4,
                            norm=rng.random() < 0.7, theta=rng.choice([1e4, 1e6]), fused=rng.random() < 0.6,
                            stretch=rng.choice([1.0, 1.0, 4.0]), origin=32768)
            lengths = _lengths(c)
            longest = max(new + past for new, past in lengths)
            # what the plain form lays out padded: keys of every sequence, scores of every query
            if (seqs * longest * kv_heads * dim > 6e8
                    or kind == "attend" and seqs * c["heads"] * max(new for new, _ in lengths) * longest > 9e8):
                continue
        cost = work(c)
        if cost["bytes"] <= bound[kind]["bytes"] and cost["flops"] <= bound[kind]["flops"]:
            return c


def _lengths(c):
    """(new tokens, tokens cached before them) of each sequence; the first has the most of both."""
    r = random.Random(c["mix"])
    spread = [(r.random(), r.random()) for _ in range(c["seqs"])]
    return [((c["new"] if i == 0 else 1 + int(a * (c["new"] - 1))) if i < c["chunks"] else 1,
             c["past"] if i == 0 else int(b * c["past"])) for i, (a, b) in enumerate(spread)]


def _history_lengths(c):
    """(prompt tokens, all tokens) of each row; the first has the longest history."""
    r = random.Random(c["mix"])
    spread = [(r.random(), r.random()) for _ in range(c["rows"])]
    whole = [c["history"] if i == 0 else int(a * (c["history"] + 1)) for i, (a, _) in enumerate(spread)]
    return [(int(b * (n + 1)), n) for n, (_, b) in zip(whole, spread)]


def _visible(c, new, past):
    """(pairs of query and visible key, keys that any query of the sequence sees)"""
    w = c["window"] or new + past
    pairs = sum(min(w, past + i + 1) for i in range(new))
    return pairs, min(past + new, w - 1 + new)


def work(c):
    if c["kind"] == "penalty":
        read = c["rows"] * c["vocab"] * 2 + sum(4 * n for _, n in _history_lengths(c)) + c["rows"] * 8 * c["biases"]
        if c["mask"]:
            read += c["rows"] * (c["vocab"] + 31) // 32 * 4
        return dict(bytes=read + c["rows"] * c["vocab"] * 2, flops=4 * c["rows"] * c["vocab"])
    lengths = _lengths(c)
    tokens = sum(new for new, _ in lengths)
    row = c["heads"] * c["dim"] * 2
    if c["kind"] == "append":
        kv_row = c["kv_heads"] * c["dim"] * 2
        return dict(bytes=2 * tokens * (row + 2 * kv_row), flops=tokens * (c["heads"] + c["kv_heads"]) * c["dim"] * 8)
    seen = [_visible(c, new, past) for new, past in lengths]
    return dict(bytes=2 * tokens * row + sum(k for _, k in seen) * c["kv_heads"] * c["dim"] * 4,
                flops=4 * c["dim"] * c["heads"] * sum(p for p, _ in seen))


# ---- inputs ----

def _frequencies(c):
    """Radians per position of each rotated pair, in 64 bits, and the factor of cos and sin. With
    stretch > 1 slow pairs turn 1 / stretch as fast, fast ones as before, with a ramp between the pairs that
    turn 32 times and once over the trained length (YaRN)."""
    half = c["rotary"] // 2
    base = [c["theta"] ** (-2.0 * j / c["rotary"]) for j in range(half)]
    if c["stretch"] == 1.0:
        return base, 1.0

    def pair_that_turns(n):
        return c["rotary"] * math.log(c["origin"] / (n * 2 * math.pi)) / (2 * math.log(c["theta"]))

    low, high = max(math.floor(pair_that_turns(32)), 0), min(math.ceil(pair_that_turns(1)), c["rotary"] - 1)
    high = high + 0.001 if high == low else high
    ramp = [min(1.0, max(0.0, (j - low) / (high - low))) for j in range(half)]
    return ([f * (1 - t) + f / c["stretch"] * t for f, t in zip(base, ramp)], 0.1 * math.log(c["stretch"]) + 1.0)


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(BF16)

    def uniform(*shape, lo, hi):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    def whole(*shape, hi):
        return torch.randint(0, hi, shape, generator=g, device="cuda", dtype=I32)

    def ints(values):
        return torch.tensor(values, dtype=I32, device="cuda")

    s = dict(c=c)
    if c["kind"] == "penalty":
        rows, vocab = c["rows"], c["vocab"]
        lengths = _history_lengths(c)
        # tokens of a text come again and again: low ids far more often than high ones
        ids = (uniform(rows, c["history"], lo=0, hi=1) ** 3 * vocab).to(I32).clamp_(max=vocab - 1)
        s.update(logits=normal(rows, vocab, std=3.0), out=torch.empty(rows, vocab, dtype=BF16, device="cuda"),
                 tokens=ids, prompt_len=ints([p for p, _ in lengths]), token_len=ints([n for _, n in lengths]),
                 repetition=uniform(rows, lo=1.0, hi=1.5), frequency=uniform(rows, lo=0.0, hi=0.5),
                 presence=uniform(rows, lo=0.0, hi=0.8), bias_tokens=None, bias=None, bias_len=None, allowed=None)
        if c["biases"]:
            s.update(bias_tokens=whole(rows, c["biases"], hi=vocab), bias=uniform(rows, c["biases"], lo=-5.0, hi=5.0),
                     bias_len=ints([c["biases"]] * rows))
        if c["mask"]:
            words = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g, device="cuda")
            s["allowed"] = words.to(I32)
        return s
    lengths = _lengths(c)
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    tokens = sum(new for new, _ in lengths)
    pages = [-(-(new + past) // page) for new, past in lengths]
    order = torch.randperm(sum(pages) + 3, generator=g, device="cuda").to(I32)
    table = torch.full((len(pages), max(pages)), -1, dtype=I32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for new, _ in lengths:
        starts.append(starts[-1] + new)
    s.update(page_table=table, q_start=ints(starts), kv_len=ints([new + past for new, past in lengths]),
             max_q_len=max(new for new, _ in lengths), max_kv_len=max(new + past for new, past in lengths),
             key_cache=normal(sum(pages) + 3, page, kv_heads, dim), value_cache=normal(sum(pages) + 3, page, kv_heads, dim))
    out = torch.zeros(tokens, heads, dim, dtype=BF16, device="cuda")
    if c["kind"] == "attend":
        s.update(out=out, q=normal(tokens, heads, dim, std=1.5), scale=1 / math.sqrt(dim), ws=None)
        if own:  # the workspace that a program keeps for these calls
            floats = _package().attention_paged_workspace_floats(
                tokens, len(lengths), heads, kv_heads, dim, s["max_q_len"], s["max_kv_len"])
            s["ws"] = torch.empty(max(floats, 1), dtype=F32, device="cuda")
        return s
    if c["fused"]:  # the rows of one q/k/v projection
        rows = normal(tokens, heads + 2 * kv_heads, dim)
        s.update(q=rows[:, :heads], k=rows[:, heads:heads + kv_heads], v=rows[:, heads + kv_heads:])
    else:
        s.update(q=normal(tokens, heads, dim), k=normal(tokens, kv_heads, dim), v=normal(tokens, kv_heads, dim))
    frequencies, factor = _frequencies(c)
    s.update(q_out=out, q_norm=None, k_norm=None, factor=factor,
             inv_freq=torch.tensor(frequencies, dtype=F64, device="cuda"))
    if c["norm"]:
        s.update(q_norm=normal(dim, std=0.1, mean=1.0), k_norm=normal(dim, std=0.1, mean=1.0))
    return s


# ---- one pass ----

def run(s):
    c = s["c"]
    if c["kind"] == "append":
        (_append_own if own else _append_plain)(s)
        return dict(q=s["q_out"], key_cache=s["key_cache"], value_cache=s["value_cache"])
    if c["kind"] == "attend":
        (_attend_own if own else _attend_plain)(s)
        return s["out"]
    (_penalty_own if own else _penalty_plain)(s)
    return s["out"]


def _append_own(s):
    _package().qk_norm_rope_paged(
        s["q_out"], s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], s["inv_freq"], s["key_cache"],
        s["value_cache"], s["page_table"], s["q_start"], s["kv_len"], EPS, s["factor"],
        interleaved=s["c"]["interleaved"])


def _attend_own(s):
    _package().attention_paged_forward(
        s["out"], s["q"], s["key_cache"], s["value_cache"], s["page_table"], s["q_start"], s["kv_len"], s["ws"],
        s["scale"], max_q_len=s["max_q_len"], max_kv_len=s["max_kv_len"], window=s["c"]["window"])


def _penalty_own(s):
    _package().logits_penalty_forward(
        s["out"], s["logits"], s["tokens"], s["prompt_len"], s["token_len"], s["repetition"], s["frequency"],
        s["presence"], s["bias_tokens"], s["bias"], s["bias_len"], s["allowed"])


def _rows(s, tokens):
    """The sequence and the position of each new token."""
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), t, right=True) - 1
    return seq, s["kv_len"][seq].long() - s["q_start"][seq + 1] + t


def _rotated(x, weight, cos, sin, c):
    x = x.to(F32)
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(F32)
    rotary = c["rotary"]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if c["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1).to(BF16)


def _append_plain(s):
    c = s["c"]
    seq, at = _rows(s, s["q"].shape[0])
    angle = at.to(F64)[:, None] * s["inv_freq"]
    cos, sin = ((f(angle) * s["factor"]).to(F32)[:, None] for f in (torch.cos, torch.sin))
    page = s["page_table"][seq, at // c["page"]].long()
    s["q_out"].copy_(_rotated(s["q"], s["q_norm"], cos, sin, c))
    s["key_cache"][page, at % c["page"]] = _rotated(s["k"], s["k_norm"], cos, sin, c)
    s["value_cache"][page, at % c["page"]] = s["v"]


def _attend_plain(s):
    c = s["c"]
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    seqs, new, longest = c["seqs"], s["max_q_len"], s["max_kv_len"]
    seq, at = _rows(s, s["q"].shape[0])
    row = torch.arange(s["q"].shape[0], device="cuda") - s["q_start"][seq]
    # queries [seqs, kv_heads, group * new, dim]; keys and values of every page of the table's rows
    q = torch.zeros(seqs, new, heads, dim, device="cuda")
    q[seq, row] = s["q"].to(F32)
    q = q.view(seqs, new, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, dim)
    table = s["page_table"].clamp(min=0).long()
    k = s["key_cache"][table].flatten(1, 2)[:, :longest].to(F32).permute(0, 2, 3, 1).contiguous()
    v = s["value_cache"][table].flatten(1, 2)[:, :longest].to(F32).permute(0, 2, 1, 3).contiguous()
    scores = (q @ k).view(seqs, kv_heads, -1, new, longest) * s["scale"]
    where = torch.full((seqs, new), -1, device="cuda")
    where[seq, row] = at
    key = torch.arange(longest, device="cuda")
    seen = key <= where[:, :, None]
    if c["window"]:
        seen &= key > where[:, :, None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=-3e38)  # rows of absent tokens see nothing
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    mixed = (weights.view(seqs, kv_heads, -1, longest) @ v).view(seqs, kv_heads, -1, new, dim)
    mixed = mixed / total.clamp(min=1e-37)
    s["out"].copy_(mixed.permute(0, 3, 1, 2, 4).reshape(seqs, new, heads, dim)[seq, row].to(BF16))


def _penalty_plain(s):
    rows, vocab = s["logits"].shape
    x = s["logits"].to(F32)
    index = torch.arange(s["tokens"].shape[1], device="cuda")
    ids = s["tokens"].long()
    whole, prompt = index < s["token_len"][:, None], index < s["prompt_len"][:, None]
    counts = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, ids, (whole & ~prompt).to(F32))
    seen = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, ids, whole.to(F32)) > 0
    repetition = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - s["frequency"][:, None] * counts - s["presence"][:, None] * (counts > 0)
    if s["bias"] is not None:  # of several entries for a token the last counts
        entry = torch.arange(s["bias"].shape[1], device="cuda").expand(rows, -1)
        last = torch.full((rows, vocab), -1, device="cuda").scatter_reduce_(1, s["bias_tokens"].long(), entry, "amax")
        x = x + torch.where(last >= 0, s["bias"].gather(1, last.clamp(min=0)), 0.0)
    if s["allowed"] is not None:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device="cuda", dtype=I32)) & 1
        x = torch.where(bits.flatten(1)[:, :vocab] != 0, x, -math.inf)
    s["out"].copy_(x.to(BF16))


# ---- the same from the definitions, in 64 bits ----

def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "penalty":
        out = s["logits"].to(F64)
        for r, (prompt, n) in enumerate(_history_lengths(c)):
            ids = s["tokens"][r, :n].long()
            z = out[r]
            met = torch.unique(ids)
            factor = s["repetition"][r].to(F64)
            z[met] = torch.maximum(z[met], z[met] * 0) / factor + torch.minimum(z[met], z[met] * 0) * factor
            answered, times = torch.unique(ids[prompt:], return_counts=True)
            z[answered] -= s["frequency"][r].to(F64) * times + s["presence"][r].to(F64)
            if s["bias"] is not None:
                entries = {int(t): float(b) for t, b in zip(s["bias_tokens"][r].tolist(), s["bias"][r].tolist())}
                z[torch.tensor(list(entries), device="cuda")] += torch.tensor(list(entries.values()), dtype=F64, device="cuda")
            if s["allowed"] is not None:
                word = s["allowed"][r].long() & 0xffffffff
                token = torch.arange(c["vocab"], device="cuda")
                z[(word[token // 32] // 2 ** (token % 32)) % 2 == 0] = -math.inf
        return out
    dim, page, group = c["dim"], c["page"], c["heads"] // c["kv_heads"]
    if c["kind"] == "append":
        def turned(x, weight, at):
            x = x.to(F64)
            if weight is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / dim + EPS) * weight.to(F64)
            n = c["rotary"]
            order = torch.arange(n, device="cuda").view(-1, 2).T if c["interleaved"] else torch.arange(n, device="cuda").view(2, -1)
            z = torch.complex(x[..., order[0]].contiguous(), x[..., order[1]].contiguous())
            angle = at.to(F64)[:, None, None] * s["inv_freq"]
            z = z * torch.polar(torch.full_like(angle, s["factor"]), angle)
            x[..., order[0]], x[..., order[1]] = z.real, z.imag
            return x
        q, keys, values = s["q_out"].to(F64), s["key_cache"].to(F64), s["value_cache"].to(F64)
        t = 0
        for i, (new, past) in enumerate(_lengths(c)):
            at = torch.arange(past, past + new, device="cuda")
            slot = s["page_table"][i].long()[at // page], at % page
            q[t:t + new] = turned(s["q"][t:t + new], s["q_norm"], at)
            keys[slot] = turned(s["k"][t:t + new], s["k_norm"], at)
            values[slot] = s["v"][t:t + new].to(F64)
            t += new
        return dict(q=q, key_cache=keys, value_cache=values)
    out, t = torch.zeros(s["out"].shape, dtype=F64, device="cuda"), 0
    for i, (new, past) in enumerate(_lengths(c)):
        n = new + past
        pages = s["page_table"][i, :-(-n // page)].long()
        at = torch.arange(past, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = (key > at) | ((at - key >= c["window"]) if c["window"] else False)
        for h in range(c["kv_heads"]):
            k, v = (s[name][pages, :, h].reshape(-1, dim)[:n].to(F64) for name in ("key_cache", "value_cache"))
            for j in range(h * group, (h + 1) * group):
                logit = (s["q"][t:t + new, j].to(F64) @ k.T.contiguous() * s["scale"]).masked_fill_(hidden, -math.inf)
                logit -= torch.logsumexp(logit, -1, keepdim=True)
                out[t:t + new, j] = logit.exp_() @ v
        t += new
    return out
